"""The attention half's operators around a paged K/V cache, as a serving program calls them: the step that turns request
lengths into page tables and slots, the append that rotates q and k and writes K and V, and the attention of the new
tokens over the cache.

`listed()` holds the named cases and `draw` makes others of the same ranges; `prepare` builds a case's inputs on the
GPU from a seed, `run` is one pass (by plain torch operations, or through mimo_stream where `own` is set), `work` what
such a pass cannot do without, and `exact` its result in 64 bits.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "mimo-on-a-mac_amd")

E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
GOLDEN = (math.sqrt(5.0) - 1.0) / 2.0

# query heads, K/V heads, key and value dimensions
WIDE = (64, 4, 192, 128)          # keys wider than values, 16 query heads on each K/V head
WIDE8 = (64, 8, 192, 128)
EVEN = (32, 8, 128, 128)
SLIM = (20, 4, 64, 64)            # five query heads on each K/V head


def _step(reqs, ctx, new, chunked=0, page=64, finish=0):
    return {"op": "step", "reqs": reqs, "ctx_lo": ctx[0], "ctx_hi": ctx[1], "new_lo": new[0], "new_hi": new[1],
            "chunked": chunked, "page": page, "finish": finish}


def _heads(dims):
    return {"heads": dims[0], "kv_heads": dims[1], "k_dim": dims[2], "v_dim": dims[3]}


def _append(tokens, dims, rotary, dtype="bf16", page=64, far=131072):
    return dict(_heads(dims), op="append", tokens=tokens, rotary=rotary, theta=10000.0 if rotary < dims[2] else 5.0e6,
                dtype=dtype, page=page, far=far)


def _attend(reqs, ctx, new, dims, chunked=0, page=64, dtype="bf16", window=0, sinks=0, logits=False):
    return dict(_heads(dims), op="attend", reqs=reqs, ctx_lo=ctx[0], ctx_hi=ctx[1], new_lo=new[0], new_hi=new[1],
                chunked=chunked, page=page, dtype=dtype, window=window, sinks=sinks, logits=logits, finish=0)


def listed():
    return [
        # one decoded token for each of a full batch: the step before every forward pass
        dict(_step(256, (1, 8191), (1, 1)), name="step_decode_256"),
        # chunks of prompts beside decoding requests, an eighth of the requests ending: 48 chunks of up to 2048
        dict(_step(1024, (0, 16384), (257, 2048), chunked=48, page=16, finish=8), name="step_chunks_1024"),
        # a decode batch's q, k and v: the call's own latency
        dict(_append(64, WIDE, 64), name="append_decode_64"),
        # a prompt chunk with a rotated part of 64 dimensions, far into a long context
        dict(_append(4096, WIDE8, 64), name="append_chunk_4096"),
        # a ragged chunk into an E4M3 cache, every dimension rotated
        dict(_append(1777, EVEN, 128, dtype="e4m3", page=32, far=16384), name="append_e4m3_1777"),
        # one request deep in a long context: a long axis with few rows
        dict(_attend(1, (32767, 32767), (1, 1), WIDE), name="decode_1x32k"),
        # a ragged decode batch on a layer that sees everything
        dict(_attend(48, (500, 16384), (1, 1), WIDE), name="decode_48"),
        # the same on a sliding-window layer: 128 keys, with sink logits
        dict(_attend(128, (90, 12000), (1, 1), WIDE8, window=128, logits=True), name="decode_window_128"),
        # a decode batch over an E4M3 cache
        dict(_attend(32, (1000, 32768), (1, 1), EVEN, dtype="e4m3"), name="decode_e4m3_32"),
        # the third chunk of a long prompt
        dict(_attend(1, (8192, 8192), (4096, 4096), WIDE, chunked=1), name="chunk_4096_at_8192"),
        # a prompt's chunk on a sliding-window layer with four first tokens visible
        dict(_attend(1, (4096, 4096), (4096, 4096), WIDE8, chunked=1, window=128, sinks=4), name="chunk_window_4096"),
        # prompt pieces of odd sizes beside decoding requests, small pages, five query heads on a K/V head
        dict(_attend(24, (0, 5000), (37, 901), SLIM, chunked=9, page=16, dtype="e4m3", sinks=5, window=1111, logits=True),
             name="mixed_24"),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.random()
    page = rng.choice((16, 32, 64, 128))
    if kind < 0.15:
        reqs = spread(1, 1024)
        chunked = rng.randint(0, min(reqs, 48))
        hi = spread(1, 2048)
        return _step(reqs, (rng.choice((0, 1)), spread(2, 16384)), (rng.randint(1, hi), hi), chunked=chunked, page=page,
                     finish=rng.choice((0, 0, 3, 8)))
    kv = rng.choice((1, 2, 4, 8))
    group = rng.choice((1, 2, 3, 4, 5, 7, 8, 12, 16))
    while kv * group > 64:
        group = rng.choice((1, 2, 3, 4, 5, 7, 8, 12, 16))
    dims = (kv * group, kv) + rng.choice(((64, 64), (128, 128), (192, 128)))
    dtype = rng.choice(("bf16", "bf16", "e4m3"))
    if kind < 0.35:
        rotary = rng.choice((32, 64, dims[2]))
        return _append(spread(1, 4096), dims, rotary, dtype=dtype, page=page, far=spread(4096, 131072))
    window = rng.choice((0, 0, 128, spread(1, 4096)))
    sinks = rng.choice((0, 4, rng.randint(1, 70))) if window else 0
    logits = rng.random() < 0.4
    if kind < 0.7:
        reqs = spread(1, 128)
        hi = spread(16, 20000 if reqs <= 24 else 5000)
        return _attend(reqs, (rng.randint(0, hi), hi), (1, 1), dims, page=page, dtype=dtype, window=window, sinks=sinks,
                       logits=logits)
    reqs = spread(1, 24)
    hi = spread(2, 4096 // max(1, reqs // 2))
    return _attend(reqs, (0, spread(1, 8192)), (rng.randint(1, hi), hi), dims, chunked=rng.randint(1, max(1, reqs // 2)),
                   page=page, dtype=dtype, window=window, sinks=sinks, logits=logits)


# ------------------------------------------------------------------ request lengths
def _between(lo, hi, i):
    """The i-th of evenly spread whole numbers of lo .. hi."""
    return lo + int((hi - lo + 1) * math.modf((i + 1) * GOLDEN)[0])


def _lengths(case):
    """Every request's length before the step and after it."""
    before = [_between(case["ctx_lo"], case["ctx_hi"], i) for i in range(case["reqs"])]
    after = []
    for i, n in enumerate(before):
        if case["finish"] and i % case["finish"] == case["finish"] - 1:
            after.append(0)
        elif i < case["chunked"]:
            after.append(n + _between(case["new_lo"], case["new_hi"], 3 * i + 1))
        else:
            after.append(n + 1)
    return before, after


def _pages(n, page):
    return (n + page - 1) // page


def _new(case):
    return [max(0, b - a) for a, b in zip(*_lengths(case))]


# ------------------------------------------------------------------ inputs (torch alone, from the seed)
def _generator(seed, part):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + part) % (1 << 62))


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _normal(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(torch.bfloat16)


def _page_state(case, lens, g):
    """Page table holding the pages of `lens`, pages in random order, and the list of the free ones."""
    page = case["page"]
    top = max(max(a, b) for a, b in zip(*_lengths(case)))
    width = max(1, _pages(top, page))
    used = sum(_pages(n, page) for n in lens)
    grown = sum(_pages(max(a, b), page) for a, b in zip(*_lengths(case)))
    n_pages = max(used, grown) + max(used, grown) // 8 + 2
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    count = _int32([_pages(n, page) for n in lens]).long()
    table = torch.zeros(len(lens), width, dtype=torch.int32, device="cuda")
    held = torch.arange(width, device="cuda")[None, :] < count[:, None]
    table[held] = order[:used]
    free = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    free[:n_pages - used] = order[used:]
    return table, free, n_pages, n_pages - used


def _scales(heads, base):
    return base * (1.0 + 0.25 * torch.arange(heads, dtype=torch.float32, device="cuda"))


def _inputs(case, seed):
    g = _generator(seed, 1)
    if case["op"] == "step":
        before, after = _lengths(case)
        table, free, n_pages, n_free = _page_state(case, before, g)
        return {"table": table, "free": free, "n_pages": n_pages, "n_free": _int32([n_free]), "lens": _int32(before),
                "target": _int32(after), "tokens": sum(_new(case)), "max_new": max(_new(case))}
    Hq, Hkv, Dk, Dv = case["heads"], case["kv_heads"], case["k_dim"], case["v_dim"]
    e4m3 = case["dtype"] == "e4m3"
    k_scale, v_scale = (_scales(Hkv, 1 / 64), _scales(Hkv, 1 / 80)) if e4m3 else (None, None)
    if case["op"] == "append":
        N, page = case["tokens"], case["page"]
        n_pages = _pages(N, page) + 1
        # q, k and v are views of one projection's rows, as a fused projection leaves them
        rows = _normal(g, N, Hq * Dk + Hkv * (Dk + Dv), scale=1.5)
        order = torch.randperm(n_pages, generator=g, device="cuda")
        at = torch.arange(N, device="cuda")
        first = int(torch.randint(0, case["far"], (1,), generator=g, device="cuda"))
        dtype = E4M3 if e4m3 else torch.bfloat16
        return {"q": rows[:, :Hq * Dk].unflatten(1, (Hq, Dk)), "k": rows[:, Hq * Dk:(Hq + Hkv) * Dk].unflatten(1, (Hkv, Dk)),
                "v": rows[:, (Hq + Hkv) * Dk:].unflatten(1, (Hkv, Dv)),
                "slots": (order[at // page] * page + at % page).to(torch.int32), "positions": (first + at).to(torch.int32),
                "k_pages": torch.zeros(n_pages, Hkv, page, Dk, device="cuda").to(dtype),
                "v_pages": torch.zeros(n_pages, Hkv, page, Dv, device="cuda").to(dtype),
                "k_scale": k_scale, "v_scale": v_scale}
    before, after = _lengths(case)
    table, _, n_pages, _ = _page_state(case, after, g)
    page = case["page"]

    def pages(dim, scale):
        x = torch.empty(n_pages, Hkv, page, dim, dtype=E4M3 if e4m3 else torch.bfloat16, device="cuda")
        for part in range(0, n_pages, 1024):
            y = torch.randn(x[part:part + 1024].shape, generator=g, device="cuda")
            if e4m3:
                y = (y / scale[:, None, None]).clamp(-E4M3_MAX, E4M3_MAX)
            x[part:part + 1024] = y.to(x.dtype)
        return x

    new = _new(case)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return {"q": _normal(g, starts[-1], Hq, Dk, scale=1.5), "k_pages": pages(Dk, k_scale), "v_pages": pages(Dv, v_scale),
            "k_scale": k_scale, "v_scale": v_scale, "table": table, "starts": _int32(starts), "lens": _int32(after),
            "new": new, "after": after, "scale": 1.0 / math.sqrt(Dk),
            "sink_logits": torch.randn(Hq, generator=g, device="cuda") if case["logits"] else None}


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if not own:
        if case["op"] == "append":
            s["inv_freq"] = _inv_freq(case, torch.float64)
        return s
    if PKG not in sys.path:
        sys.path.insert(0, PKG)
    from mimo_stream import attention
    if case["op"] == "step":
        pages = attention.PageTable(case["reqs"], s["table"].shape[1], s["n_pages"], case["page"])
        for name in ("table", "free", "n_free", "lens"):
            getattr(pages, name).copy_(s[name])
        return {"op": "step", "pages": pages, "target": s["target"], "tokens": s["tokens"], "max_new": s["max_new"]}
    cache = attention.KVCache.of(s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"])
    if case["op"] == "append":
        plan = attention.StepPlan(slots=s["slots"], positions=s["positions"])
        return {"op": "append", "cache": cache, "plan": plan, "q": s["q"], "k": s["k"], "v": s["v"],
                "rotary": attention.Rotary(case["rotary"], theta=case["theta"])}
    plan = attention.StepPlan(starts=s["starts"], lens=s["lens"], table=s["table"], max_new=max(s["new"]))
    return {"op": "attend", "q": s["q"], "cache": cache, "plan": plan, "scale": s["scale"], "window": case["window"],
            "sinks": case["sinks"], "sink_logits": s["sink_logits"]}


# ------------------------------------------------------------------ one pass
def run(state):
    if own:
        from mimo_stream import attention
        if state["op"] == "step":
            plan = state["pages"].step(state["target"], state["tokens"], max_new=state["max_new"], commit=False)
            return plan.starts, plan.lens, plan.slots, plan.positions, plan.n_free, plan.table, state["pages"].free
        if state["op"] == "append":
            q = attention.append(state["cache"], state["plan"], state["k"], state["v"], q=state["q"], rotary=state["rotary"])
            return q, state["cache"].k, state["cache"].v
        return attention.attend(state["q"], state["cache"], state["plan"], scale=state["scale"], window=state["window"],
                                sink_tokens=state["sinks"], sink_logits=state["sink_logits"])
    op = state["case"]["op"]
    return {"step": _plain_step, "append": _plain_append, "attend": _plain_attend}[op](state)


# ------------------------------------------------------------------ the plain forms
def _exclusive(counts):
    total = torch.cumsum(counts, 0)
    return total - counts, total[-1]


def _plain_step(s):
    page, N = s["case"]["page"], s["tokens"]
    lens, target, table, free = s["lens"].long(), s["target"].long(), s["table"], s["free"]
    width = table.shape[1]
    new = (target - lens).clamp(min=0)
    first, total = _exclusive(new)
    had, has = (lens + page - 1) // page, (target + page - 1) // page
    column = torch.arange(width, device="cuda")[None, :]
    gone = (column >= has[:, None]) & (column < had[:, None])
    grown = (column >= had[:, None]) & (column < has[:, None])
    freed = table[gone]                                     # requests in order, each one's pages in order
    n_free = s["n_free"].long()
    top = n_free + freed.numel()
    taken = torch.arange(int(grown.sum()), device="cuda")
    stack = torch.cat([free[:int(n_free)], freed.flip(0)])
    table[grown] = stack[top - 1 - taken]
    left = top - taken.numel()
    if int(left) > int(n_free):
        free[int(n_free):int(left)] = stack[int(n_free):int(left)]
    owner = torch.repeat_interleave(torch.arange(lens.numel(), device="cuda"), new, output_size=N)
    positions = lens[owner] + torch.arange(N, device="cuda") - first[owner]
    slots = table[owner, positions // page].long() * page + positions % page
    starts = torch.cat([first, total[None]])
    return (starts.to(torch.int32), target.to(torch.int32), slots.to(torch.int32), positions.to(torch.int32),
            left.to(torch.int32), table, free)


def _inv_freq(case, dtype):
    i = torch.arange(0, case["rotary"], 2, dtype=dtype, device="cuda")
    return torch.pow(torch.tensor(case["theta"], dtype=dtype, device="cuda"), -i / case["rotary"])


def _rotated(x, cos, sin, half):
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _stored(x, scale, dtype):
    if scale is None:
        return x.to(dtype)
    return (x / scale[None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(dtype)


def _plain_append(s):
    case = s["case"]
    half, page = case["rotary"] // 2, case["page"]
    angle = s["positions"].double()[:, None] * s["inv_freq"]
    cos, sin = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]
    q = _rotated(s["q"].float(), cos, sin, half).to(torch.bfloat16)
    k = _rotated(s["k"].float(), cos, sin, half)
    at, row = s["slots"].long() // page, s["slots"].long() % page
    s["k_pages"][at, :, row] = _stored(k, s["k_scale"], s["k_pages"].dtype)
    s["v_pages"][at, :, row] = _stored(s["v"].float(), s["v_scale"], s["v_pages"].dtype)
    return q, s["k_pages"], s["v_pages"]


def _plain_attend(s):
    case = s["case"]
    Hq, Hkv, window, sinks = case["heads"], case["kv_heads"], case["window"], case["sinks"]
    G, page = Hq // Hkv, case["page"]
    outs = []
    at = 0
    for b, (n, length) in enumerate(zip(s["new"], s["after"])):
        first = length - n                                  # position of the first new token
        low = max(0, first - window + 1) if window else 0
        keys = torch.arange(low, length, device="cuda")
        if low and sinks:
            keys = torch.cat([torch.arange(min(low, sinks), device="cuda"), keys])
        at_page, row = s["table"][b].long()[keys // page], keys % page
        K = s["k_pages"][at_page, :, row].float().transpose(0, 1)
        V = s["v_pages"][at_page, :, row].float().transpose(0, 1)
        if s["k_scale"] is not None:
            K, V = K * s["k_scale"][:, None, None], V * s["v_scale"][:, None, None]
        q = s["q"][at:at + n].float().unflatten(1, (Hkv, G)).permute(1, 2, 0, 3)      # [Hkv, G, n, Dk]
        position = torch.arange(first, length, device="cuda")[:, None]
        seen = keys <= position
        if window:
            seen &= (position - keys < window) | (keys < sinks)
        out = torch.empty(n, Hkv, G, case["v_dim"], device="cuda")
        some = max(1, (1 << 28) // (G * n * keys.numel()))  # K/V heads at once: scores of at most a gigabyte or of one head
        for h in range(0, Hkv, some):
            at_heads = slice(h, min(Hkv, h + some))
            score = (q[at_heads].flatten(1, 2) @ K[at_heads].transpose(1, 2)).unflatten(1, (G, n)) * s["scale"]
            score.masked_fill_(~seen, -math.inf)
            top = score.amax(-1, keepdim=True)
            if s["sink_logits"] is not None:
                sink = s["sink_logits"].view(Hkv, G, 1, 1)[at_heads]
                top = torch.maximum(top, sink)
            weight = torch.exp(score - top)
            total = weight.sum(-1, keepdim=True)
            if s["sink_logits"] is not None:
                total = total + torch.exp(sink - top)
            part = (weight.flatten(1, 2) @ V[at_heads]).unflatten(1, (G, n)) / total
            out[:, at_heads] = part.permute(2, 0, 1, 3)
        outs.append(out.flatten(1, 2).to(torch.bfloat16))
        at += n
    return torch.cat(outs)


# ------------------------------------------------------------------ what a pass needs
def _visible(first, n, window, sinks):
    """Keys that n tokens from position `first` on see, summed over the tokens, and the keys that any of them sees."""
    pairs = 0
    for p in range(first, first + n):
        if window and p + 1 > window:
            pairs += window + min(sinks, p + 1 - window)
        else:
            pairs += p + 1
    low = max(0, first - window + 1) if window else 0
    return pairs, first + n - low + min(sinks if window else 0, low)


def work(case):
    if case["op"] == "step":
        before, after = _lengths(case)
        page, N = case["page"], sum(_new(case))
        moved = sum(abs(_pages(b, page) - _pages(a, page)) for a, b in zip(before, after))
        return {"bytes": 4 * (4 * len(before) + 2 * moved + 2 * N), "flops": 0}
    Hq, Hkv, Dk, Dv = case["heads"], case["kv_heads"], case["k_dim"], case["v_dim"]
    size = 1 if case["dtype"] == "e4m3" else 2
    if case["op"] == "append":
        N = case["tokens"]
        return {"bytes": N * (4 * Hq * Dk + Hkv * (Dk + Dv) * (2 + size) + 8), "flops": 3 * N * (Hq + Hkv) * case["rotary"]}
    pairs = keys = 0
    for length, n in zip(_lengths(case)[1], _new(case)):
        p, k = _visible(length - n, n, case["window"], case["sinks"])
        pairs, keys = pairs + p, keys + k
    tokens = sum(_new(case))
    return {"bytes": keys * Hkv * (Dk + Dv) * size + 2 * tokens * Hq * (Dk + Dv), "flops": 2 * pairs * Hq * (Dk + Dv)}


# ------------------------------------------------------------------ 64 bits
def _exact_step(case, s):
    page = case["page"]
    table, free = s["table"].cpu().numpy().copy(), s["free"].cpu().numpy().copy()
    n_free = int(s["n_free"][0])
    before, after = _lengths(case)
    released = [int(table[b, j]) for b, (x, y) in enumerate(zip(before, after)) for j in range(_pages(y, page), _pages(x, page))]
    stack = free[:n_free].tolist() + released[::-1]
    starts, slots, positions = [0], [], []
    for b, (x, y) in enumerate(zip(before, after)):
        for j in range(_pages(x, page), _pages(y, page)):
            table[b, j] = stack.pop()
        for p in range(x, y):
            positions.append(p)
            slots.append(int(table[b, p // page]) * page + p % page)
        starts.append(len(slots))
    if len(stack) > n_free:
        free[n_free:len(stack)] = stack[n_free:]
    return tuple(np.asarray(v, dtype=np.int32) for v in (starts, after, slots, positions, [len(stack)], table, free))


def _exact_append(case, s):
    half, page = case["rotary"] // 2, case["page"]
    freq = case["theta"] ** (-2.0 * torch.arange(half, dtype=torch.float64, device="cuda") / case["rotary"])
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["positions"].double()[:, None] * freq)[:, None, :]

    def rotate(x):
        x = x.double()
        z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn
        x[..., :half], x[..., half:2 * half] = z.real, z.imag
        return x

    k, v = rotate(s["k"]), s["v"].double()
    if s["k_scale"] is not None:
        k, v = k / s["k_scale"].double()[:, None], v / s["v_scale"].double()[:, None]
    kp, vp = s["k_pages"].double(), s["v_pages"].double()
    slot = s["slots"].long()
    for h in range(case["kv_heads"]):
        kp[slot // page, h, slot % page] = k[:, h]
        vp[slot // page, h, slot % page] = v[:, h]
    return rotate(s["q"]), kp, vp


def _exact_attend(case, s):
    Hq, window, sinks, page = case["heads"], case["window"], case["sinks"], case["page"]
    group = Hq // case["kv_heads"]
    out = torch.zeros(s["q"].shape[0], Hq, case["v_dim"], dtype=torch.float64, device="cuda")
    starts = s["starts"].tolist()
    for b, length in enumerate(s["lens"].tolist()):
        n = starts[b + 1] - starts[b]
        count = _pages(length, page)
        K = s["k_pages"][s["table"][b, :count].long()].double()             # [pages, Hkv, page, Dk]
        V = s["v_pages"][s["table"][b, :count].long()].double()
        for part in range(0, n, 1024):
            rows = torch.arange(part, min(n, part + 1024), device="cuda")
            i = (length - n + rows)[:, None]
            lo = max(0, length - n + part - window + 1) if window else 0
            j = torch.cat([torch.arange(min(lo, sinks), device="cuda"), torch.arange(lo, length, device="cuda")])
            hidden = j > i
            if window:
                hidden = hidden | ((i - j >= window) & (j >= sinks))
            for h in range(Hq):
                kv = h // group
                k = K[:, kv].reshape(-1, case["k_dim"])[j]
                v = V[:, kv].reshape(-1, case["v_dim"])[j]
                q = s["q"][starts[b] + rows, h].double() * s["scale"]
                if s["k_scale"] is not None:
                    q, v = q * s["k_scale"][kv].double(), v * s["v_scale"][kv].double()
                score = torch.where(hidden, -math.inf, q @ k.T)
                if s["sink_logits"] is not None:
                    score = torch.cat([score, s["sink_logits"][h].double().expand(len(rows), 1)], 1)
                    v = torch.cat([v, torch.zeros(1, v.shape[1], dtype=torch.float64, device="cuda")])
                out[starts[b] + rows, h] = torch.softmax(score, 1) @ v
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    return {"step": _exact_step, "append": _exact_append, "attend": _exact_attend}[case["op"]](case, s)
