"""Operators of the attention half around an 8-bit K/V cache that needs no calibration, as a serving program calls them: the
append that rotates q and k (pairs of either layout, frequencies stretched for long contexts) and quantises K and V as it
writes them, one power of two for each 16 tokens and head; the read that turns cached tokens back into rows; and the
attention of new tokens over that cache.

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
E8M0 = torch.float8_e8m0fnu
E4M3_MAX = 448.0
TOP_SCALE = 246                    # the largest scale byte: 448 * 2^(246 - 127) is finite in bf16
BLOCK = 16                         # tokens that share a scale
GOLDEN = (math.sqrt(5.0) - 1.0) / 2.0

# query heads, K/V heads, key and value dimensions
WIDE = (64, 4, 192, 128)           # keys wider than values, 16 query heads on each K/V head
WIDE8 = (64, 8, 192, 128)
EVEN = (32, 8, 128, 128)
SLIM = (20, 4, 64, 64)             # five query heads on each K/V head


def _heads(dims):
    return {"heads": dims[0], "kv_heads": dims[1], "k_dim": dims[2], "v_dim": dims[3]}


def _append(reqs, new, far, dims, rotary, kind="block", interleaved=False, factor=1.0, page=64):
    """new: the fewest and the most tokens that a request brings; far: positions before them, at most; factor: how far the
    context is stretched past the 4096 tokens that the frequencies stem from (1: not at all)."""
    return dict(_heads(dims), op="append", reqs=reqs, new_lo=new[0], new_hi=new[1], far=far, rotary=rotary, kind=kind,
                theta=10000.0 if rotary < dims[2] else 5.0e6, interleaved=interleaved, factor=factor, page=page)


def _read(tokens, dims, kind="block", page=64):
    return dict(_heads(dims), op="read", tokens=tokens, kind=kind, page=page)


def _attend(reqs, ctx, new, dims, chunked=0, page=64, window=0, sinks=0, logits=False):
    return dict(_heads(dims), op="attend", reqs=reqs, ctx_lo=ctx[0], ctx_hi=ctx[1], new_lo=new[0], new_hi=new[1],
                chunked=chunked, page=page, window=window, sinks=sinks, logits=logits)


def listed():
    return [
        # a decode batch: every token joins a block that holds earlier ones, whose scale may grow
        dict(_append(64, (1, 1), 16384, WIDE, 64), name="append8_decode_64"),
        # a prompt's chunk far into a stretched context, pairs side by side
        dict(_append(1, (4096, 4096), 131072, WIDE8, 64, interleaved=True, factor=32.0), name="append8_chunk_4096"),
        # ragged pieces of many prompts, every dimension rotated, small pages
        dict(_append(24, (1, 147), 9000, EVEN, 128, page=16), name="append8_ragged_24"),
        # a decode batch into a bf16 cache, pairs side by side: the call's own latency
        dict(_append(32, (1, 1), 4096, SLIM, 64, kind="bf16", interleaved=True, page=16), name="append_pairs_32"),
        # a prompt's chunk into a bf16 cache, stretched frequencies in the half layout
        dict(_append(1, (2048, 2048), 65536, WIDE, 64, kind="bf16", factor=8.0), name="append_stretched_2048"),
        # a short prompt's keys and values, handed on as rows
        dict(_read(137, WIDE), name="read8_137"),
        # a long context, moved to where a program needs it in bf16
        dict(_read(32768, WIDE), name="read8_32768"),
        # one request deep in a long context: a long axis with few rows
        dict(_attend(1, (32767, 32767), (1, 1), WIDE), name="decode8_1x32k"),
        # a ragged decode batch on a layer that sees everything
        dict(_attend(48, (500, 16384), (1, 1), EVEN), name="decode8_48"),
        # the same on a sliding-window layer: 128 keys, with sink logits
        dict(_attend(128, (90, 12000), (1, 1), WIDE8, window=128, logits=True), name="decode8_window_128"),
        # the third chunk of a long prompt
        dict(_attend(1, (8192, 8192), (4096, 4096), WIDE, chunked=1), name="chunk8_4096_at_8192"),
        # prompt pieces of odd sizes beside decoding requests, small pages, five query heads on a K/V head
        dict(_attend(24, (0, 5000), (37, 901), SLIM, chunked=9, page=16, sinks=5, window=1111, logits=True), name="mixed8_24"),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    part = rng.random()
    page = rng.choice((16, 32, 64, 128))
    kv = rng.choice((1, 2, 4, 8))
    group = rng.choice([g for g in (1, 2, 3, 4, 5, 7, 8, 12, 16) if g * kv <= 64])
    dims = (kv * group, kv) + rng.choice(((64, 64), (128, 128), (192, 128)))
    if part < 0.4:
        reqs = spread(1, 128)
        hi = spread(1, 4096 // reqs)
        kind = rng.choice(("block", "block", "block", "bf16", "e4m3"))
        interleaved = rng.random() < 0.5
        factor = rng.choice((1.0, round(rng.uniform(1.5, 40.0), 2)))
        if kind != "block" and not interleaved and factor == 1.0:
            interleaved = True                             # else it would not be of this file
        return _append(reqs, (rng.randint(1, hi), hi), spread(64, 131072), dims, rng.choice((32, 64, dims[2])), kind=kind,
                       interleaved=interleaved, factor=factor, page=page)
    if part < 0.55:
        return _read(spread(1, 32768), dims, kind=rng.choice(("block", "block", "bf16", "e4m3")), page=page)
    window = rng.choice((0, 0, 128, spread(1, 4096)))
    sinks = rng.choice((0, 4, rng.randint(1, 70))) if window else 0
    logits = rng.random() < 0.4
    if part < 0.8:
        reqs = spread(1, 128)
        hi = spread(16, 20000 if reqs <= 24 else 5000)
        return _attend(reqs, (rng.randint(0, hi), hi), (1, 1), dims, page=page, window=window, sinks=sinks, logits=logits)
    reqs = spread(1, 24)
    hi = spread(2, 4096 // max(1, reqs // 2))
    return _attend(reqs, (0, spread(1, 8192)), (rng.randint(1, hi), hi), dims, chunked=rng.randint(1, max(1, reqs // 2)),
                   page=page, window=window, sinks=sinks, logits=logits)


# ------------------------------------------------------------------ request lengths
def _between(lo, hi, i):
    """The i-th of evenly spread whole numbers of lo .. hi."""
    return lo + int((hi - lo + 1) * math.modf((i + 1) * GOLDEN)[0])


def _lengths(case):
    """Every request's length before the new tokens, and how many it brings."""
    if case["op"] == "append":
        return ([_between(0, case["far"], i) for i in range(case["reqs"])],
                [_between(case["new_lo"], case["new_hi"], 3 * i + 1) for i in range(case["reqs"])])
    return ([_between(case["ctx_lo"], case["ctx_hi"], i) for i in range(case["reqs"])],
            [_between(case["new_lo"], case["new_hi"], 3 * i + 1) if i < case["chunked"] else 1 for i in range(case["reqs"])])


def _pages(n, page):
    return (n + page - 1) // page


# ------------------------------------------------------------------ inputs (torch alone, from the seed)
def _generator(seed, part):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + part) % (1 << 62))


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _normal(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(torch.bfloat16)


def _loud(heads, dim):
    """Some dimensions of some heads are larger than the rest, as keys and values have them."""
    x = torch.ones(heads, dim, device="cuda")
    x[::2, 5::37] = 9.0
    x[1::3] *= 0.02
    return x


def _per_head(heads, base):
    return base * (1.0 + 0.25 * torch.arange(heads, dtype=torch.float32, device="cuda"))


def _filled(case, n_pages, dim, base, g):
    """Page contents of a case's kind with its scales (bytes, fp32 of each head, or None), made of random values."""
    heads, page, kind = case["kv_heads"], case["page"], case["kind"]
    loud = _loud(heads, dim)[:, None, :]
    x = torch.empty(n_pages, heads, page, dim, dtype=torch.bfloat16 if kind == "bf16" else E4M3, device="cuda")
    scale = None
    if kind == "e4m3":
        scale = _per_head(heads, base)
    elif kind == "block":
        scale = torch.empty(n_pages, heads, page // BLOCK, dtype=torch.uint8, device="cuda")
    for at in range(0, n_pages, 512):
        y = torch.randn(x[at:at + 512].shape, generator=g, device="cuda") * loud
        if kind == "e4m3":
            y = (y / scale[:, None, None]).clamp(-E4M3_MAX, E4M3_MAX)
        elif kind == "block":
            # tokens of a block are alike in size, blocks differ
            y = y.unflatten(2, (-1, BLOCK)) * torch.exp2(torch.randint(-3, 4, (y.shape[0], heads, page // BLOCK, 1, 1), generator=g, device="cuda").float())
            most = y.abs().amax((-1, -2))
            byte = torch.ceil(torch.log2(most / E4M3_MAX)) + 127.0
            scale[at:at + 512] = byte.to(torch.uint8)
            y = (y * torch.exp2(127.0 - byte)[..., None, None]).clamp(-E4M3_MAX, E4M3_MAX).flatten(2, 3)
        x[at:at + 512] = y.to(x.dtype)
    return x, scale


def _append_inputs(case, seed):
    g = _generator(seed, 1)
    Hq, Hkv, Dk, Dv, page = case["heads"], case["kv_heads"], case["k_dim"], case["v_dim"], case["page"]
    before, new = _lengths(case)
    N = sum(new)
    # the pages that hold the new tokens; the earlier ones of a request play no part
    first = [n // page for n in before]
    count = [_pages(a + b, page) - f for a, b, f in zip(before, new, first)]
    n_pages = sum(count) + 1
    order = torch.randperm(n_pages, generator=g, device="cuda")
    base = np.concatenate([[0], np.cumsum(count)])
    positions = torch.tensor(np.concatenate([np.arange(a, a + b) for a, b in zip(before, new)]), device="cuda")
    place = torch.tensor(np.concatenate([np.arange(a, a + b) // page - f + p for a, b, f, p in zip(before, new, first, base)]), device="cuda")
    slots = order[place] * page + positions % page
    # q, k and v are views of one projection's rows, as a fused projection leaves them
    rows = _normal(g, N, Hq * Dk + Hkv * (Dk + Dv), scale=1.5)
    k = rows[:, Hq * Dk:(Hq + Hkv) * Dk].unflatten(1, (Hkv, Dk))
    v = rows[:, (Hq + Hkv) * Dk:].unflatten(1, (Hkv, Dv))
    k.copy_(k * _loud(Hkv, Dk))
    v.copy_(v * _loud(Hkv, Dv))
    k_pages, k_scale = _filled(case, n_pages, Dk, 1 / 16, g)
    v_pages, v_scale = _filled(case, n_pages, Dv, 1 / 16, g)
    return {"q": rows[:, :Hq * Dk].unflatten(1, (Hq, Dk)), "k": k, "v": v, "slots": slots.to(torch.int32),
            "positions": positions.to(torch.int32), "k_pages": k_pages, "v_pages": v_pages, "k_scale": k_scale, "v_scale": v_scale}


def _read_inputs(case, seed):
    g = _generator(seed, 2)
    N, page = case["tokens"], case["page"]
    n_pages = _pages(N, page) + 2
    order = torch.randperm(n_pages, generator=g, device="cuda")
    at = torch.arange(N, device="cuda")
    k_pages, k_scale = _filled(case, n_pages, case["k_dim"], 1 / 64, g)
    v_pages, v_scale = _filled(case, n_pages, case["v_dim"], 1 / 80, g)
    return {"slots": (order[at // page] * page + at % page).to(torch.int32), "k_pages": k_pages, "v_pages": v_pages,
            "k_scale": k_scale, "v_scale": v_scale}


def _attend_inputs(case, seed):
    g = _generator(seed, 3)
    page, Hq = case["page"], case["heads"]
    before, new = _lengths(case)
    lens = [a + b for a, b in zip(before, new)]
    count = [_pages(n, page) for n in lens]
    n_pages = sum(count) + 2
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), max(count), dtype=torch.int32, device="cuda")
    table[torch.arange(max(count), device="cuda")[None, :] < _int32(count)[:, None]] = order[:sum(count)]
    kind = dict(case, kind="block")
    k_pages, k_scale = _filled(kind, n_pages, case["k_dim"], 0.0, g)
    v_pages, v_scale = _filled(kind, n_pages, case["v_dim"], 0.0, g)
    starts = np.concatenate([[0], np.cumsum(new)]).tolist()
    return {"q": _normal(g, starts[-1], Hq, case["k_dim"], scale=0.5), "k_pages": k_pages, "v_pages": v_pages, "k_scale": k_scale,
            "v_scale": v_scale, "table": table, "starts": _int32(starts), "lens": _int32(lens), "max_new": max(new),
            "scale": 1.0 / math.sqrt(case["k_dim"]),
            "sink_logits": torch.randn(Hq, generator=g, device="cuda") if case["logits"] else None}


INPUTS = {"append": _append_inputs, "read": _read_inputs, "attend": _attend_inputs}


# the context length that frequencies stem from, and between how many turns over it they are stretched in part
ORIGINAL, FEW_TURNS, MANY_TURNS = 4096, 1.0, 32.0


def _magnitude(case):
    return 0.1 * math.log(case["factor"]) + 1.0


def _frequencies(case):
    """theta ** (-2 i / dim); under a factor, pairs of few turns over the original length turn that much slower, pairs of many
    as before, and those between them in proportion to the pair's number."""
    dim, theta, factor = case["rotary"], case["theta"], case["factor"]
    i = torch.arange(dim // 2, dtype=torch.float64, device="cuda")
    freq = torch.pow(torch.tensor(theta, dtype=torch.float64, device="cuda"), -2.0 * i / dim)
    lo, hi = (dim * math.log(ORIGINAL / (2.0 * math.pi * turns)) / (2.0 * math.log(theta)) for turns in (MANY_TURNS, FEW_TURNS))
    lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), dim // 2 - 1)
    slow = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
    return freq * (1.0 - slow) + freq / factor * slow


def prepare(case, seed):
    s = dict(INPUTS[case["op"]](case, seed), case=case)
    if not own:
        if case["op"] == "append":
            s["freq"] = _frequencies(case)
        return s
    if PKG not in sys.path:
        sys.path.insert(0, PKG)
    from mimo_stream import attention
    cache = attention.KVCache.of(s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"])
    if case["op"] == "append":
        dim, theta, factor = case["rotary"], case["theta"], case["factor"]
        freq = attention.stretched(dim, theta, factor, ORIGINAL, FEW_TURNS, MANY_TURNS) if factor != 1.0 else None
        rotary = attention.Rotary(dim, theta, interleaved=case["interleaved"], frequencies=freq, magnitude=_magnitude(case))
        return {"op": "append", "cache": cache, "plan": attention.StepPlan(slots=s["slots"], positions=s["positions"]),
                "q": s["q"], "k": s["k"], "v": s["v"], "rotary": rotary}
    if case["op"] == "read":
        return {"op": "read", "cache": cache, "slots": s["slots"]}
    plan = attention.StepPlan(starts=s["starts"], lens=s["lens"], table=s["table"], max_new=s["max_new"])
    return {"op": "attend", "q": s["q"], "cache": cache, "plan": plan, "scale": s["scale"], "window": case["window"],
            "sinks": case["sinks"], "sink_logits": s["sink_logits"]}


# ------------------------------------------------------------------ one pass
def _held(k, v, k_scale, v_scale):
    """What a cache holds, as values: codes, and the powers of two of the scale bytes."""
    if k_scale is None or k_scale.dtype != torch.uint8:
        return k, v
    return k, v, k_scale.view(E8M0), v_scale.view(E8M0)


def run(state):
    if own:
        from mimo_stream import attention
        cache = state["cache"]
        if state["op"] == "append":
            q = attention.append(cache, state["plan"], state["k"], state["v"], q=state["q"], rotary=state["rotary"])
            return (q,) + _held(cache.k, cache.v, cache.k_scale, cache.v_scale)
        if state["op"] == "read":
            return attention.read(cache, state["slots"])
        return attention.attend(state["q"], cache, state["plan"], scale=state["scale"], window=state["window"],
                                sink_tokens=state["sinks"], sink_logits=state["sink_logits"])
    return {"append": _plain_append, "read": _plain_read, "attend": _plain_attend}[state["case"]["op"]](state)


# ------------------------------------------------------------------ the plain forms
def _rotated(x, cos, sin, case):
    dim = case["rotary"]
    turned, rest = x[..., :dim], x[..., dim:]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if case["interleaved"] else turned.chunk(2, -1)
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if case["interleaved"] else torch.cat([a, b], -1)
    return torch.cat([turned, rest], -1)


def _two_to(power):
    """2.0 ** power in 32 bits, by its bits; 2 ** -126 for less."""
    return ((power.int().clamp(-126, 127) + 127) << 23).view(torch.float32)


def _write_block(x, slots, pages, scale, case):
    """x [N, heads, dim] to its slots; a run of rows is those of one block of 16 slots."""
    page = case["page"]
    block = torch.div(slots, BLOCK, rounding_mode="floor")
    of, run = torch.unique_consecutive(block, return_inverse=True)         # the runs' blocks, every row's run
    runs = of.numel()
    most = torch.zeros(runs, x.shape[1], device="cuda").index_reduce_(0, run, x.abs().amax(-1), "amax")
    fraction, exponent = torch.frexp(most / E4M3_MAX)                      # most = fraction 2^exponent 448, 0.5 <= fraction < 1
    need = torch.where(fraction == 0.5, exponent - 1, exponent) + 127
    need = need.clamp(1, TOP_SCALE)
    anew = torch.zeros(runs, dtype=torch.bool, device="cuda")
    anew[run[slots % BLOCK == 0]] = True                                   # a block's first token begins it anew
    at, part = of // (page // BLOCK), of % (page // BLOCK)
    had = scale[at, :, part].int()
    has = torch.where(anew[:, None], need, torch.maximum(had, need))
    rows = part[:, None] * BLOCK + torch.arange(BLOCK, device="cuda")
    codes = pages.view(torch.uint8)
    old = pages[at[:, None], :, rows]                                      # [runs, 16, heads, dim]
    kept = (old.float() * _two_to(had - has)[:, None, :, None]).to(E4M3)
    kept = torch.where(anew[:, None, None, None], old.view(torch.uint8), kept.view(torch.uint8))
    codes[at[:, None], :, rows] = kept
    scale[at, :, part] = has.to(torch.uint8)
    y = (x * _two_to(127 - has)[run][..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3)
    codes[slots // page, :, slots % page] = y.view(torch.uint8)


def _plain_append(s):
    case = s["case"]
    angle = s["positions"].double()[:, None] * s["freq"]
    m = _magnitude(case)
    cos, sin = (torch.cos(angle) * m).float()[:, None, :], (torch.sin(angle) * m).float()[:, None, :]
    q, k = _rotated(s["q"].float(), cos, sin, case).to(torch.bfloat16), _rotated(s["k"].float(), cos, sin, case)
    slots, page = s["slots"].long(), case["page"]
    for x, pages, scale in ((k, s["k_pages"], s["k_scale"]), (s["v"].float(), s["v_pages"], s["v_scale"])):
        if case["kind"] == "block":
            _write_block(x, slots, pages, scale, case)
        elif case["kind"] == "e4m3":
            pages.view(torch.uint8)[slots // page, :, slots % page] = (x / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3).view(torch.uint8)
        else:
            pages[slots // page, :, slots % page] = x.to(torch.bfloat16)
    return (q,) + _held(s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"])


def _rows_of(pages, scale, at, row):
    """Values [*at, heads, dim] in 32 bits of the cache's tokens."""
    x = pages.view(torch.uint8)[at, :, row].view(E4M3).float() if pages.dtype == E4M3 else pages[at, :, row].float()
    if scale is None:
        return x
    if scale.dtype != torch.uint8:
        return x * scale[:, None]
    return x * _two_to(scale[at, :, row // BLOCK].int() - 127)[..., None]


def _plain_read(s):
    page, slots = s["case"]["page"], s["slots"].long()
    return tuple(_rows_of(p, c, slots // page, slots % page).to(torch.bfloat16)
                 for p, c in ((s["k_pages"], s["k_scale"]), (s["v_pages"], s["v_scale"])))


def _plain_attend(s):
    """All requests at once, padded to the most new tokens and the most keys that one of them looks at."""
    case = s["case"]
    Hq, Hkv, window, sinks, page = case["heads"], case["kv_heads"], case["window"], case["sinks"], case["page"]
    G, B, n_most = Hq // Hkv, case["reqs"], s["max_new"]
    starts, lens = s["starts"].long(), s["lens"].long()
    new = starts[1:] - starts[:-1]
    first = lens - new                                                     # position of each request's first new token
    low = (first - window + 1).clamp(min=0) if window else torch.zeros_like(first)
    ahead = min(sinks, page * s["table"].shape[1])                         # room for the first tokens, before the window's
    span = int((lens - low).max())
    column = torch.arange(ahead + span, device="cuda")
    key = torch.where(column < ahead, column, low[:, None] + column - ahead)             # [B, keys]
    there = torch.where(column < ahead, key < low[:, None], key < lens[:, None])
    safe = torch.where(there, key, 0)
    at = torch.gather(s["table"].long(), 1, safe // page)
    K = _rows_of(s["k_pages"], s["k_scale"], at, safe % page)              # [B, keys, Hkv, Dk]
    V = _rows_of(s["v_pages"], s["v_scale"], at, safe % page)
    i = torch.arange(n_most, device="cuda")
    row = torch.where(i < new[:, None], starts[:-1, None] + i, 0)          # [B, n_most]
    q = s["q"].float()[row].unflatten(2, (Hkv, G))                         # [B, n_most, Hkv, G, Dk]
    position = (first[:, None] + i)[:, :, None]
    seen = there[:, None, :] & (key[:, None, :] <= position)               # [B, n_most, keys]
    if window:
        seen &= (position - key[:, None, :] < window) | (key[:, None, :] < sinks)
    out = torch.empty(B, n_most, Hkv, G, case["v_dim"], device="cuda")
    for h in range(Hkv):                                                   # a K/V head at a time, for the memory of its scores
        Qh = q[:, :, h].transpose(1, 2).reshape(B, G * n_most, -1)
        score = torch.matmul(Qh, K[:, :, h].transpose(1, 2).contiguous()).unflatten(1, (G, n_most)) * s["scale"]
        score.masked_fill_(~seen[:, None], -math.inf)
        top = score.amax(-1, keepdim=True)
        if s["sink_logits"] is not None:
            sink = s["sink_logits"].view(Hkv, G)[h][None, :, None, None]
            top = torch.maximum(top, sink)
        weight = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
        total = weight.sum(-1, keepdim=True)
        if s["sink_logits"] is not None:
            total = total + torch.exp(sink - top)
        y = torch.matmul(weight.flatten(1, 2), V[:, :, h].contiguous()).unflatten(1, (G, n_most)) / total
        out[:, :, h] = y.transpose(1, 2)
    return out[i < new[:, None]].flatten(1, 2).to(torch.bfloat16)


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
    Hq, Hkv, Dk, Dv, page = case["heads"], case["kv_heads"], case["k_dim"], case["v_dim"], case["page"]
    if case["op"] == "attend":
        pairs = keys = 0
        for before, n in zip(*_lengths(case)):
            p, k = _visible(before, n, case["window"], case["sinks"])
            pairs, keys = pairs + p, keys + k
        tokens = sum(_lengths(case)[1])
        return {"bytes": keys * Hkv * (Dk + Dv + 2 / BLOCK) + 2 * tokens * Hq * (Dk + Dv), "flops": 2 * pairs * Hq * (Dk + Dv)}
    size = {"bf16": 2, "e4m3": 1, "block": 1 + 2 / BLOCK / (Dk + Dv)}[case["kind"]]
    N = case["tokens"] if case["op"] == "read" else sum(_lengths(case)[1])
    if case["op"] == "read":
        return {"bytes": N * (Hkv * (Dk + Dv) * (2 + size) + 4), "flops": 0}
    return {"bytes": N * (4 * Hq * Dk + Hkv * (Dk + Dv) * (2 + size) + 8), "flops": 3 * N * (Hq + Hkv) * case["rotary"]}


# ------------------------------------------------------------------ 64 bits
def _exact_append(case, s):
    dim, page, kind = case["rotary"], case["page"], case["kind"]
    half = dim // 2
    pairs = np.arange(half)
    freq = case["theta"] ** (-2.0 * pairs / dim)
    if case["factor"] != 1.0:
        edge = [dim / 2 * math.log(ORIGINAL / (2 * math.pi * t), case["theta"]) for t in (MANY_TURNS, FEW_TURNS)]
        lo, hi = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), half - 1)
        share = np.clip((pairs - lo) / max(hi - lo, 0.001), 0, 1)
        freq = freq * (1 - share + share / case["factor"])
    angle = s["positions"].cpu().numpy().astype(np.float64)[:, None] * freq
    turn = torch.tensor(np.exp(1j * angle) * (0.1 * math.log(case["factor"]) + 1), device="cuda")[:, None, :]

    def rotate(x):
        x = x.double()
        at = (slice(0, dim, 2), slice(1, dim, 2)) if case["interleaved"] else (slice(0, half), slice(half, dim))
        z = torch.complex(x[..., at[0]].contiguous(), x[..., at[1]].contiguous()) * turn
        x[..., at[0]], x[..., at[1]] = z.real, z.imag
        return x

    slots = s["slots"].cpu().numpy().astype(np.int64)
    outs = []
    bytes_out = []
    for x, pages, scale in ((rotate(s["k"]), s["k_pages"], s["k_scale"]), (s["v"].double(), s["v_pages"], s["v_scale"])):
        held = pages.double()
        if kind != "block":
            if kind == "e4m3":
                x = (x / scale.double()[:, None]).clamp(-448, 448)
            t = s["slots"].long()
            for h in range(case["kv_heads"]):
                held[t // page, h, t % page] = x[:, h]
            outs.append(held)
            continue
        size = x.abs().amax(-1).cpu().numpy()                              # [N, heads]
        bytes_ = scale.cpu().numpy().astype(np.int64)
        shift = np.zeros(bytes_.shape)                                     # what earlier tokens' codes are divided by, as a power
        edges = np.flatnonzero(np.diff(slots // 16)) + 1
        for rows in np.split(np.arange(len(slots)), edges):
            block = slots[rows[0]] // 16
            at = (block // (page // 16), slice(None), block % (page // 16))
            most = size[rows].max(0)
            power = np.ceil(np.log2(np.maximum(most, 1e-300) / 448)).astype(np.int64)
            power -= (most <= 448 * 2.0 ** (power - 1))
            power += (most > 448 * 2.0 ** power)
            byte = np.clip(power + 127, 1, TOP_SCALE)
            if not (slots[rows] % 16 == 0).any():
                byte = np.maximum(byte, bytes_[at])
                shift[at] = byte - bytes_[at]
            bytes_[at] = byte
        held /= torch.tensor(2.0 ** shift, device="cuda").repeat_interleave(16, 2)[..., None]
        two = torch.tensor(2.0 ** (bytes_ - 127.0), device="cuda")
        t = s["slots"].long()
        for h in range(case["kv_heads"]):
            held[t // page, h, t % page] = (x[:, h] / two[t // page, h, t % page // 16][:, None]).clamp(-448, 448)
        outs.append(held)
        bytes_out.append(two)
    return tuple([rotate(s["q"])] + outs + bytes_out)


def _cached(pages, scale, at):
    """Values [pages, heads, page, dim] of whole pages."""
    x = pages[at].double()
    if scale is None:
        return x
    if scale.dtype != torch.uint8:
        return x * scale.double()[:, None, None]
    powers = torch.tensor([2.0 ** (b - 127) for b in range(256)], dtype=torch.float64, device="cuda")
    return (x.unflatten(2, (-1, 16)) * powers[scale[at].long()][..., None, None]).flatten(2, 3)


def _exact_read(case, s):
    every = torch.arange(s["k_pages"].shape[0], device="cuda")
    slots = s["slots"].long()
    return tuple(_cached(p, c, every).transpose(1, 2).flatten(0, 1)[slots] for p, c in ((s["k_pages"], s["k_scale"]), (s["v_pages"], s["v_scale"])))


def _exact_attend(case, s):
    Hq, window, sinks, page = case["heads"], case["window"], case["sinks"], case["page"]
    group = Hq // case["kv_heads"]
    out = torch.zeros(s["q"].shape[0], Hq, case["v_dim"], dtype=torch.float64, device="cuda")
    starts = s["starts"].tolist()
    for b, length in enumerate(s["lens"].tolist()):
        n = starts[b + 1] - starts[b]
        at = s["table"][b, :_pages(length, page)].long()
        K, V = _cached(s["k_pages"], s["k_scale"], at), _cached(s["v_pages"], s["v_scale"], at)
        for part in range(0, n, 1024):
            rows = torch.arange(part, min(n, part + 1024), device="cuda")
            i = (length - n + rows)[:, None]
            lo = max(0, length - n + part - window + 1) if window else 0
            j = torch.cat([torch.arange(min(lo, sinks), device="cuda"), torch.arange(lo, length, device="cuda")])
            hidden = j > i
            if window:
                hidden = hidden | ((i - j >= window) & (j >= sinks))
            for h in range(Hq):
                k = K[:, h // group].reshape(-1, case["k_dim"])[j]
                v = V[:, h // group].reshape(-1, case["v_dim"])[j]
                score = torch.where(hidden, -math.inf, (s["q"][starts[b] + rows, h].double() * s["scale"]) @ k.T)
                if s["sink_logits"] is not None:
                    score = torch.cat([score, s["sink_logits"][h].double().expand(len(rows), 1)], 1)
                    v = torch.cat([v, torch.zeros(1, v.shape[1], dtype=torch.float64, device="cuda")])
                out[starts[b] + rows, h] = torch.softmax(score, 1) @ v
    return out


def exact(case, seed):
    s = INPUTS[case["op"]](case, seed)
    return {"append": _exact_append, "read": _exact_read, "attend": _exact_attend}[case["op"]](case, s)
