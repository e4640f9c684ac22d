"""The paged-cache operators (PageTable.step, append, attend) against the 64-bit oracle.

Tolerances, from the roundings alone.  append: a rotated value is two 32-bit products and a sum of an angle good to 2^-23
turns (a sine or cosine within 2 pi 2^-23 + 2^-23 < 2^-20), then one rounding: |x - ref| <= 2^-20 (|a| + |b|) + half a step
of the stored type (bf16 2^-8 |ref|; E4M3 2^-4 |ref|, or 2^-10 of the scale below its normal range).  attend: the weights are
rounded to bf16 for the product with V (2^-8 of the weighted mean of |v|), the output is rounded to bf16 (2^-8 |ref|), and
scores, exponentials and sums in 32 bits add less than 2^-11 of the weighted mean of |v|: a score of |q||k| scale <= 32 is
off by at most (192 + 4) 2^-24 32 < 2^-11, as much relative to its weight, and only differences of scores count."""
import threading

import numpy as np
import pytest
import torch

from mimo_stream import KVCache, PageTable, Rotary, StepPlan, append, attend
from oracle import attention as oa

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
DIMS = {"64": (64, 64), "128": (128, 128), "192": (192, 128)}


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def f64(t):
    return t.detach().to(torch.float32).cpu().numpy().astype(np.float64)


# ------------------------------------------------------------------ step
def _random_state(rng, B, page, width, spare=5):
    lens = rng.integers(0, width * page + 1, B)
    target = rng.integers(0, width * page + 1, B)
    for b in range(B):                                   # the cases that matter: no change, one token, ended, page borders
        kind = rng.integers(0, 7)
        if kind == 0:
            target[b] = lens[b]
        elif kind == 1:
            target[b] = min(lens[b] + 1, width * page)
        elif kind == 2:
            target[b] = 0
        elif kind == 3:
            lens[b] = lens[b] // page * page
        elif kind == 4:
            target[b] = target[b] // page * page
    most = int(max(sum(oa.pages(n, page) for n in lens), sum(oa.pages(n, page) for n in np.maximum(lens, target))))
    n_pages = most + spare
    order = rng.permutation(n_pages)
    table = np.full((B, width), -7)
    at = 0
    for b in range(B):
        k = oa.pages(int(lens[b]), page)
        table[b, :k] = order[at:at + k]
        at += k
    free = np.full(n_pages, -9)
    free[:n_pages - at] = order[at:]
    return lens, target, table, free, n_pages - at, n_pages


def _page_table(lens, table, free, n_free, n_pages, page):
    pt = PageTable(len(lens), table.shape[1], n_pages, page)
    pt.lens.copy_(i32(lens))
    pt.table.copy_(i32(table))
    pt.free.copy_(i32(free))
    pt.n_free.fill_(n_free)
    return pt


@pytest.mark.parametrize("B,page,width", [(1, 16, 1), (1, 64, 9), (3, 16, 5), (64, 32, 7), (257, 16, 4), (1025, 16, 3), (4096, 128, 2)])
def test_step_matches_oracle(rng, B, page, width):
    lens, target, table, free, n_free, n_pages = _random_state(rng, B, page, width)
    new = int(np.maximum(target - lens, 0).sum())
    for pad in (0, 3):
        pt = _page_table(lens, table, free, n_free, n_pages, page)
        want = oa.step(lens.tolist(), target.tolist(), table, free, n_free, page, new + pad)
        for commit in (False, True):
            plan = pt.step(i32(target), new + pad, commit=commit)
            plan.check()
            for name, got, ref in zip(("starts", "lens", "slots", "positions", "n_free", "table", "free"),
                                      (plan.starts, plan.lens, plan.slots, plan.positions, plan.n_free, pt.table, pt.free), want):
                assert np.array_equal(got.cpu().numpy().reshape(-1), np.asarray(ref).reshape(-1)), (name, commit, pad)
            state = (target, want[4]) if commit else (lens, n_free)
            assert np.array_equal(pt.lens.cpu().numpy(), state[0]) and pt.n_free.item() == state[1]


def test_step_and_its_inverse_restore_the_stack(rng):
    lens, target, table, free, n_free, n_pages = _random_state(rng, 40, 16, 6)
    target = np.maximum(lens, target)
    pt = _page_table(lens, table, free, n_free, n_pages, 16)
    pt.step(i32(target), int((target - lens).sum())).check()
    pt.step(i32(lens), 0).check()
    assert pt.n_free.item() == n_free and np.array_equal(pt.free.cpu().numpy()[:n_free], free[:n_free])
    assert np.array_equal(pt.lens.cpu().numpy(), lens)


@pytest.mark.parametrize("what", ["pages", "long", "negative", "rows", "max_new", "state"])
def test_step_failures_leave_the_state(what):
    pt = PageTable(3, 4, 6, 16)
    pt.step(i32([20, 0, 64]), 84).check()
    before = [t.clone() for t in (pt.lens, pt.n_free, pt.free[:0])]
    target, rows, kw = [20, 0, 64], 64, {}
    if what == "pages":
        target = [20, 1, 64]
    elif what == "long":
        target = [65, 0, 64]
        rows = 100
    elif what == "negative":
        target = [20, -1, 64]
    elif what == "rows":
        target, rows = [30, 0, 64], 9
    elif what == "max_new":
        target, kw = [30, 0, 64], {"max_new": 9}
    else:
        pt.n_free.fill_(7)
        before[1] = pt.n_free.clone()
        target = [30, 0, 64]
    plan = pt.step(i32(target), rows, **kw)
    with pytest.raises(ValueError, match="pages" if what == "pages" else "lengths"):
        plan.check()
    assert torch.equal(pt.lens, before[0]) and torch.equal(pt.n_free, before[1])
    assert plan.starts.abs().sum().item() == 0 and (plan.slots == -1).all() and torch.equal(plan.lens, pt.lens)


def test_step_refuses_more_returned_pages_than_32_bits_hold():
    # lengths that were never written, at the largest table: the pages that ending all requests gives back are 2^31 - 4096
    width, page, n_pages = (1 << 19) - 1, 16, 1 << 20
    pt = PageTable(4096, width, n_pages, page)
    pt.lens.fill_(width * page)
    plan = pt.step(torch.zeros_like(pt.lens), 4)
    with pytest.raises(ValueError, match="lengths"):
        plan.check()
    assert int(pt.n_free.item()) == n_pages and bool((pt.lens == width * page).all()) and (plan.slots == -1).all()
    assert torch.equal(pt.free, torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device="cuda"))


# ------------------------------------------------------------------ append
def _scales(rng, heads):
    return torch.from_numpy((2.0 ** rng.uniform(-6, -3, heads)).astype(np.float32)).cuda()


@pytest.mark.parametrize("dims", list(DIMS))
@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("N,Hq,Hkv,rot,page", [(1, 4, 2, 16, 16), (7, 5, 1, 64, 32), (65, 3, 3, 32, 16), (33, 12, 2, 0, 64)])
def test_append_matches_oracle(rng, dims, dtype, N, Hq, Hkv, rot, page):
    Dk, Dv = DIMS[dims]
    theta = 10000.0
    n_pages = N // page + 3
    rows = torch.from_numpy(rng.standard_normal((N, Hq * Dk + Hkv * (Dk + Dv))).astype(np.float32) * 2).to(torch.bfloat16).cuda()
    q = rows[:, :Hq * Dk].unflatten(1, (Hq, Dk))
    k = rows[:, Hq * Dk:(Hq + Hkv) * Dk].unflatten(1, (Hkv, Dk))
    v = rows[:, (Hq + Hkv) * Dk:].unflatten(1, (Hkv, Dv))
    slots = rng.permutation(n_pages * page)[:N]
    slots[rng.random(N) < 0.1] = -1
    positions = rng.integers(0, 1 << 20, N)
    positions[0] = 0
    scales = (_scales(rng, Hkv), _scales(rng, Hkv)) if dtype == E4M3 else (None, None)
    cache = KVCache(n_pages, page, Hkv, Dk, Dv, dtype, *scales)
    cache.k.view(torch.uint8).fill_(1)
    cache.v.view(torch.uint8).fill_(1)
    untouched = cache.k.clone(), cache.v.clone()
    plan = StepPlan(slots=i32(slots), positions=i32(positions), status=torch.zeros(1, dtype=torch.int32, device="cuda"))
    got = append(cache, plan, k, v, q=q, rotary=Rotary(rot, theta) if rot else None)
    plan.check()

    def close(x, ref, slack, half, floor):
        assert (np.abs(x - ref) <= 2.0 ** -20 * slack + half * np.abs(ref) + floor).all()

    def turned(x):
        return oa.rotate(f64(x), positions, rot, theta) if rot else f64(x)

    def slack(x):                                        # |a| + |b| of each rotated pair
        m = np.abs(f64(x))
        if rot:
            h = rot // 2
            m[..., :h] = m[..., h:rot] = m[..., :h] + m[..., h:rot]
        return m
    close(f64(got), turned(q), slack(q), 2.0 ** -8, 0.0)
    keep = slots >= 0
    for pages, before, x, ref, size, scale in ((cache.k, untouched[0], k, turned(k), slack(k), scales[0]),
                                               (cache.v, untouched[1], v, f64(v), np.abs(f64(v)), scales[1])):
        flat = f64(pages).transpose(0, 2, 1, 3).reshape(n_pages * page, Hkv, -1)
        old = f64(before).transpose(0, 2, 1, 3).reshape(n_pages * page, Hkv, -1)
        s = 1.0 if scale is None else f64(scale)[None, :, None]
        ref, size = ref / s, size / s
        if dtype == E4M3:
            ref = np.clip(ref, -448, 448)
        close(flat[slots[keep]], ref[keep], size[keep], 2.0 ** (-4 if dtype == E4M3 else -8), 2.0 ** -10 if dtype == E4M3 else 0.0)
        rest = np.setdiff1d(np.arange(n_pages * page), slots[keep])
        assert np.array_equal(flat[rest], old[rest])
    if dtype == torch.bfloat16:                          # what is not rotated is copied bit for bit
        assert np.array_equal(f64(cache.v).transpose(0, 2, 1, 3).reshape(n_pages * page, Hkv, -1)[slots[keep]], f64(v)[keep])
    assert torch.equal(got[..., rot:], q[..., rot:])


def test_append_special_values():
    """NaN stays NaN and infinities saturate in E4M3; both pass through bf16."""
    x = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device="cuda")
    x[0, 0, :4] = torch.tensor([float("nan"), float("inf"), -float("inf"), 1e30])
    plan = StepPlan(slots=i32([3]), positions=i32([9]))
    for dtype, scale in ((torch.bfloat16, None), (E4M3, 0.5)):
        c = KVCache(1, 16, 1, 64, 64, dtype, scale, scale)
        append(c, plan, x, x)
        for t in (c.k, c.v):
            g = t.float()[0, 0, 3, :4]
            assert torch.isnan(g[0])
            assert g[1:].tolist() == ([448.0, -448.0, 448.0] if dtype == E4M3 else x[0, 0, 1:4].float().tolist())


def test_append_reports_a_slot_past_the_cache():
    c = KVCache(1, 16, 1, 64, 64)
    x = torch.ones(2, 1, 64, dtype=torch.bfloat16, device="cuda")
    plan = StepPlan(slots=i32([16, 2]), positions=i32([0, 1]), status=torch.zeros(1, dtype=torch.int32, device="cuda"))
    append(c, plan, x, x)
    with pytest.raises(ValueError, match="slot"):
        plan.check()
    assert c.k.float().sum().item() == 64 and (c.k[0, 0, 2] == 1).all()


# ------------------------------------------------------------------ attend
def _attend_case(rng, lens, new, Hq, Hkv, Dk, Dv, page, dtype=torch.bfloat16, window=0, sinks=0, logits=False, pad=0, fill=1e4,
                 gain=1.0, spare=2):
    """Random requests with `new` tokens of their `lens`; cache rows past every length hold `fill`."""
    B, width = len(lens), max(1, max(oa.pages(n, page) for n in lens)) + 1
    count = [oa.pages(n, page) for n in lens]
    n_pages = sum(count) + spare
    order = rng.permutation(n_pages)
    table = np.full((B, width), 1 << 30)                 # entries past a request's pages are never read
    at = 0
    for b in range(B):
        table[b, :count[b]] = order[at:at + count[b]]
        at += count[b]
    scales = (_scales(rng, Hkv), _scales(rng, Hkv)) if dtype == E4M3 else (None, None)

    def pages(dim, scale):
        x = torch.from_numpy(rng.standard_normal((n_pages, Hkv, page, dim)).astype(np.float32)).cuda()
        if scale is not None:
            x = (x / scale[:, None, None]).clamp(-448, 448)
        live = torch.zeros(n_pages, page, dtype=torch.bool, device="cuda")
        for b in range(B):
            for j in range(count[b]):
                live[table[b, j], :max(0, min(page, lens[b] - j * page))] = True
        return torch.where(live[:, None, :, None], x, torch.full_like(x, fill)).to(dtype)
    cache = KVCache.of(pages(Dk, scales[0]), pages(Dv, scales[1]), *scales)
    starts = np.concatenate([[0], np.cumsum(new)])
    N = int(starts[-1]) + pad
    q = (torch.from_numpy(rng.standard_normal((N, Hq, Dk)).astype(np.float32)) * gain).to(torch.bfloat16).cuda()
    sink = torch.from_numpy(rng.standard_normal(Hq).astype(np.float32)).cuda() if logits else None
    plan = StepPlan(starts=i32(starts), lens=i32(lens), table=i32(table), max_new=int(max(new)),
                    status=torch.zeros(1, dtype=torch.int32, device="cuda"))
    return q, cache, plan, dict(window=window, sink_tokens=sinks, sink_logits=sink)


def _oracle(q, cache, plan, kw, scale=None):
    k, v = f64(cache.k), f64(cache.v)
    if cache.k_scale is not None:
        k, v = k * f64(cache.k_scale)[:, None, None], v * f64(cache.v_scale)[:, None, None]
    logits = kw.get("sink_logits")
    return oa.attend(f64(q), k, v, plan.starts.cpu().numpy(), plan.lens.cpu().numpy(), plan.table.cpu().numpy(),
                     cache.k_dim ** -0.5 if scale is None else scale, kw.get("window", 0), kw.get("sink_tokens", 0),
                     None if logits is None else f64(logits))


def _check(q, cache, plan, kw, scale=None):
    out = torch.full((q.shape[0], q.shape[1], cache.v_dim), float("nan"), dtype=torch.bfloat16, device="cuda")
    got = attend(q, cache, plan, scale=scale, out=out, **kw)
    assert got is out
    plan.check()
    ref, size = _oracle(q, cache, plan, kw, scale)
    x = f64(out)
    assert np.isfinite(x).all() == np.isfinite(ref).all()
    off = np.abs(x - ref) - (2.0 ** -8 * np.abs(ref) + (2.0 ** -8 + 2.0 ** -11) * size)
    assert not (off > 0).any(), f"worst {off.max():.3e} at {np.unravel_index(off.argmax(), off.shape)}"
    return out


def _tight(q, cache, plan, kw, scale=None):
    """As _check, for calls of few rows, whose weights keep 16 bits of their own (rounded rests included, off by 2^-17): no
    term for weights rounded to bf16, their rest is within what 2^-11 leaves over."""
    out = attend(q, cache, plan, scale=scale, **kw)
    plan.check()
    ref, size = _oracle(q, cache, plan, kw, scale)
    tol = 2.0 ** -8 * np.abs(ref) + 2.0 ** -11 * size
    off = np.abs(f64(out) - ref) - tol
    assert not (off > 0).any(), f"worst {off.max():.3e} at {np.unravel_index(off.argmax(), off.shape)}"
    return ref, tol


RAGGED = ([1, 15, 16, 17, 63, 64, 65, 130, 300], [1] * 9)


@pytest.mark.parametrize("dims", list(DIMS))
@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("heads", [(1, 1), (4, 4), (6, 2), (20, 1), (10, 2), (33, 1)])
def test_attend_decode(rng, dims, dtype, heads):
    _check(*_attend_case(rng, *RAGGED, *heads, *DIMS[dims], 16, dtype=dtype))


@pytest.mark.parametrize("dims", list(DIMS))
@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("lens,new,heads", [(*RAGGED, (6, 2)), (*RAGGED, (32, 1)), ([3000, 7, 20000], [1, 1, 1], (8, 2)), ([900, 77], [4, 2], (8, 1))])
def test_attend_few_rows_keep_their_weights(rng, dims, dtype, lens, new, heads):
    _tight(*_attend_case(rng, lens, new, *heads, *DIMS[dims], 16, dtype=dtype, logits=True))


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("length", [33, 300, 5000])
@pytest.mark.parametrize("window", [0, 200])
def test_attend_few_rows_at_the_worst_rounding(rng, dtype, length, window):
    """Weights of 1 and, for two of three keys, just below 0.5 + 2^-9, which bf16 rounds to 0.5, on values that cancel: weights
    rounded once (worked out here) miss the tolerance."""
    q, cache, plan, kw = _attend_case(rng, [length], [1], 4, 2, 64, 64, 16, dtype=dtype, window=window)
    down = np.arange(length) % 3 != 0
    want = np.log(0.5 + 2.0 ** -9 * 0.97)                # the score of those keys, in 8 dimensions of what the cache can hold
    k = np.zeros((length, 64), np.float64)
    scale = 1.0 if dtype == torch.bfloat16 else 2.0 ** -8
    rest = want / scale
    for d in range(8):
        piece = torch.tensor(rest, dtype=torch.float32).to(dtype).float().item()
        k[down, d] = piece
        rest -= piece
    v = rng.choice([0.5, 0.75, 1.0, 1.5, -0.5, -1.25], (1, 64)) * np.where(down, -1.0, 1.0)[:, None]
    table = plan.table.cpu().numpy()[0]
    for j in range(length):
        cache.k[table[j // 16], :, j % 16] = torch.from_numpy(k[j]).to(dtype).cuda()
        cache.v[table[j // 16], :, j % 16] = torch.from_numpy(v[j]).to(dtype).cuda()
    if dtype == E4M3:
        cache.k_scale.fill_(scale)
        cache.v_scale.fill_(1.0)
    q.zero_()
    q[:, :, :8] = 1.0
    ref, tol = _tight(q, cache, plan, kw, scale=1.0)
    seen = np.arange(length) >= (length - window if window else 0)
    w = np.exp(scale * k.sum(1)) * seen
    once = torch.from_numpy(w).to(torch.bfloat16).double().numpy()
    assert np.allclose((w @ v) / w.sum(), ref[0])
    assert (np.abs((once @ v) / w.sum() - ref[0, 0]) > tol[0, 0]).all()


@pytest.mark.parametrize("page", [16, 32, 64, 128, 1024])
@pytest.mark.parametrize("lens,new", [([5], [5]), ([64], [64]), ([200], [130]), ([129, 1, 77, 256], [129, 1, 3, 255]),
                                      ([40, 300, 9], [0, 65, 0]), ([1, 1, 1], [1, 1, 1])])
def test_attend_chunks(rng, page, lens, new):
    _check(*_attend_case(rng, lens, new, 6, 2, 128, 128, page, pad=3))


@pytest.mark.parametrize("dims", list(DIMS))
@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("heads", [(3, 1), (20, 1), (10, 2), (4, 4), (40, 1), (160, 1)])
def test_attend_mixed_batch(rng, dims, dtype, heads):
    _check(*_attend_case(rng, [150, 33, 200, 70, 1], [150, 1, 41, 5, 1], *heads, *DIMS[dims], 32, dtype=dtype, logits=True))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 0), (16, 4), (64, 3), (100, 40), (128, 200), (1000, 5), (0, 5)])
@pytest.mark.parametrize("lens,new", [([300, 90, 17], [1, 1, 1]), ([300, 90, 17], [170, 90, 2])])
@pytest.mark.parametrize("logits", [False, True])
def test_attend_window_and_sinks(rng, window, sinks, lens, new, logits):
    _check(*_attend_case(rng, lens, new, 8, 2, 192, 128, 16, window=window, sinks=sinks, logits=logits))


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("lens,new,heads", [([5000], [1], (16, 1)), ([3000, 7, 20000], [1, 1, 1], (8, 2)), ([4100], [100], (4, 2)),
                                            ([9000, 100], [3, 60], (16, 2))])
def test_attend_long_contexts(rng, lens, new, heads, dtype):
    """A long axis split over many blocks and joined again."""
    _check(*_attend_case(rng, lens, new, *heads, 128, 128, 64, dtype=dtype, gain=2.0))


@pytest.mark.parametrize("new", [[150], [200], [304], [420], [130, 60], [7, 150, 1]])
def test_attend_tiles_that_fill_the_card_in_part(rng, new):
    # a tile a token: these counts are split into one or two rounds of blocks, some requests' shorter tiles into fewer parts
    _check(*_attend_case(rng, [2600 + 13 * i for i in range(len(new))], new, 128, 1, 64, 64, 64))


def test_attend_large_scores(rng):
    """Scores far apart (one key takes all the weight) and far from 0, and a scale of the caller's."""
    q, cache, plan, kw = _attend_case(rng, [100, 400], [3, 100], 4, 2, 64, 64, 16)
    for scale in (4.0, -1.0, 0.0):
        _check(q, cache, plan, kw, scale=scale)


@pytest.mark.parametrize("heads", [(16, 1), (2, 2)])
@pytest.mark.parametrize("new", [[1, 1, 1], [200, 30, 5]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_attend_never_looks_at_masked_values(rng, heads, new, dtype):
    """NaN and infinities in rows past the end, before the window and (for earlier tokens of a chunk) in later tokens."""
    lens = [210, 30, 70]
    bad = float("nan") if dtype == E4M3 else float("inf")
    for window, sinks in ((0, 0), (20, 0), (20, 3)):
        q, cache, plan, kw = _attend_case(rng, lens, new, *heads, 128, 128, 16, dtype=dtype, window=window, sinks=sinks, fill=float("nan"))
        table = plan.table.cpu().numpy()
        for b, n in enumerate(lens):                     # keys that no row of the request sees
            first = n - new[b]
            for j in range(sinks, max(sinks, first - window + 1) if window else sinks):
                cache.k[table[b, j // 16], :, j % 16] = bad
                cache.v[table[b, j // 16], :, j % 16] = float("nan")
        _check(q, cache, plan, kw)
        b = 0                                            # the last token's value: only the last row of the request sees it
        cache.v[table[b, (lens[b] - 1) // 16], :, (lens[b] - 1) % 16] = float("nan")
        out = attend(q, cache, plan, **kw)
        rows = out[:new[0]].float()
        assert torch.isnan(rows[-1]).all() and torch.isfinite(rows[:-1]).all() and torch.isfinite(out[new[0]:].float()).all()
        ref, size = _oracle(q, cache, plan, kw)
        x, ref, size = f64(out)[:new[0] - 1], ref[:new[0] - 1], size[:new[0] - 1]
        assert (np.abs(x - ref) <= 2.0 ** -8 * np.abs(ref) + (2.0 ** -8 + 2.0 ** -11) * size).all()


@pytest.mark.parametrize("lens,new,heads", [([3000], [4], (4, 1)), ([5000, 90], [40, 90], (2, 1)), ([400], [300], (6, 2))])
@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_attend_keeps_one_rows_nan_from_the_others(rng, lens, new, heads, dtype):
    """A chunk's last token holds NaN in K or V, over contexts that are split and that are not: only its own row turns NaN."""
    for what in ("k", "v"):
        q, cache, plan, kw = _attend_case(rng, lens, new, *heads, 128, 128, 16, dtype=dtype)
        table = plan.table.cpu().numpy()
        want, size = _oracle(q, cache, plan, kw)
        getattr(cache, what)[table[0, (lens[0] - 1) // 16], :, (lens[0] - 1) % 16] = float("nan")
        out = f64(attend(q, cache, plan, **kw))
        last = new[0] - 1
        assert np.isnan(out[last]).all()
        rest = np.arange(len(out)) != last
        assert (np.abs(out - want) <= 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 2.0 ** -11) * size)[rest].all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("heads,new,window", [((32, 1), 4, 0), ((64, 2), 7, 0), ((40, 1), 3, 0), ((130, 1), 2, 0), ((32, 1), 4, 20),
                                              ((16, 1), 3, 20), ((8, 1), 5, 20), ((16, 1), 3, 64), ((48, 3), 11, 33)])
@pytest.mark.parametrize("length", [50, 301, 3000])
def test_attend_nan_beside_a_wave_of_one_token(rng, heads, new, window, length, dtype):
    """Waves whose rows are one token's, in a tile of several tokens: a NaN that another token of the tile sees (the last
    one's own value; with a window the oldest key of the first one too) stays with the tokens that see it."""
    last = np.arange(new) == new - 1
    places = [(length - 1, last)] + ([(length - new - window + 1, np.arange(new) == 0)] if window and length - new >= window else [])
    for key, sees in places:
        q, cache, plan, kw = _attend_case(rng, [length], [new], *heads, 64, 64, 16, dtype=dtype, window=window)
        want, size = _oracle(q, cache, plan, kw)
        table = plan.table.cpu().numpy()
        cache.v[table[0, key // 16], :, key % 16] = float("nan")
        out = f64(attend(q, cache, plan, **kw))
        assert np.isnan(out[sees]).all()
        assert (np.abs(out - want) <= 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 2.0 ** -11) * size)[~sees].all()


@pytest.mark.parametrize("new,heads", [([60, 2], (4, 2)), ([1, 1], (4, 2)), ([4, 2], (8, 2)), ([1, 1], (130, 1))])
@pytest.mark.parametrize("key", [3, 295])
def test_attend_non_finite_values_that_rows_see(rng, new, heads, key):
    """An infinity in V reaches every row that weighs it, with its sign, wherever it lies; a NaN in one request's q stays in
    that request."""
    q, cache, plan, kw = _attend_case(rng, [300, 40], new, *heads, 64, 64, 16)
    table = plan.table.cpu().numpy()
    G, n = heads[0] // heads[1], new[0]
    cache.v[table[0, key // 16], 0, key % 16, 7] = float("inf")
    cache.v[table[0, key // 16], 0, key % 16, 9] = -float("inf")
    q[n] = float("nan")
    out = attend(q, cache, plan, **kw).float()
    sees = torch.arange(300 - n, 300, device="cuda") >= key
    assert (out[:n][sees][:, :G, 7] == float("inf")).all() and (out[:n][sees][:, :G, 9] == -float("inf")).all()
    assert torch.isnan(out[n]).all()
    out[:n, :G, 7] = torch.where(sees[:, None], 0.0, out[:n, :G, 7])
    out[:n, :G, 9] = torch.where(sees[:, None], 0.0, out[:n, :G, 9])
    assert torch.isfinite(out[:n]).all() and torch.isfinite(out[n + 1:]).all()


@pytest.mark.parametrize("max_new", [None, 1, 64])
def test_attend_does_not_depend_on_max_new(rng, max_new):
    q, cache, plan, kw = _attend_case(rng, [300, 40, 9], [50, 1, 9], 6, 2, 128, 128, 16)
    plan.max_new = max_new
    _check(q, cache, plan, kw)


@pytest.mark.parametrize("B,most", [(65, 1), (300, 1), (130, 40)])
def test_attend_many_requests(rng, B, most):
    """More requests than lanes, some of them idle, in one call."""
    new = rng.integers(0, most + 1, B)
    lens = new + rng.integers(0, 200, B)
    new[lens == 0] = 0
    _check(*_attend_case(rng, lens.tolist(), new.tolist(), 4, 2, 64, 64, 32, window=70, sinks=3))


def test_attend_and_append_past_32_bit_offsets(rng):
    """Pages whose bytes lie past 2^32 in the cache."""
    pages, page, heads, dim = 70000, 32, 8, 128            # 4.3 GiB of K and of V
    cache = KVCache.of(*(torch.empty(pages, heads, page, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2)))
    small = KVCache(4, page, heads, dim, dim)
    high = [69999, 66000, 69998, 65999]
    N = 100
    x = torch.from_numpy(rng.standard_normal((N, 16 + 2 * heads, dim)).astype(np.float32)).to(torch.bfloat16).cuda()
    outs = []
    for c, ids in ((cache, high), (small, [0, 1, 2, 3])):
        pos = np.arange(N)
        plan = StepPlan(starts=i32([0, N]), lens=i32([N]), table=i32([ids]), positions=i32(pos),
                        slots=i32(np.asarray(ids)[pos // page] * page + pos % page), status=torch.zeros(1, dtype=torch.int32, device="cuda"))
        q = append(c, plan, x[:, 16:16 + heads], x[:, 16 + heads:], q=x[:, :16], rotary=Rotary(128))
        outs.append(attend(q, c, plan))
        plan.check()
    assert torch.equal(*outs)
    assert torch.equal(cache.k[high[1]], small.k[1]) and torch.equal(cache.v[high[2]], small.v[2])


@pytest.mark.parametrize("N", [33, 1])
@pytest.mark.parametrize("length", [300_000_000, (1 << 31) - (1 << 16)])
def test_attend_longest_requests(rng, length, N):
    """Contexts past 2^28 keys, whose table names the same 16 pages again and again: 33 rows (wide tiles) and one (narrow).
    With scale 0 every visible key weighs 1, and V is a whole number from -2 to 2 that changes from one sixteenth of the
    context to the next, so a part's sums (2^22 keys, below 2^24) are exact.  What is left is the join's 512 products and
    sums (2 x 512 x 2^-24 of the mean of |v|), its division, and the output's rounding (2^-8 |ref|)."""
    page, dim = 1024, 64
    width = (length + page - 1) // page
    ids = (np.arange(width, dtype=np.int64) * 16 // width).astype(np.int32)
    values = rng.integers(-2, 3, (16, dim))
    v = torch.from_numpy(values.astype(np.float32)).to(torch.bfloat16).cuda()[:, None, None, :].expand(16, 1, page, dim).contiguous()
    cache = KVCache.of(torch.ones_like(v), v)
    q = torch.ones(N, 1, dim, dtype=torch.bfloat16, device="cuda")
    plan = StepPlan(starts=i32([0, N]), lens=i32([length]), table=torch.from_numpy(ids).cuda()[None], max_new=N,
                    status=torch.zeros(1, dtype=torch.int32, device="cuda"))
    out = f64(attend(q, cache, plan, scale=0.0))[:, 0]
    plan.check()
    for i in range(N):
        keys = length - N + i + 1                        # keys that row i sees
        count = np.bincount(ids[:keys // page], minlength=16) * page
        count[ids[min(keys // page, width - 1)]] += keys % page
        assert count.sum() == keys
        ref, size = count @ values / keys, count @ np.abs(values) / keys
        assert (np.abs(out[i] - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -13 * size).all()


def test_a_failed_step_writes_nothing(rng):
    pt, cache = PageTable(2, 4, 3, 16), KVCache(3, 16, 1, 64, 64)
    x = torch.ones(40, 3, 64, dtype=torch.bfloat16, device="cuda")
    plan = pt.step(i32([33, 7]), 40)                       # four pages of three
    q = append(cache, plan, x[:, 1:2], x[:, 2:], q=x[:, :1])
    out = attend(q, cache, plan)
    assert (out == 0).all() and (cache.k == 0).all() and (cache.v == 0).all()
    with pytest.raises(ValueError, match="pages"):
        plan.check()
    assert pt.lens.tolist() == [0, 0] and pt.n_free.item() == 3


def test_attend_malformed_starts_stay_in_range(rng):
    """starts that run backwards, past the rows or over one another: no fault, and other calls are as before."""
    q, cache, plan, kw = _attend_case(rng, [40, 90, 20], [3, 33, 1], 4, 2, 64, 64, 16)
    want = attend(q, cache, plan)
    good = plan.starts.clone()
    for bad in ([5, 3, 40, 2], [0, 37, 0, 37], [-9, 1 << 30, -5, 7], [40, 40, 40, 40], [2 ** 31 - 1] * 4, [-2 ** 31] * 4):
        plan.starts.copy_(i32(bad))
        for max_new in (1, 33):
            plan.max_new = max_new
            attend(q, cache, plan)
    torch.cuda.synchronize()
    plan.starts.copy_(good)
    plan.max_new = 33
    assert torch.equal(attend(q, cache, plan), want)


@pytest.mark.parametrize("heads", [(4, 2), (64, 2)])
@pytest.mark.parametrize("long", [90, 5000])
def test_attend_refuses_malformed_starts(rng, heads, long):
    """starts that run backwards, before the rows or past them (a plan of more rows than q has): every row is 0, the status
    says so, and a request in order beside the bad one is not answered in part; also where rows were split a call before."""
    q, cache, plan, kw = _attend_case(rng, [40, long, 20], [3, 33, 1], *heads, 64, 64, 16)
    good = plan.starts.clone()
    for max_new in (1, 33):
        plan.max_new = max_new
        want = attend(q, cache, plan)
        plan.check()
        for bad in ([5, 3, 40, 2], [0, 37, 0, 37], [-9, 1 << 30, -5, 7], [40, 40, 40, 40], [2 ** 31 - 1] * 4, [-2 ** 31] * 4,
                    [0, 3, 36, 38], [-1, 3, 36, 37], [0, 3, 2, 37], [3, 2, 36, 37]):
            plan.starts.copy_(i32(bad))
            out = torch.full_like(want, float("nan"))
            attend(q, cache, plan, out=out)
            with pytest.raises(ValueError, match="starts"):
                plan.check()
            assert (out == 0).all(), bad
            plan.status.zero_()
        plan.starts.copy_(good)
        assert torch.equal(attend(q, cache, plan), want)
        plan.check()
    out = torch.full_like(want[:-1], float("nan"))         # q without the plan's last row
    attend(q[:-1], cache, plan, out=out)
    with pytest.raises(ValueError, match="starts"):
        plan.check()
    assert (out == 0).all()


@pytest.mark.parametrize("max_new", [1, 1 << 20])
def test_attend_refuses_starts_that_ask_for_millions_of_tiles(max_new):
    N, B = 1 << 20, 256
    cache = KVCache(2, 16, 1, 64, 64)
    plan = StepPlan(starts=i32([0, N] * (B // 2) + [0]), lens=i32([N] * B), table=torch.zeros(B, N // 16, dtype=torch.int32, device="cuda"),
                    max_new=max_new, status=torch.zeros(1, dtype=torch.int32, device="cuda"))
    out = torch.full((N, 1, 64), float("nan"), dtype=torch.bfloat16, device="cuda")
    attend(torch.zeros_like(out), cache, plan, out=out)
    with pytest.raises(ValueError, match="starts"):
        plan.check()
    assert (out == 0).all()


def test_attend_scores_of_minus_infinity(rng):
    """Visible keys of score -inf weigh nothing; a row of only such keys, with no sink, is 0."""
    q, cache, plan, kw = _attend_case(rng, [40], [3], 2, 1, 64, 64, 16)
    q[:, :, 0] = 1.0
    cache.k[..., 0] = -float("inf")
    out = attend(q, cache, plan, **kw)
    assert (out == 0).all()
    table = plan.table.cpu().numpy()
    cache.k[table[0, 1], 0, 5, 0] = 0.0                  # key 21 alone keeps a finite score
    out = attend(q, cache, plan, **kw)
    assert torch.equal(out, cache.v[table[0, 1], 0, 5].expand_as(out))


def test_attend_sink_logits_of_infinity(rng):
    q, cache, plan, kw = _attend_case(rng, [40, 100], [1, 80], 2, 1, 64, 64, 16)
    plain = attend(q, cache, plan)
    none = attend(q, cache, plan, sink_logits=torch.full((2,), -float("inf"), device="cuda"))
    assert torch.equal(plain, none)
    _check(q, cache, plan, dict(sink_logits=torch.tensor([60.0, -60.0], device="cuda")))


def test_attend_reports_bad_pages_and_lengths(rng):
    q, cache, plan, kw = _attend_case(rng, [40, 20], [1, 1], 2, 1, 64, 64, 16, pad=1)
    good = attend(q, cache, plan)
    plan.check()
    assert (good[2] == 0).all()
    plan.table[0, 1] = cache.n_pages
    out = attend(q, cache, plan)
    with pytest.raises(ValueError, match="page"):
        plan.check()
    assert torch.equal(out[1], good[1])
    plan.table[0, 1] = -1
    plan.status.zero_()
    attend(q, cache, plan)
    with pytest.raises(ValueError, match="page"):
        plan.check()
    plan.table[0, 1] = 0
    for bad in (0, -5, plan.table.shape[1] * 16 + 1, 2 ** 31 - 1):
        plan.status.zero_()
        plan.lens[0] = bad
        out = attend(q, cache, plan)
        with pytest.raises(ValueError, match="length"):
            plan.check()
        assert (out[0] == 0).all() and torch.equal(out[1], good[1])


def test_attend_strided_rows_and_zero_tokens(rng):
    q, cache, plan, kw = _attend_case(rng, [40, 90], [1, 33], 4, 2, 128, 128, 32)
    want = attend(q, cache, plan)
    wide = torch.zeros(q.shape[0], 3 * 4 * 128 + 8, dtype=torch.bfloat16, device="cuda")
    wide[:, 512:1024] = q.flatten(1)
    assert torch.equal(attend(wide[:, 512:1024].unflatten(1, (4, 128)), cache, plan), want)
    odd = torch.zeros(q.shape[0], 515, dtype=torch.bfloat16, device="cuda")    # rows the kernel cannot read: copied first
    odd[:, 3:] = q.flatten(1)
    assert torch.equal(attend(odd[:, 3:].unflatten(1, (4, 128)), cache, plan), want)
    assert attend(q[:0], cache, plan).shape == (0, 4, 128)
    with pytest.raises(ValueError):
        attend(q[:, :3], cache, plan)
    with pytest.raises(ValueError):
        attend(q, cache, plan, sink_logits=torch.zeros(3, device="cuda"))
    with pytest.raises(ValueError):
        attend(q, cache, plan, out=torch.zeros(2, 4, 128, dtype=torch.bfloat16, device="cuda"))


def test_attend_repeats_bit_for_bit(rng):
    q, cache, plan, kw = _attend_case(rng, [7000, 100, 2500], [1, 70, 1], 20, 2, 192, 128, 64, logits=True)
    first = attend(q, cache, plan, **kw)
    for _ in range(3):
        assert torch.equal(attend(q, cache, plan, **kw), first)


# ------------------------------------------------------------------ the operators together
def _run_steps(rng, chunks, Hq=8, Hkv=2, dims=(192, 128), window=0, sinks=0, n_pages=40, page=16):
    """Requests grow by the given chunks, step by step; returns each step's outputs and the q, k, v they came from."""
    B = len(chunks[0])
    Dk, Dv = dims
    pt = PageTable(B, 16, n_pages, page)
    cache = KVCache(n_pages, page, Hkv, Dk, Dv)
    rotary = Rotary(64)
    total = np.zeros(B, np.int64)
    steps = []
    for new in chunks:
        total = total + new
        N = int(sum(new))
        rows = torch.from_numpy(rng.standard_normal((N, Hq * Dk + Hkv * (Dk + Dv))).astype(np.float32)).to(torch.bfloat16).cuda()
        q = rows[:, :Hq * Dk].unflatten(1, (Hq, Dk))
        k = rows[:, Hq * Dk:(Hq + Hkv) * Dk].unflatten(1, (Hkv, Dk))
        v = rows[:, (Hq + Hkv) * Dk:].unflatten(1, (Hkv, Dv))
        plan = pt.step(i32(total), N, max_new=int(max(new)))
        qr = append(cache, plan, k, v, q=q, rotary=rotary)
        out = attend(qr, cache, plan, window=window, sink_tokens=sinks)
        plan.check()
        steps.append((new, q, k, v, qr, out))
    return steps


@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 2)])
def test_step_append_attend_like_one_sequence(rng, window, sinks):
    """Prompt chunks, single tokens and idle requests over many steps equal attention over each whole sequence at once."""
    chunks = [[50, 0, 3], [1, 1, 1], [20, 70, 1], [0, 1, 1], [1, 1, 40]]
    steps = _run_steps(rng, chunks, window=window, sinks=sinks)
    B, page = 3, 256
    for b in range(B):
        ks, vs, qs, outs = [], [], [], []
        for new, q, k, v, qr, out in steps:
            s = slice(sum(new[:b]), sum(new[:b + 1]))
            ks.append(f64(k[s])), vs.append(f64(v[s])), qs.append(f64(qr[s])), outs.append(f64(out[s]))
        k, v, q, got = (np.concatenate(x) for x in (ks, vs, qs, outs))
        L = len(k)
        k = oa.rotate(k, np.arange(L), 64, 10000.0).astype(np.float32)
        k = f64(torch.from_numpy(k).to(torch.bfloat16))
        kp, vp = np.zeros((1, 2, page, 192)), np.zeros((1, 2, page, 128))
        kp[0, :, :L], vp[0, :, :L] = k.transpose(1, 0, 2), v.transpose(1, 0, 2)
        ref, size = oa.attend(q, kp, vp, [0, L], [L], [[0]], 192 ** -0.5, window, sinks)
        # the oracle's k may round the other way at a tie of the 32-bit rotation: a step of 2^-7 on a key of one position
        # moves a score by under 2^-7 |q_i k_i| scale < 2^-7, a weight by as much
        assert (np.abs(got - ref) <= 2.0 ** -8 * np.abs(ref) + (2.0 ** -7 + 2.0 ** -8 + 2.0 ** -11) * size).all()


def test_a_step_of_other_pages_is_refused():
    pt, cache = PageTable(1, 4, 8, 64), KVCache(8, 16, 1, 64, 64)
    plan = pt.step(i32([20]), 20)
    x = torch.ones(20, 1, 64, dtype=torch.bfloat16, device="cuda")
    for call in (lambda: append(cache, plan, x, x), lambda: attend(x, cache, plan)):
        with pytest.raises(ValueError, match="pages of 64 tokens"):
            call()
    assert (cache.k == 0).all() and plan.page_size == 64


def test_rollback_gives_the_same_step_again(rng):
    """Tokens taken back (a rejected speculation) leave no trace: the same step again gives the same bits."""
    pt, cache, rotary = PageTable(2, 8, 9, 16), KVCache(9, 16, 1, 128, 128), Rotary(128)
    x = torch.from_numpy(rng.standard_normal((40, 3, 128)).astype(np.float32)).to(torch.bfloat16).cuda()

    def go(target, rows):
        plan = pt.step(i32(target), rows)
        q = append(cache, plan, x[:rows, 2:], x[:rows, 1:2], q=x[:rows, :1], rotary=rotary)
        out = attend(q, cache, plan)
        plan.check()
        return out
    go([14, 26], 40)
    first = go([22, 32], 14)
    pt.step(i32([14, 26]), 0).check()
    assert torch.equal(go([22, 32], 14), first)


def test_a_growing_step_can_be_dropped_after_its_append(rng):
    """New tokens written in a step that is not committed and gives no pages back change nothing for the requests as they
    were; the step made again, with other tokens, is as if the first had not been."""
    x = torch.from_numpy(rng.standard_normal((60, 3, 128)).astype(np.float32)).to(torch.bfloat16).cuda()
    y = torch.from_numpy(rng.standard_normal((60, 3, 128)).astype(np.float32)).to(torch.bfloat16).cuda()

    def go(pt, cache, target, rows, x, commit=True):
        plan = pt.step(i32(target), rows, commit=commit)
        q = append(cache, plan, x[:rows, 2:], x[:rows, 1:2], q=x[:rows, :1], rotary=Rotary(128))
        out = attend(q, cache, plan)
        plan.check()
        return out
    outs = []
    for drop in (False, True):
        pt, cache = PageTable(3, 8, 9, 16), KVCache(9, 16, 1, 128, 128)
        go(pt, cache, [14, 26, 0], 40, x)
        if drop:
            go(pt, cache, [34, 27, 5], 26, y, commit=False)
        outs.append([go(pt, cache, [15, 27, 1], 3, x, commit=False), go(pt, cache, [14, 50, 3], 27, x), pt.n_free.clone()])
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_graph_replays_follow_the_state(rng):
    """A captured decode step (step, append, attend) replayed as the lengths grow equals the eager steps; two captured graphs
    and eager work in between do not disturb each other."""
    def make():
        pt, cache = PageTable(3, 80, 200, 16), KVCache(200, 16, 2, 128, 128)
        plan = pt.step(i32([1000, 5, 0]), 1005)
        x = torch.from_numpy(np.random.default_rng(3).standard_normal((1005, 2, 128)).astype(np.float32)).to(torch.bfloat16).cuda()
        append(cache, plan, x, x)
        return pt, cache
    rotary = Rotary(64)
    one = i32([1, 1, 1])

    def step(pt, cache, x):
        target = pt.lens + one
        plan = pt.step(target, 3, max_new=1)
        q = append(cache, plan, x[:, 8:10], x[:, 10:12], q=x[:, :8], rotary=rotary)
        return attend(q, cache, plan), plan
    xs = [torch.from_numpy(rng.standard_normal((3, 12, 128)).astype(np.float32)).to(torch.bfloat16).cuda() for _ in range(6)]
    state = make()
    want = []
    for x in xs:
        out, plan = step(*state, x)
        plan.check()
        want.append(out.clone())
    graphs = []
    for _ in range(2):
        pt, cache = make()
        x = xs[0].clone()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out, plan = step(pt, cache, x)
        graphs.append((g, x, out, plan, pt, cache))          # a graph does not keep the state that it works on
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i, x in enumerate(xs):
        for (g, gx, *_), s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                gx.copy_(x)
                g.replay()
        step(*state, x)                                  # eager work of another state on the default stream
        torch.cuda.synchronize()
        for g, gx, out, plan, *_ in graphs:
            assert plan.status.item() == 0 and torch.equal(out, want[i]), i


def test_on_another_stream(rng):
    q, cache, plan, kw = _attend_case(rng, [3000, 77], [1, 40], 8, 2, 128, 128, 64)
    want = attend(q, cache, plan, **kw)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = attend(q, cache, plan, **kw)
    s.synchronize()
    assert torch.equal(got, want)


def test_threads_on_one_stream(rng):
    """Calls of two threads on one stream, whose rows are split and joined over the stream's one workspace."""
    cases = [_attend_case(rng, [5000, 900], [1, 1], 8, 2, 64, 64, 16), _attend_case(rng, [4000], [90], 4, 2, 128, 128, 64),
             _attend_case(rng, [3000, 7, 2000], [1, 1, 1], 8, 2, 64, 64, 32)]
    want = [attend(q, cache, plan, **kw) for q, cache, plan, kw in cases]
    torch.cuda.synchronize()
    bad = []

    def work(first):
        for i in range(20):
            order = [(first + i + k) % len(cases) for k in range(12)]
            got = [attend(q, cache, plan, **kw) for q, cache, plan, kw in (cases[k] for k in order)]
            bad.extend((first, i, k) for g, k in zip(got, order) if not torch.equal(g, want[k]))
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad[:5]
