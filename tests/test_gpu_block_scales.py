"""The cache with block scales (append, read, attend) and the rotary forms against the 64-bit oracle.

Tolerances, from the roundings alone.  append: a rotated value is two 32-bit products and a sum of sines and cosines good to
2^-20 times the magnitude: |x - ref| <= 2^-20 m (|a| + |b|) + half a step of the stored type (bf16 2^-8 |ref|; E4M3 2^-4 of the
code, or 2^-10 below its normal range).  A block's byte is exact unless its largest magnitude is within 2^-19 m (|a| + |b|) of
the border between two bytes, where either is right.  What a block held is multiplied by a power of two and rounded: exact
bits, as torch rounds them on the CPU.  read: exact for bf16 and block scales, half a step of bf16 for scales per head.
attend: as for the other caches, on the values that codes and bytes stand for: weights rounded to bf16 (2^-8 of the weighted
mean of |v|; calls of few rows 2^-17), the output to bf16 (2^-8 |ref|), and everything else in 32 bits within 2^-11 of the
weighted mean of |v|, for scores of |q| |k| scale <= 32."""
import numpy as np
import pytest
import torch

from helpers import rand_bf16, to_dev_bf16
from mimo_stream import AttentionLayer, KVCache, PageTable, Rotary, StepPlan, append, attend, read, stretched
from oracle import attention as oa, layer as ol, mxfp4 as oq

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
BF = torch.bfloat16
DIMS = {"64": (64, 64), "128": (128, 128), "192": (192, 128)}


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def f64(t):
    return t.detach().to(torch.float32).cpu().numpy().astype(np.float64)


def word():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


def _empty(n_pages, page, heads, dk, dv):
    return KVCache(n_pages, page, heads, dk, dv, dtype=E4M3, block_scales=True)


def _random_cache(rng, n_pages, page, heads, dk, dv, lo=100, hi=140):
    """Random codes (no NaN) and random bytes."""
    def codes(dim):
        c = rng.integers(0, 127, (n_pages, heads, page, dim)) + 128 * rng.integers(0, 2, (n_pages, heads, page, dim))
        return torch.from_numpy(c.astype(np.uint8)).cuda().view(E4M3)

    def bytes_():
        return torch.from_numpy(rng.integers(lo, hi, (n_pages, heads, page // 16)).astype(np.uint8)).cuda()
    return KVCache.of(codes(dk), codes(dv), bytes_(), bytes_())


def _values(cache):
    """float64 k and v of a cache of any kind."""
    k, v = f64(cache.k), f64(cache.v)
    if cache.block_scales:
        return oa.block_values(k, cache.k_scale.cpu().numpy()), oa.block_values(v, cache.v_scale.cpu().numpy())
    if cache.k_scale is not None:
        return k * f64(cache.k_scale)[:, None, None], v * f64(cache.v_scale)[:, None, None]
    return k, v


def _slots(rng, N, n_pages, page):
    """Rows in runs of one block each: whole blocks, pieces that begin or end anywhere, single rows, rows out of order in a
    block, and rows that are left out."""
    blocks = list(rng.permutation(n_pages * page // 16))
    out = []
    while len(out) < N:
        kind = rng.integers(0, 6)
        if kind == 0:
            out += [-1] * int(rng.integers(1, 4))
            continue
        b = int(blocks.pop())
        a, z = (0, 16) if kind == 1 else sorted(rng.choice(17, 2, replace=False))
        rows = [16 * b + i for i in range(a, z)]
        if kind == 2:
            rows = rows[:1]
        if kind == 3:
            rng.shuffle(rows)
        out += rows
    return np.array(out[:N])


FORMS = {"half": (False, None, 1.0), "side": (True, None, 1.0), "half stretched": (False, 8.0, 1.2), "side stretched": (True, 32.0, 1.35)}


def _rotary(rot, form):
    side, factor, magnitude = FORMS[form]
    freq = 10000.0 ** (-2.0 * np.arange(rot // 2) / rot) if factor is None else oa.stretched(rot, 10000.0, factor, 4096, 1.0, 32.0)
    rotary = Rotary(rot, 10000.0, interleaved=side, frequencies=None if factor is None else stretched(rot, 10000.0, factor, 4096), magnitude=magnitude)
    return rotary, lambda x, at: oa.turn(x, at, freq, side, magnitude), lambda x: _slack(x, rot, side, magnitude)


def _slack(x, rot, side, magnitude):
    """m (|a| + |b|) of each rotated pair, |x| of the rest."""
    m = np.abs(x)
    h = rot // 2
    at = (slice(0, rot, 2), slice(1, rot, 2)) if side else (slice(0, h), slice(h, rot))
    both = magnitude * (m[..., at[0]] + m[..., at[1]])
    m[..., at[0]], m[..., at[1]] = both, both
    return m


def _check_blocks(pages, scale, before, byte_before, ref, slack, slots, page):
    """One of a cache's two sides after an append of ref [N, heads, D] that is known to within 2^-20 slack."""
    N, heads, _ = ref.shape
    got, byte = pages.cpu(), scale.cpu().numpy().astype(np.int64)
    values = f64(pages)
    untouched = np.ones(values.shape[0] * page // 16, bool)
    n = 0
    while n < N:
        rows = [n]
        while slots[n] >= 0 and n + 1 < N and slots[n + 1] >= 0 and slots[n + 1] // 16 == slots[n] // 16:
            n += 1
            rows.append(n)
        n += 1
        if slots[rows[0]] < 0:
            continue
        block = slots[rows[0]] // 16
        p, part = block * 16 // page, block % (page // 16)
        untouched[block] = False
        anew = any(slots[r] % 16 == 0 for r in rows)
        others = [16 * part + i for i in range(16) if 16 * block + i not in {int(slots[r]) for r in rows}]
        for h in range(heads):
            x = np.abs(ref[rows, h])
            near = (x + 2.0 ** -20 * slack[rows, h] + 1e-300)[np.isfinite(x)].max(initial=0.0)
            below = (x - 2.0 ** -20 * slack[rows, h])[np.isfinite(x)].max(initial=0.0)
            old = int(byte_before[p, h, part])
            wants = {max(oa.block_byte(v), 0 if anew else old) for v in (max(below, 0.0), near)}
            now = int(byte[p, h, part])
            assert now in wants, (block, h, now, wants)
            two = 2.0 ** (now - 127.0)
            for r in rows:
                want = np.clip(ref[r, h] / two, -448, 448)
                off = np.abs(values[p, h, slots[r] % page] - want) - (2.0 ** -4 * np.abs(want) + 2.0 ** -10 + 2.0 ** -20 * slack[r, h] / two)
                assert not (off > 0).any(), (r, h, off.max())
            kept = before[p, h, others]
            if not anew:
                kept = (kept.float() * 2.0 ** max(old - now, -140)).to(E4M3)
            assert torch.equal(got[p, h, others].view(torch.uint8), kept.view(torch.uint8)), (block, h)
    for block in np.flatnonzero(untouched):
        p, part = block * 16 // page, block % (page // 16)
        assert (byte[p, :, part] == byte_before[p, :, part]).all()
        span = slice(16 * part, 16 * part + 16)
        assert torch.equal(got[p, :, span].view(torch.uint8), before[p, :, span].view(torch.uint8))


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("dims", list(DIMS))
@pytest.mark.parametrize("N,Hq,Hkv,rot,page", [(1, 4, 2, 16, 16), (7, 5, 1, 64, 32), (65, 3, 3, 32, 16), (133, 12, 2, 0, 64), (90, 8, 4, -1, 128)])
def test_append_matches_oracle(rng, dims, form, N, Hq, Hkv, rot, page):
    Dk, Dv = DIMS[dims]
    rot = Dk if rot < 0 else rot
    n_pages = 8 * N // page + 20
    cache = _random_cache(rng, n_pages, page, Hkv, Dk, Dv)
    before = [t.cpu().clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    rows = torch.from_numpy(rng.standard_normal((N, Hq * Dk + Hkv * (Dk + Dv))).astype(np.float32) * 2.0 ** rng.integers(-9, 10, (N, 1))).to(BF).cuda()
    q = rows[:, :Hq * Dk].unflatten(1, (Hq, Dk))
    k = rows[:, Hq * Dk:(Hq + Hkv) * Dk].unflatten(1, (Hkv, Dk))
    v = rows[:, (Hq + Hkv) * Dk:].unflatten(1, (Hkv, Dv))
    slots = _slots(rng, N, n_pages, page)
    positions = rng.integers(0, 1 << 20, N)
    positions[0] = 0
    rotary, turn, slack = _rotary(rot, form) if rot else (None, lambda x, at: x, np.abs)
    plan = StepPlan(slots=i32(slots), positions=i32(positions), status=word())
    got = append(cache, plan, k, v, q=q, rotary=rotary)
    plan.check()
    want, room = turn(f64(q), positions), slack(f64(q))
    assert (np.abs(f64(got) - want) <= 2.0 ** -20 * room + 2.0 ** -8 * np.abs(want)).all()
    assert torch.equal(got[..., rot:], q[..., rot:])
    _check_blocks(cache.k, cache.k_scale, before[0], before[2].numpy().astype(np.int64), turn(f64(k), positions), slack(f64(k)), slots, page)
    _check_blocks(cache.v, cache.v_scale, before[1], before[3].numpy().astype(np.int64), f64(v), np.zeros(v.shape), slots, page)


@pytest.mark.parametrize("form", ["side", "half stretched", "side stretched"])
@pytest.mark.parametrize("dtype", [BF, E4M3])
@pytest.mark.parametrize("dims,rot", [("64", 64), ("128", 32), ("192", 64), ("192", 192), ("64", 16)])
def test_rotary_forms_in_the_other_caches(rng, dims, rot, dtype, form):
    Dk, Dv = DIMS[dims]
    N, Hq, Hkv, page = 37, 6, 2, 16
    k_scale = torch.tensor([0.25, 0.0625], device="cuda") if dtype == E4M3 else None
    cache = KVCache(4, page, Hkv, Dk, Dv, dtype, k_scale, k_scale)
    q, k, v = (torch.from_numpy(rng.standard_normal((N, h, d)).astype(np.float32)).to(BF).cuda() for h, d in ((Hq, Dk), (Hkv, Dk), (Hkv, Dv)))
    slots, positions = rng.permutation(4 * page)[:N], rng.integers(0, 1 << 20, N)
    rotary, turn, slack = _rotary(rot, form)
    plan = StepPlan(slots=i32(slots), positions=i32(positions), status=word())
    got = append(cache, plan, k, v, q=q, rotary=rotary)
    plan.check()
    want = turn(f64(q), positions)
    assert (np.abs(f64(got) - want) <= 2.0 ** -20 * slack(f64(q)) + 2.0 ** -8 * np.abs(want)).all()
    assert torch.equal(got[..., rot:], q[..., rot:])
    ref, room = turn(f64(k), positions), slack(f64(k))
    held = f64(cache.k).transpose(0, 2, 1, 3).reshape(4 * page, Hkv, Dk)[slots]
    if dtype == E4M3:
        s = f64(k_scale)[:, None]
        ref, room = np.clip(ref / s, -448, 448), room / s
        assert (np.abs(held - ref) <= 2.0 ** -20 * room + 2.0 ** -4 * np.abs(ref) + 2.0 ** -10).all()
    else:
        assert (np.abs(held - ref) <= 2.0 ** -20 * room + 2.0 ** -8 * np.abs(ref)).all()


def test_append_without_q_and_of_one_row(rng):
    cache = _empty(2, 32, 3, 192, 128)
    k, v = (torch.from_numpy(rng.standard_normal((1, 3, d)).astype(np.float32)).to(BF).cuda() for d in (192, 128))
    assert append(cache, StepPlan(slots=i32([21]), positions=i32([5])), k, v) is None
    assert append(cache, StepPlan(slots=i32([]), positions=i32([])), k[:0], v[:0], q=k[:0]).shape == (0, 3, 192)
    got = read(cache, i32([21, 20, 22]))
    assert (got[0][0].float() - k[0].float()).abs().max() <= 2.0 ** -4 * k.float().abs().max()
    # the block was not begun by its first slot: its byte of 1.0 stayed, and its other rows are the zeros they were
    assert (cache.k_scale == 127).all() and not got[0][1:].any() and not got[1][1:].any()


def test_append_special_values():
    """NaN stays NaN, infinities and values past 448 * 2^119 saturate and take no part in a scale, small values keep theirs."""
    x = torch.zeros(3, 1, 64, dtype=BF, device="cuda")
    nan, inf = float("nan"), float("inf")
    x[0, 0, :4] = torch.tensor([nan, inf, -inf, 3.0])
    x[1, 0, :3] = torch.tensor([3.3895e38, -3.3895e38, 2.0 ** 120])
    x[2, 0, :3] = torch.tensor([2.0 ** -133, 2.0 ** -126, 0.0])
    cache = _empty(1, 64, 1, 64, 64)
    append(cache, StepPlan(slots=i32([0, 16, 32]), positions=i32([0, 0, 0])), x, x)
    for codes, byte, got in zip((cache.k, cache.v), (cache.k_scale, cache.v_scale), read(cache, i32([0, 16, 32]))):
        assert byte.flatten().tolist() == [oa.block_byte(3.0), 246, 1, 127]
        assert torch.isnan(codes.float()[0, 0, 0, 0]) and codes.float()[0, 0, 0, 1:4].tolist() == [448.0, -448.0, 384.0]
        g = got.float()[:, 0]
        assert torch.isnan(g[0, 0]) and g[0, 3] == 3.0
        assert g[1, 0] == 448 * 2.0 ** 119 and g[1, 1] == -448 * 2.0 ** 119 and g[1, 2] == 2.0 ** 120
        # 2^-133 is 2^-7 of the least scale 2^-126: a code below the normal range; read gives it unless bf16 subnormals are lost
        assert codes.float()[0, 0, 32, 1] == 1.0 and codes.float()[0, 0, 32, 0] == 2.0 ** -7 and g[2, 1] == 2.0 ** -126


def test_append_of_nothing_but_zeros_leaves_room():
    cache = _empty(1, 16, 1, 64, 64)
    x = torch.zeros(2, 1, 64, dtype=BF, device="cuda")
    append(cache, StepPlan(slots=i32([0, 1]), positions=i32([0, 1])), x, x)
    assert cache.k_scale.item() == 1
    append(cache, StepPlan(slots=i32([2]), positions=i32([2])), x[:1] + 5.0, x[:1] - 7.0)
    k, v = read(cache, i32([0, 1, 2]))
    assert not k[:2].any() and not v[:2].any() and (k[2] == 5.0).all() and (v[2] == -7.0).all()


@pytest.mark.parametrize("cuts", [[1] * 100, [7, 1, 1, 16, 30, 2, 43], [99, 1], [16] * 6 + [4]])
def test_a_block_holds_the_same_however_it_was_written(rng, cuts):
    """Token by token or at once: bit for bit, for values whose codes stay in the normal range under any scale they meet."""
    H, Dk, Dv, page = 2, 128, 128, 32

    def rows(d):                                           # |x| from 2^-3 to 2^3: codes of at least 2^-6 under a scale of 2^-5
        x = 2.0 ** rng.uniform(-3, 2.99, (100, H, d)) * rng.choice([-1.0, 1.0], (100, H, d))
        return torch.from_numpy(x.astype(np.float32)).to(BF).cuda()
    k, v = rows(Dk), rows(Dv)

    def held(pieces):
        cache, pt, at = _empty(8, page, H, Dk, Dv), PageTable(1, 4, 8, page), 0
        cache.k_scale.fill_(200)                           # what the pages held before does not matter
        for n in pieces:
            plan = pt.step(i32([at + n]), n)
            append(cache, plan, k[at:at + n], v[at:at + n])
            plan.check()
            at += n
        slots = pt.slots(0, 100)
        return read(cache, slots), [s.view(8, H, 2).transpose(1, 2).flatten(0, 1)[slots.long() // 16] for s in (cache.k_scale, cache.v_scale)]
    (k1, v1), s1 = held([100])
    (k2, v2), s2 = held(cuts)
    assert torch.equal(k1, k2) and torch.equal(v1, v2) and all(torch.equal(a, b) for a, b in zip(s1, s2))


def test_tokens_taken_back_and_written_again(rng):
    """Rejected drafts of large values leave a block's scale where they raised it; what stays keeps its values to the steps of
    that scale, and a block that begins anew has its own."""
    H, Dk, Dv, page = 1, 64, 64, 16
    cache, pt = _empty(4, page, H, Dk, Dv), PageTable(1, 3, 4, page)
    small = torch.from_numpy(rng.standard_normal((40, H, Dk)).astype(np.float32)).to(BF).cuda()
    append(cache, pt.step(i32([20]), 20), small[:20], small[:20])
    first = read(cache, pt.slots(0, 20))
    append(cache, pt.step(i32([36]), 16), small[:16] * 4096, small[:16] * 4096)
    pt.step(i32([20]), 0).check()
    now = read(cache, pt.slots(0, 20))
    top = 2.0 ** (int(cache.k_scale.flatten()[pt.slots(0, 20)[16].item() // 16]) - 127)
    assert torch.equal(now[0][:16], first[0][:16])
    assert (now[0][16:].float() - first[0][16:].float()).abs().max() <= top * 2.0 ** -10
    append(cache, pt.step(i32([16]), 0), small[:0], small[:0])
    plan = pt.step(i32([32]), 16)
    append(cache, plan, small[16:32], small[16:32])
    plan.check()
    again = read(cache, pt.slots(0, 32))
    assert (again[0][16:].float() - small[16:32].float()).abs().max() <= 2.0 ** -4 * 8.0
    assert torch.equal(read(cache, plan.slots)[1], again[1][16:])


def test_append_reports_slots(rng):
    x = torch.ones(3, 1, 64, dtype=BF, device="cuda")
    for slots in ([16, 2, -1], [5, 5, 6]):
        cache = _empty(1, 16, 1, 64, 64)
        plan = StepPlan(slots=i32(slots), positions=i32([0, 1, 2]), status=word())
        append(cache, plan, x, x)
        with pytest.raises(ValueError, match="slot"):
            plan.check()
        k = read(cache, i32([2, 5, 6]))[0]
        assert (k[0] == (1.0 if slots[0] == 16 else 0.0)).all()
    for slots in ([5, 20, 5], [5, 20, 6], [5, -1, 6], [5] + list(range(32, 47)) + [7]):   # a block's rows that others part
        cache = _empty(4, 16, 1, 64, 64)
        z = torch.ones(len(slots), 1, 64, dtype=BF, device="cuda")
        plan = StepPlan(slots=i32(slots), positions=i32([0] * len(slots)), status=word())
        append(cache, plan, z, z)
        with pytest.raises(ValueError, match="slot"):
            plan.check()
        others = [s for s in slots if s >= 16]
        assert not others or (read(cache, i32(others))[0] == 1.0).all()
        assert not cache.k[3].float().any()
    cache = _empty(2, 16, 1, 64, 64)
    y = torch.ones(20, 1, 64, dtype=BF, device="cuda")
    plan = StepPlan(slots=i32([3] * 20), positions=i32([0] * 20), status=word())
    append(cache, plan, y, y)
    with pytest.raises(ValueError, match="slot"):
        plan.check()
    assert not cache.k[1].float().any()


def test_append_far_into_a_large_cache(rng):
    """Slots whose bytes are past 2^31: 40000 pages of 64 tokens, 8 heads of 128."""
    cache = KVCache(40000, 64, 8, 128, 128, dtype=E4M3, block_scales=True)
    slots = np.array([64 * 39999 + i for i in range(14, 35)] + [64 * 36000 + 63])
    k, v = (torch.from_numpy(rng.standard_normal((22, 8, 128)).astype(np.float32)).to(BF).cuda() for _ in range(2))
    plan = StepPlan(slots=i32(slots), positions=i32(np.arange(22)), status=word())
    append(cache, plan, k, v)
    plan.check()
    got = read(cache, plan.slots)
    for x, y in zip(got, (k, v)):
        assert (x.float() - y.float()).abs().max() <= 2.0 ** -4 * y.float().abs().max()
    table, lens = i32([[36000, 39999]]), i32([64 + 35])
    cache.k[36000].view(torch.uint8).zero_()
    q = torch.from_numpy(rng.standard_normal((1, 8, 128)).astype(np.float32)).to(BF).cuda()
    out = attend(q, cache, StepPlan(starts=i32([0, 1]), lens=lens, table=table, max_new=1), window=21)
    kk, vv = (f64(x[:21]) for x in got)
    s = np.einsum("hd,jhd->hj", f64(q)[0], kk) * 128 ** -0.5
    w = np.exp(s - s.max(1, keepdims=True))
    w /= w.sum(1, keepdims=True)
    ref, size = np.einsum("hj,jhd->hd", w, vv), np.einsum("hj,jhd->hd", w, np.abs(vv))
    assert (np.abs(f64(out)[0] - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -11 * size).all()


# ------------------------------------------------------------------ read
@pytest.mark.parametrize("kind", ["bf16", "heads", "blocks"])
@pytest.mark.parametrize("dims", list(DIMS))
@pytest.mark.parametrize("N,heads,page", [(1, 1, 16), (77, 3, 16), (500, 2, 128), (5000, 4, 64)])
def test_read_matches_oracle(rng, dims, kind, N, heads, page):
    Dk, Dv = DIMS[dims]
    n_pages = 7
    cache = _random_cache(rng, n_pages, page, heads, Dk, Dv)
    if kind == "bf16":
        cache = KVCache.of(*(torch.from_numpy(rng.standard_normal((n_pages, heads, page, d)).astype(np.float32)).to(BF).cuda() for d in (Dk, Dv)))
    elif kind == "heads":
        scale = [torch.from_numpy(rng.uniform(0.01, 3.0, heads).astype(np.float32)).cuda() for _ in range(2)]
        cache = KVCache.of(cache.k, cache.v, *scale)
    slots = rng.integers(-1, n_pages * page, N)            # some twice, some left out
    status = word()
    got = read(cache, i32(slots), status=status)
    assert status.item() == 0
    for x, values in zip(got, _values(cache)):
        ref = values.transpose(0, 2, 1, 3).reshape(n_pages * page, heads, -1)[slots]
        ref[slots < 0] = 0.0
        assert (np.abs(f64(x) - ref) <= (2.0 ** -8 + 2.0 ** -24 if kind == "heads" else 0.0) * np.abs(ref)).all()


def test_read_into_given_rows_and_past_the_cache(rng):
    cache = _random_cache(rng, 3, 16, 2, 64, 64)
    k, v = torch.full((4, 2, 64), 9.0, dtype=BF, device="cuda"), torch.full((4, 2, 64), 9.0, dtype=BF, device="cuda")
    status = word()
    got = read(cache, i32([3, 48, -1, 47]), out=(k, v), status=status)
    assert got[0] is k and got[1] is v and status.item() != 0
    assert not k[1:3].any() and not v[1:3].any()
    alone = read(cache, i32([3, 47]))
    assert torch.equal(alone[0], k[[0, 3]]) and torch.equal(alone[1], v[[0, 3]])
    assert read(cache, i32([]))[0].shape == (0, 2, 64)
    with pytest.raises(ValueError, match="slots"):
        read(cache, torch.zeros(2, device="cuda"))
    with pytest.raises(ValueError, match="out"):
        read(cache, i32([1]), out=(k, v))
    with pytest.raises(ValueError, match="overlap"):
        read(cache, i32([1] * 4), out=(k, k))


def test_read_special_values():
    cache = _empty(1, 16, 1, 64, 64)
    cache.k.view(torch.uint8)[0, 0, 0, :4] = torch.tensor([0x7F, 0xFF, 0x80, 0x7E], dtype=torch.uint8)
    cache.k_scale.fill_(130)
    k = read(cache, i32([0]))[0][0, 0].float()
    assert torch.isnan(k[:2]).all() and k[2] == 0.0 and torch.signbit(k[2]) and k[3] == 448.0 * 8


# ------------------------------------------------------------------ attend
def _attend_case(rng, lens, new, Hq, Hkv, Dk, Dv, page, window=0, sinks=0, logits=False, pad=0, spare=2):
    """Random requests over a cache whose blocks have scales of their own; rows past every length hold NaN."""
    B, width = len(lens), max(1, max(oa.pages(n, page) for n in lens)) + 1
    count = [oa.pages(n, page) for n in lens]
    n_pages = sum(count) + spare
    order = rng.permutation(n_pages)
    table = np.full((B, width), 1 << 30)                 # entries past a request's pages are never read
    at = 0
    live = np.zeros((n_pages, page), bool)
    for b in range(B):
        table[b, :count[b]] = order[at:at + count[b]]
        at += count[b]
        for j in range(count[b]):
            live[table[b, j], :max(0, min(page, lens[b] - j * page))] = True
    live = torch.from_numpy(live).cuda()[:, None, :, None]

    def side(dim):
        byte = torch.from_numpy(rng.integers(115, 124, (n_pages, Hkv, page // 16)).astype(np.uint8)).cuda()
        x = torch.from_numpy(rng.standard_normal((n_pages, Hkv, page, dim)).astype(np.float32)).cuda()
        loud = torch.from_numpy(2.0 ** rng.integers(-2, 2, (n_pages, Hkv, page // 16)).astype(np.float32)).cuda()
        by = loud / torch.exp2(byte.float() - 127.0)
        codes = (x * by.repeat_interleave(16, 2)[..., None]).clamp(-448, 448).to(E4M3).view(torch.uint8)
        return torch.where(live, codes, torch.full_like(codes, 0x7F)).view(E4M3), byte
    (k, ks), (v, vs) = side(Dk), side(Dv)
    cache = KVCache.of(k, v, ks, vs)
    starts = np.concatenate([[0], np.cumsum(new)])
    N = int(starts[-1]) + pad
    q = torch.from_numpy(rng.standard_normal((N, Hq, Dk)).astype(np.float32)).to(BF).cuda()
    sink = torch.from_numpy(rng.standard_normal(Hq).astype(np.float32)).cuda() if logits else None
    plan = StepPlan(starts=i32(starts), lens=i32(lens), table=i32(table), max_new=int(max(new)), status=word())
    return q, cache, plan, dict(window=window, sink_tokens=sinks, sink_logits=sink)


def _check(q, cache, plan, kw, scale=None, few=False):
    out = torch.full((q.shape[0], q.shape[1], cache.v_dim), float("nan"), dtype=BF, device="cuda")
    assert attend(q, cache, plan, scale=scale, out=out, **kw) is out
    plan.check()
    k, v = _values(cache)
    logits = kw.get("sink_logits")
    ref, size = oa.attend(f64(q), k, v, plan.starts.cpu().numpy(), plan.lens.cpu().numpy(), plan.table.cpu().numpy(),
                          cache.k_dim ** -0.5 if scale is None else scale, kw.get("window", 0), kw.get("sink_tokens", 0),
                          None if logits is None else f64(logits))
    x = f64(out)
    assert np.array_equal(np.isfinite(x), np.isfinite(ref))
    with np.errstate(invalid="ignore"):
        off = np.abs(x - ref) - (2.0 ** -8 * np.abs(ref) + ((0.0 if few else 2.0 ** -8) + 2.0 ** -11) * size)
    assert not (off > 0).any(), f"worst {np.nanmax(off):.3e} at {np.unravel_index(np.nanargmax(off), off.shape)}"
    return out


RAGGED = ([1, 15, 16, 17, 63, 64, 65, 130, 300], [1] * 9)


@pytest.mark.parametrize("dims", list(DIMS))
@pytest.mark.parametrize("heads", [(1, 1), (4, 4), (6, 2), (20, 1), (10, 2), (33, 1)])
def test_attend_decode(rng, dims, heads):
    few = heads[0] // heads[1] <= 32
    _check(*_attend_case(rng, *RAGGED, *heads, *DIMS[dims], 16), few=few)


@pytest.mark.parametrize("dims", list(DIMS))
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("lens,new,heads", [([3000, 7, 20000], [1, 1, 1], (8, 2)), ([900, 77], [4, 2], (8, 1)), ([300] * 40, [1] * 40, (3, 3))])
def test_attend_long_and_many(rng, dims, page, lens, new, heads):
    _check(*_attend_case(rng, lens, new, *heads, *DIMS[dims], page, logits=True), few=True)


@pytest.mark.parametrize("dims", list(DIMS))
@pytest.mark.parametrize("window,sinks,logits", [(0, 0, False), (0, 0, True), (50, 0, False), (16, 5, True), (1, 0, False), (130, 33, False)])
@pytest.mark.parametrize("page", [16, 64])
def test_attend_chunks(rng, dims, window, sinks, logits, page):
    _check(*_attend_case(rng, [200, 65, 1, 330, 129], [200, 64, 1, 37, 128], 6, 2, *DIMS[dims], page, window, sinks, logits, pad=3))


@pytest.mark.parametrize("dims", list(DIMS))
@pytest.mark.parametrize("window,sinks", [(128, 0), (128, 4), (40, 70), (1, 1), (5000, 3)])
def test_attend_decode_window(rng, dims, window, sinks):
    _check(*_attend_case(rng, [1, 16, 128, 129, 200, 1000, 4097], [1] * 7, 8, 2, *DIMS[dims], 16, window, sinks, True), few=True)


@pytest.mark.parametrize("dims", list(DIMS))
def test_attend_chunk_split_over_blocks(rng, dims):
    _check(*_attend_case(rng, [3000], [40], 8, 2, *DIMS[dims], 32))


@pytest.mark.parametrize("dims", list(DIMS))
@pytest.mark.parametrize("new", [1, 3, 60])
def test_attend_values_that_only_later_rows_see(rng, dims, new):
    """A NaN in the newest token's value stays out of the earlier tokens' rows."""
    q, cache, plan, kw = _attend_case(rng, [100 + new], [new], 4, 1, *DIMS[dims], 16)
    at = 100 + new - 1
    page = int(plan.table[0, at // 16])
    cache.v.view(torch.uint8)[page, :, at % 16, 3] = 0x7F
    out = _check(q, cache, plan, kw, few=new * 4 <= 32)
    assert torch.isnan(out[-1, :, 3]).all() and torch.isfinite(out[:-1]).all()


@pytest.mark.parametrize("dims", list(DIMS))
@pytest.mark.parametrize("heads,new", [((5, 1), 3), ((8, 2), 4), ((1, 1), 16), ((16, 1), 1), ((14, 2), 2), ((34, 2), 1)])
@pytest.mark.parametrize("window,sinks,page", [(0, 0, 16), (21, 3, 16), (100, 40, 64)])
def test_attend_up_to_sixteen_rows(rng, dims, heads, new, window, sinks, page):
    """Requests of several tokens that fill a tile of 16 rows, or leave some free; the last one has a row too many for it."""
    lens = [new, new + 15, 64, 0, 129, 143, 500, 4001]
    _check(*_attend_case(rng, lens, [new, new, 1, 0, new, new, new, new], *heads, *DIMS[dims], page, window, sinks, True, pad=2), few=True)


@pytest.mark.parametrize("dims", list(DIMS))
@pytest.mark.parametrize("heads,new,said", [((17, 1), 1, 0), ((40, 2), 1, 0), ((64, 1), 2, 0), ((132, 2), 1, 0), ((4, 2), 3, 0), ((16, 1), 3, 1), ((8, 2), 9, 2)])
def test_attend_with_more_new_tokens_than_said(rng, dims, heads, new, said):
    """max_new picks the kernel and nothing else, also where it says that no request has new tokens."""
    q, cache, plan, kw = _attend_case(rng, [new, 64, 150, 700], [new, 1, new, new], *heads, *DIMS[dims], 16, 0, 0, True, pad=1)
    plan.max_new = said
    _check(q, cache, plan, kw, few=max(said, 1) * heads[0] // heads[1] <= 32)


@pytest.mark.parametrize("dims", list(DIMS))
@pytest.mark.parametrize("reqs,heads,longest,window", [(130, (8, 4), 900, 0), (66, (4, 4), 2000, 480), (40, (4, 4), 480, 0), (129, (8, 4), 1100, 0)])
def test_attend_many_tiles_whole_and_split(rng, dims, reqs, heads, longest, window):
    """Tiles that fill the card and are not split, one as long as the table beside short ones, and some that are."""
    lens = rng.integers(1, 60, reqs).tolist()
    lens[reqs // 2], lens[-1] = longest, longest - 77
    _check(*_attend_case(rng, lens, [1] * reqs, *heads, *DIMS[dims], 64, window, 0, True), few=True)


@pytest.mark.parametrize("dims", list(DIMS))
@pytest.mark.parametrize("window,sinks", [(0, 0), (30, 0), (30, 20)])
def test_attend_few_rows_with_values_that_are_not_finite(rng, dims, window, sinks):
    """NaN in keys' values at both ends of a window: only the rows that see them have it, tile by tile."""
    q, cache, plan, kw = _attend_case(rng, [400, 70], [4, 4], 4, 1, *DIMS[dims], 16, window, sinks)
    codes = cache.v.view(torch.uint8)
    for b, at in [(0, 397), (0, 370), (0, 18), (1, 40), (1, 69)]:
        codes[int(plan.table[b, at // 16]), :, at % 16, at % 7] = 0x7F
    out = _check(q, cache, plan, kw, few=True)
    assert torch.isnan(out).any() and torch.isfinite(out).any()


def test_attend_scales_far_apart(rng):
    """Blocks whose values differ by 2^40: the large ones decide, and the small ones are there when they are alone."""
    q, cache, plan, kw = _attend_case(rng, [48, 16], [1, 1], 2, 1, 64, 64, 16)
    pages = plan.table[:, :3].tolist()
    cache.k_scale.fill_(60)                                # keys of next to nothing: equal weights
    cache.v_scale[pages[0][0]], cache.v_scale[pages[0][1]], cache.v_scale[pages[0][2]], cache.v_scale[pages[1][0]] = 160, 120, 121, 80
    _check(q, cache, plan, kw, few=True)


@pytest.mark.parametrize("what", ["page", "lens", "starts"])
def test_attend_refuses_bad_plans(rng, what):
    q, cache, plan, kw = _attend_case(rng, [40, 20], [3, 2], 4, 2, 64, 64, 16)
    if what == "page":
        plan.table[0, 1] = cache.n_pages + 5
    elif what == "lens":
        plan.lens[0] = 2
    else:
        plan.starts[1] = 9
    out = attend(q, cache, plan, **kw)
    with pytest.raises(ValueError):
        plan.check()
    if what != "page":
        assert not out[:3].any()


# ------------------------------------------------------------------ together
H, HEADS, KV, DK, DV, PAGE = 512, 8, 2, 192, 128, 16


def _layer(rng, rotary, pages=64, **kw):
    rows = HEADS * DK + KV * (DK + DV)
    return AttentionLayer(to_dev_bf16(rand_bf16(rng, (H,), 0.1) + 1.0), 1e-5, to_dev_bf16(rand_bf16(rng, (rows, H), H ** -0.5)),
                          to_dev_bf16(rand_bf16(rng, (H, HEADS * DV), (HEADS * DV) ** -0.5)), HEADS,
                          _empty(pages, PAGE, KV, DK, DV), rotary=rotary, **kw)


@pytest.mark.parametrize("window,form", [(0, "half stretched"), (24, "side stretched")])
def test_layer_steps(rng, window, form):
    """AttentionLayer over a cache with block scales: chunks, single tokens, rejected tokens, a request that ends, another in
    its pages.  Every step's output against attention in 64 bits over what read gives back, and what is read against the keys
    and values that went in, to E4M3's step under the scale of the largest of their block."""
    rotary, turn, _ = _rotary(64, form)
    layer = _layer(rng, rotary, window=window)
    c, pt = layer.cache, PageTable(2, 8, 12, PAGE)
    lens = [0, 0]
    history = [[], []]
    for target in ([40, 7], [41, 8], [44, 28], [42, 29], [0, 30], [50, 31], [51, 32]):
        new = [max(0, t - n) for t, n in zip(target, lens)]
        N = sum(new)
        x = to_dev_bf16(rand_bf16(rng, (N, H)))
        plan = pt.step(i32(target), N)
        h = layer(x, plan)
        plan.check()
        if N == 0:
            lens = list(target)
            continue
        r = torch.nn.functional.rms_norm(x.float(), (H,), layer.norm_weight.float(), 1e-5)
        q, k, v = (t.double().cpu().numpy() for t in torch.matmul(r.to(BF), layer.qkv_weight.T).split(layer.split, 1))
        positions = plan.positions.cpu().numpy()
        q, k, v = turn(q.reshape(N, HEADS, DK), positions), turn(k.reshape(N, KV, DK), positions), v.reshape(N, KV, DV)
        at = 0
        o = np.zeros((N, HEADS, DV))
        for b in range(2):
            history[b] = history[b][:target[b]] + [(k[at + i], v[at + i]) for i in range(new[b])]
            if not new[b]:
                continue
            kk, vv = (f64(t) for t in read(c, pt.slots(b, target[b])))
            for got, side in ((kk, 0), (vv, 1)):
                want = np.stack([p[side] for p in history[b]])
                # half a step of E4M3 is 2^-4 of a value; the scale may be that of a rejected token's larger values, and q, k
                # and v come from another order of sums than the layer's, a bf16 step apart
                for j in range(0, target[b], 16):
                    assert np.abs(got[j:j + 16] - want[j:j + 16]).max() <= 2.0 ** -3 * max(1.0, np.abs(want[j:j + 16]).max())
            pos = np.arange(target[b] - new[b], target[b])
            for head in range(HEADS):
                g = head // (HEADS // KV)
                s = q[at:at + new[b], head] @ kk[:, g].T * DK ** -0.5
                j = np.arange(target[b])
                seen = j <= pos[:, None]
                if window:
                    seen &= pos[:, None] - j < window
                w = np.where(seen, np.exp(s - np.where(seen, s, -np.inf).max(1, keepdims=True)), 0.0)
                o[at:at + new[b], head] = (w / w.sum(1, keepdims=True)) @ vv[:, g]
            at += new[b]
        # q is rounded to bf16 before and after its rotation, o before its product, y and h once: some 2^-8 each of values of
        # the size of o, spread over 1024 products whose errors are of either sign
        want = x.double().cpu().numpy() + o.reshape(N, -1) @ layer.o_weight.double().cpu().numpy().T
        assert np.abs(f64(h) - want).max() <= 2.0 ** -5 * max(1.0, np.abs(want).max())
        lens = list(target)


def test_a_graph_of_steps_replays(rng):
    """step, append, read and attend captured once, replayed over growing requests with eager work between, each replay against
    the eager calls on a copy of the state."""
    rotary = Rotary(64, interleaved=True, frequencies=stretched(64, 10000.0, 8.0, 4096), magnitude=1.2)
    B, n_pages = 3, 30
    caches = [_empty(n_pages, PAGE, KV, DK, DV) for _ in range(2)]
    tables = [PageTable(B, 8, n_pages, PAGE) for _ in range(2)]
    target = i32([1, 1, 1])
    rows = [torch.zeros(B, h, d, dtype=BF, device="cuda") for h, d in ((HEADS, DK), (KV, DK), (KV, DV))]

    def step(cache, pt):
        plan = pt.step(target, B, max_new=1)
        q = append(cache, plan, rows[1], rows[2], q=rows[0], rotary=rotary)
        return attend(q, cache, plan), read(cache, plan.slots), plan.status
    warm = _empty(n_pages, PAGE, KV, DK, DV), PageTable(B, 8, n_pages, PAGE)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*warm)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, back, status = step(caches[0], tables[0])
    for n in range(1, 40):
        target.fill_(n)
        for t in rows:
            t.copy_(torch.from_numpy(rng.standard_normal(t.shape).astype(np.float32) * 2.0 ** rng.integers(-4, 5)))
        graph.replay()
        want, want_back, want_status = step(caches[1], tables[1])
        torch.cuda.synchronize()
        assert status.item() == 0 and want_status.item() == 0
        assert torch.equal(out, want) and torch.equal(back[0], want_back[0]) and torch.equal(back[1], want_back[1]), n
        for a, b in ((caches[0].k, caches[1].k), (caches[0].v, caches[1].v)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        assert torch.equal(caches[0].k_scale, caches[1].k_scale) and torch.equal(caches[0].v_scale, caches[1].v_scale)


def test_calls_on_another_stream(rng):
    q, cache, plan, kw = _attend_case(rng, *RAGGED, 8, 2, 192, 128, 16, logits=True)
    want, rows = attend(q, cache, plan, **kw), read(cache, i32(np.arange(0, 160, 3)))
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got, again = attend(q, cache, plan, **kw), read(cache, i32(np.arange(0, 160, 3)))
    other.synchronize()
    assert torch.equal(got, want) and torch.equal(again[0].view(torch.int16), rows[0].view(torch.int16))


@pytest.mark.parametrize("dims", list(DIMS))
@pytest.mark.parametrize("what", ["nan", "inf", "-inf"])
def test_attend_queries_that_are_not_finite(rng, dims, what):
    """A query that holds a NaN or an infinity makes its own row what the formula makes it, and no other."""
    q, cache, plan, kw = _attend_case(rng, [150, 40], [70, 33], 4, 2, *DIMS[dims], 16, window=30)
    q[5, 1, 7] = q[80, 2, 63] = float(what)
    x = torch.full((q.shape[0], 4, cache.v_dim), -1.0, dtype=BF, device="cuda")
    attend(q, cache, plan, out=x, **kw)
    plan.check()
    clean = q.clone()
    clean[5, 1, 7] = clean[80, 2, 63] = 0.0
    want = attend(clean, cache, plan, **kw)
    others = torch.ones(q.shape[:2], dtype=torch.bool, device="cuda")
    others[5, 1] = others[80, 2] = False
    # the rows beside it may be taken again in 32 bits: both within the rounding of weights and output of the same value
    assert torch.isfinite(x[others]).all() and (x[others].float() - want[others].float()).abs().max() <= 2.0 ** -5
    if what == "nan":
        assert torch.isnan(x[5, 1]).all() and torch.isnan(x[80, 2]).all()
    else:
        k, v = _values(cache)
        ref, _ = oa.attend(f64(q), k, v, plan.starts.cpu().numpy(), plan.lens.cpu().numpy(), plan.table.cpu().numpy(), cache.k_dim ** -0.5, 30)
        got = f64(x)
        for n, h in ((5, 1), (80, 2)):
            assert np.array_equal(np.isnan(got[n, h]), np.isnan(ref[n, h]))


@pytest.mark.parametrize("dims", list(DIMS))
@pytest.mark.parametrize("new", [1, 50])
def test_attend_queries_of_far_sizes(rng, dims, new):
    """Dimensions of a query from 2^-12 of its largest up: every one counts, against keys that weigh the small ones more."""
    q, cache, plan, kw = _attend_case(rng, [90], [new], 4, 2, *DIMS[dims], 16)
    Dk = DIMS[dims][0]
    small = 2.0 ** -rng.integers(0, 12, (q.shape[0], 4, Dk))
    q.copy_(torch.from_numpy((rng.standard_normal(q.shape) * small).astype(np.float32)).to(BF))
    _check(q, cache, plan, kw, scale=0.2, few=new == 1)
    tiny = (q.float() * 2.0 ** -100).to(BF)                # the same far below 1, and a scale that takes it back
    _check(tiny, cache, plan, kw, scale=0.2 * 2.0 ** 100, few=new == 1)


@pytest.mark.parametrize("scale", [-0.1, 0.0])
def test_attend_scales_of_either_sign(rng, scale):
    _check(*_attend_case(rng, [150, 40], [70, 33], 4, 2, 192, 128, 16), scale=scale)


@pytest.mark.parametrize("heads,N,piece", [(1, 40000, 997), (2, 5000, 613), (9, 2100, 250)])
def test_long_calls_are_their_pieces(rng, heads, N, piece):
    """Calls of every number of rows that a block of threads may look at, bit for bit as in pieces that do not end with a block
    of slots; values whose codes stay in the normal range under any scale they meet."""
    D, page = 64, 64

    def rows():
        x = 2.0 ** rng.uniform(-3, 2.99, (N, heads, D)) * rng.choice([-1.0, 1.0], (N, heads, D))
        return torch.from_numpy(x.astype(np.float32)).to(BF).cuda()
    k, v = rows(), rows()
    ends = np.minimum(np.arange(piece, N + piece, piece), N)
    held = []
    for cuts in ([N], ends):
        n_pages = oa.pages(N, page) + 1
        cache, pt, at = _empty(n_pages, page, heads, D, D), PageTable(1, n_pages, n_pages, page), 0
        for end in cuts:
            plan = pt.step(i32([end]), int(end) - at)
            append(cache, plan, k[at:end], v[at:end])
            plan.check()
            at = int(end)
        held.append((cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale))
    assert all(torch.equal(a, b) for a, b in zip(*held))
    got = read(cache, pt.slots(0, N))
    assert ((got[0].float() - k.float()).abs() <= 2.0 ** -4 * k.float().abs()).all()
    assert ((got[1].float() - v.float()).abs() <= 2.0 ** -4 * v.float().abs()).all()


def test_a_padded_step(rng):
    """Rows behind a step's last token: not written, their attention is 0, and what the cache holds beside them stays."""
    cache, pt = _random_cache(rng, 6, 16, KV, DK, DV, 119, 124), PageTable(2, 3, 6, 16)
    before = [t.view(torch.uint8).clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    plan = pt.step(i32([5, 17]), 40)
    q, k, v = (torch.from_numpy(rng.standard_normal((40, h, d)).astype(np.float32)).to(BF).cuda() for h, d in ((HEADS, DK), (KV, DK), (KV, DV)))
    q = append(cache, plan, k, v, q=q, rotary=Rotary(64))
    out = attend(q, cache, plan)
    plan.check()
    assert not out[22:].any() and bool(out[:22].any())
    written = torch.zeros(6 * 16, dtype=torch.bool, device="cuda")
    written[plan.slots[:22].long()] = True
    for t, old in ((cache.k, before[0]), (cache.v, before[1])):
        now = t.view(torch.uint8).transpose(1, 2).flatten(0, 1)
        assert torch.equal(now[~written], old.transpose(1, 2).flatten(0, 1)[~written])
    blocks = torch.zeros(6, dtype=torch.bool, device="cuda")
    blocks[plan.slots[:22].long() // 16] = True
    for t, old in ((cache.k_scale, before[2]), (cache.v_scale, before[3])):
        assert torch.equal(t[~blocks], old[~blocks])
    none = pt.step(i32([5, 17]), 3)
    assert not attend(q[:3].contiguous(), cache, none).any()
