"""Values at the edges of what a cache with block scales holds: infinities and NaN in blocks that several waves share, and the least
scales, whose products lie below bf16's normal range."""
import numpy as np
import pytest
import torch

from mimo_stream import KVCache, StepPlan, append, attend, read
from test_gpu_block_scales import BF, DIMS, _check_blocks, _empty, _random_cache, _rotary, f64, i32, word

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ["half", "side", "half stretched"])
@pytest.mark.parametrize("dims", list(DIMS))
@pytest.mark.parametrize("Hkv,rot", [(3, 0), (3, 32), (8, 64), (5, -1)])
def test_append_of_values_that_are_not_finite(rng, dims, form, Hkv, rot):
    """Runs of 1 to 16 rows of a block: what is not finite in a row and head leaves every scale to the finite values, the codes of
    the others as they are, and the units that a block of threads takes after it too."""
    Dk, Dv = DIMS[dims]
    rot = Dk if rot < 0 else rot
    page, n_pages = 64, 16
    blocks = rng.permutation(n_pages * page // 16)
    slots = np.array([16 * b + i for n, b in zip([16, 5, 11, 3, 16, 8, 1, 13, 6, 16, 7, 2, 15], blocks) for i in rng.permutation(16)[:n]])
    N = len(slots)
    cache = _random_cache(rng, n_pages, page, Hkv, Dk, Dv, 118, 126)
    before = [t.cpu().clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]

    def rows(d):
        x = rng.standard_normal((N, Hkv, d)) * 2.0 ** rng.integers(-3, 4, (N, Hkv, 1))
        for _ in range(N * Hkv // 6):
            x[rng.integers(N), rng.integers(Hkv), rng.integers(d)] = rng.choice([np.inf, -np.inf, np.nan])
        x[3, 1], x[20, 2] = np.nan, np.inf                 # nothing finite at all
        return torch.from_numpy(x.astype(np.float32)).to(BF).cuda()
    k, v = rows(Dk), rows(Dv)
    positions = rng.integers(1, 1 << 20, N)
    rotary, turn, slack = _rotary(rot, form) if rot else (None, lambda x, at: x, np.abs)
    plan = StepPlan(slots=i32(slots), positions=i32(positions), status=word())
    append(cache, plan, k, v, rotary=rotary)
    plan.check()
    with np.errstate(invalid="ignore"):
        for pages, scale, held, byte, ref, room in ((cache.k, cache.k_scale, before[0], before[2], turn(f64(k), positions), slack(f64(k))),
                                                    (cache.v, cache.v_scale, before[1], before[3], f64(v), np.zeros(v.shape))):
            _check_blocks(pages, scale, held, byte.numpy().astype(np.int64), ref, room, slots, page)
            codes = f64(pages).transpose(0, 2, 1, 3).reshape(n_pages * page, Hkv, -1)[slots]
            assert np.isnan(ref).any() and np.isinf(ref).any()
            assert np.array_equal(np.isnan(codes), np.isnan(ref))
            assert (codes[ref == np.inf] == 448.0).all() and (codes[ref == -np.inf] == -448.0).all()


@pytest.mark.parametrize("byte", [1, 2, 3])
def test_the_least_scales(byte):
    """Every code times 2^(byte - 127), rounded to nearest even where it lies between bf16's subnormal steps of 2^-133 (bytes 1 and
    2), is what read gives, and attend too of one key, in tiles of 16, 32 and 128 rows."""
    codes = torch.arange(256, dtype=torch.uint8).view(2, 128)
    codes[:, 127] = 0x7E                                   # no NaN
    want = (codes.view(torch.float8_e4m3fn).double() * 2.0 ** (byte - 127)).float().to(BF)   # fp32 holds the products
    cache = _empty(2, 16, 2, 128, 128)
    for side, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        side.view(torch.uint8)[1, :, 5] = codes.cuda()
        scale.fill_(byte)
    for got in read(cache, i32([16 + 5])):
        assert torch.equal(got[0].cpu().view(torch.int16), want.view(torch.int16))
    one = KVCache.of(cache.k[1:, :, :, :].contiguous(), cache.v[1:].contiguous(), cache.k_scale[1:].clone(), cache.v_scale[1:].clone())
    for side in (one.k, one.v):
        side.view(torch.uint8)[0, :, 0] = codes.cuda()
    for G in (1, 20, 40):
        q = torch.zeros(1, 2 * G, 128, dtype=BF, device="cuda")
        out = attend(q, one, StepPlan(starts=i32([0, 1]), lens=i32([1]), table=i32([[0]]), max_new=1)).cpu().view(2, G, 128)
        assert torch.equal(out, want[:, None].expand(2, G, 128)), G


def test_the_least_values_come_back():
    """2^-133, bf16's least, and 2^-126 through append and read."""
    x = torch.zeros(1, 1, 64, dtype=BF, device="cuda")
    x[0, 0, :3] = torch.tensor([2.0 ** -133, -(2.0 ** -126), 2.0 ** -127])
    cache = _empty(1, 16, 1, 64, 64)
    append(cache, StepPlan(slots=i32([0]), positions=i32([0])), x, x)
    assert cache.k_scale.item() == 1
    for got in read(cache, i32([0])):
        assert torch.equal(got, x)
