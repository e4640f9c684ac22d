"""Wide tiles over block scales take q as two planes of E4M3: exact down to 2^-13 of the largest of a row's 64 dimensions, and to within
2^-21 of it below.  (Two planes of 4 bits, the second of 16 times what the first leaves: with the largest above 224, values of 2^-6
and more have all 8 bits of bf16; below, the second plane's half step of 2^-10 is 2^-14 of the first's unit, 2^-21.8 of 224.)"""
import numpy as np
import pytest
import torch

from mimo_stream import KVCache, StepPlan, attend
from oracle import attention as oa
from test_gpu_block_scales import BF, DIMS, E4M3, _values, f64, i32, word

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dims", list(DIMS))
@pytest.mark.parametrize("far", [13, 16, 20, 26])
def test_dimensions_far_below_the_largest(rng, dims, far):
    """Some dimensions of q 2^-far of the others, and keys that are larger there, so that the scores hang on them."""
    Dk, Dv = DIMS[dims]
    heads, kv, new, length, page = 4, 2, 50, 90, 16
    small = np.zeros(Dk, int)
    for b in range(Dk // 64):
        small[64 * b + rng.permutation(64)[:6]] = far
    q = torch.from_numpy((rng.standard_normal((new, heads, Dk)) * 2.0 ** -small).astype(np.float32)).to(BF).cuda()
    n_pages = oa.pages(length, page)
    # keys of 2^-9 in the large dimensions' codes and up to 2^6 in the small ones'
    loud = 2.0 ** (np.minimum(small, 13) - 8.0)
    k, v = (torch.from_numpy((rng.standard_normal((n_pages, kv, page, d)) * by).astype(np.float32)).cuda().clamp(-448, 448).to(E4M3)
            for d, by in ((Dk, loud), (Dv, 1.0)))
    byte = torch.full((n_pages, kv, 1), 127, dtype=torch.uint8, device="cuda")
    cache = KVCache.of(k, v, byte, byte.clone())
    plan = StepPlan(starts=i32([0, new]), lens=i32([length]), table=i32([np.arange(n_pages)]), max_new=new, status=word())
    scale = 64.0 * Dk ** -0.5 * 2.0 ** (max(far, 13) - 13)
    out = f64(attend(q, cache, plan, scale=scale))
    plan.check()
    kk, vv = _values(cache)
    ref, size = oa.attend(f64(q), kk, vv, np.array([0, new]), np.array([length]), np.arange(n_pages)[None], scale)
    x = np.abs(f64(q)).reshape(new, heads, -1, 64)
    largest = x.max(-1, keepdims=True)
    lost = np.where(x < 2.0 ** -13 * largest, 2.0 ** -21 * largest, 0.0).reshape(new, heads, Dk)
    most = np.abs(kk).max((0, 2)).repeat(heads // kv, 0)   # [heads, Dk]
    off = scale * (lost * most).sum(-1)[..., None]         # of a score, at most
    # weights are off by exp(2 off), and as elsewhere by their rounding and by 32-bit scores
    assert (np.abs(out - ref) <= 2.0 ** -8 * np.abs(ref) + (2.0 ** -8 + 2.0 ** -11 + np.expm1(2.0 * off)) * size).all()
