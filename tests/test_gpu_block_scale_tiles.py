"""Attention over block scales of requests with several new tokens, on both sides of the rules that leave tiles of 16 rows whole."""
import pytest

from test_gpu_block_scales import DIMS, _attend_case, _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dims", list(DIMS))
@pytest.mark.parametrize("reqs,new,heads,window", [(8, 16, (4, 4), 0), (9, 16, (4, 4), 480), (16, 16, (8, 8), 0), (32, 4, (16, 4), 0), (31, 4, (16, 4), 500),
                                                   (70, 2, (8, 4), 0)])
def test_drafts(rng, dims, reqs, new, heads, window):
    lens = rng.integers(new, 900, reqs).tolist()
    lens[0], lens[-1] = 1024, new
    _check(*_attend_case(rng, lens, [new] * (reqs - 1) + [1], *heads, *DIMS[dims], 64, window, 0, True, pad=3), few=True)
