"""The frequencies of stretched contexts against values worked out by hand.

Pair i turns original theta^(-2 i / dim) / 2 pi times over the original length, so t turns belong to the real pair number
n(t) = dim ln(original / 2 pi t) / 2 ln theta.  With a = floor n(32) (0 at least) and b = ceil n(1) (dim - 1 at most), pair i has its
frequency times 1 - s (1 - 1 / factor), s = (i - a) / (b - a) between them, 0 up to a and 1 from b on."""
import numpy as np
import pytest

from mimo_stream import stretched
from oracle import attention as oa


def both(dim, theta, factor, original, few=1.0, many=32.0):
    """The share that is left of every pair's frequency, by the package and by the oracle."""
    plain = theta ** (-2.0 * np.arange(dim // 2) / dim)
    return [np.asarray(f) / plain for f in (stretched(dim, theta, factor, original, few, many).numpy(), oa.stretched(dim, theta, factor, original, few, many))]


# n(32) and n(1); what is left is 1 - (i - a) / (b - a) * 3 / 4
@pytest.mark.parametrize("dim,original,a,b", [(64, 131072, 22, 35),        # 22.51, 34.55: the slowest pair turns 2.78 times
                                              (64, 65536, 20, 33),         # 20.11, 32.15
                                              (128, 131072, 45, 70),       # 45.03, 69.11
                                              (64, 4096, 10, 23)])         # 10.47, 22.51: the slowest pair turns 0.09 times
def test_the_blend_goes_past_the_last_pair(dim, original, a, b):
    i = np.arange(dim // 2)
    want = 1.0 - 0.75 * np.clip((i - a) / (b - a), 0.0, 1.0)
    for got in both(dim, 10000.0, 4.0, original):
        assert np.allclose(got, want, rtol=1e-12, atol=0)


def test_the_last_pairs_by_hand():
    for got in both(64, 10000.0, 4.0, 131072):
        assert got[31] == pytest.approx(25.0 / 52.0, rel=1e-12) and got[23] == pytest.approx(49.0 / 52.0, rel=1e-12) and got[22] == 1.0
    for got in both(64, 10000.0, 4.0, 65536):
        assert got[31] == pytest.approx(19.0 / 52.0, rel=1e-12)
    for got in both(128, 10000.0, 4.0, 131072):
        assert got[63] == pytest.approx(0.46, rel=1e-12)


def test_the_blend_ends_at_dim_less_one():
    """theta 2, dim 16: 265 tokens are 3.19 pairs for 32 turns and 43.2 for one, taken as 3 and 15."""
    for got in both(16, 2.0, 4.0, 265):
        assert np.allclose(got, [1, 1, 1, 1, 1 - 0.75 / 12, 1 - 1.5 / 12, 1 - 2.25 / 12, 0.75], rtol=1e-12, atol=0)


@pytest.mark.parametrize("theta,original", [(2.0, 2000), (10000.0, 1 << 40)])
def test_pairs_of_many_turns_keep_theirs(theta, original):
    for got in both(16, theta, 4.0, original):
        assert np.allclose(got, 1.0, rtol=1e-14, atol=0)


@pytest.mark.parametrize("original", [1, 3, 6])
def test_no_pair_of_few_turns_keeps_its_own(original):
    """6 tokens are 0.95 turns of pair 0, the fastest."""
    for got in both(16, 10000.0, 4.0, original):
        assert np.allclose(got, 0.25, rtol=1e-14, atol=0)


@pytest.mark.parametrize("name", ["theta", "factor", "original", "many"])
def test_numbers_without_an_end_are_refused(name):
    with pytest.raises(ValueError, match="finite"):
        stretched(**{**dict(dim=16, theta=10000.0, factor=2.0, original=4096), name: float("inf")})


def test_between_few_and_many_from_pair_0_on():
    """theta 16, dim 16: 100 tokens are 15.9 turns of pair 0 and n(1) = 7.98, so pairs 0 to 7 of 8."""
    for got in both(16, 16.0, 4.0, 100):
        assert np.allclose(got, 1.0 - 0.75 * np.arange(8) / 8, rtol=1e-12, atol=0)
