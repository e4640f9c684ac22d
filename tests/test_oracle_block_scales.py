"""The oracle of the cache with block scales and of the rotary forms, against hand values and other ways to the same."""
import numpy as np
import pytest

from oracle import attention as oa


@pytest.mark.parametrize("most,byte", [(0.0, 1), (2.0 ** -140, 1), (448.0, 127), (448.0000001, 128), (449.0, 128), (224.0, 126), (1.0, 119),
                                       (1.75, 119), (1.7500001, 120), (3.0e38, 246), (448 * 2.0 ** 119, 246), (2.0 ** -119, 1)])
def test_block_byte(most, byte):
    assert oa.block_byte(most) == byte


def test_block_byte_is_the_least_that_holds():
    for most in np.exp(np.random.default_rng(1).uniform(-80, 80, 500)):
        s = oa.block_byte(most)
        assert most <= 448 * 2.0 ** (s - 127) and (s == 1 or most > 448 * 2.0 ** (s - 128))


def test_block_write_by_hand():
    held, byte = np.full((1, 1, 32, 1), 100.0), np.array([[[120, 130]]])
    x = np.array([[[1000.0]], [[2.0]], [[5.0]]])
    codes, after = oa.block_write(held, byte, x, np.array([3, 5, 16]), 32)
    assert after.tolist() == [[[129, 121]]]                # 1000 needs 2^2: 1000 / 4 = 250; 5 alone needs 2^-6
    assert codes[0, 0, 3, 0] == 250.0 and codes[0, 0, 5, 0] == 0.5 and codes[0, 0, 0, 0] == 100.0 / 512
    assert codes[0, 0, 16, 0] == 320.0 and codes[0, 0, 17, 0] == 100.0
    assert oa.block_values(codes, after)[0, 0, [0, 3, 16], 0].tolist() == [100.0 / 128, 1000.0, 5.0]


def test_block_write_keeps_non_finite_values_out_of_the_scale():
    x = np.array([[[np.nan, np.inf, -np.inf, 3.0]]])
    codes, byte = oa.block_write(np.zeros((1, 1, 16, 4)), np.zeros((1, 1, 1)), x, np.array([0]), 16)
    assert byte.tolist() == [[[oa.block_byte(3.0)]]]
    assert np.isnan(codes[0, 0, 0, 0]) and codes[0, 0, 0, 1:3].tolist() == [448.0, -448.0]


def test_turn_is_rotate_in_the_half_layout(rng):
    x = rng.standard_normal((5, 2, 64))
    at = rng.integers(0, 1 << 20, 5)
    f = 10000.0 ** (-2.0 * np.arange(16) / 32)
    assert np.allclose(oa.turn(x, at, f), oa.rotate(x, at, 32, 10000.0), rtol=0, atol=1e-12)


def test_turn_side_by_side_is_a_complex_product(rng):
    x = rng.standard_normal((5, 2, 64))
    at = rng.integers(0, 1 << 20, 5)
    f = 10000.0 ** (-2.0 * np.arange(16) / 32)
    z = (x[..., :32:2] + 1j * x[..., 1:32:2]) * 1.5 * np.exp(1j * at[:, None, None] * f)
    y = oa.turn(x, at, f, True, 1.5)
    assert np.allclose(y[..., :32:2], z.real, atol=1e-9) and np.allclose(y[..., 1:32:2], z.imag, atol=1e-9)
    assert np.array_equal(y[..., 32:], x[..., 32:])


def test_stretched_ends_and_middle():
    plain = 10000.0 ** (-2.0 * np.arange(32) / 64)
    f = oa.stretched(64, 10000.0, 8.0, 4096, 1.0, 32.0)
    turns = 4096 * plain / (2 * np.pi)
    assert np.allclose(f[turns >= 40], plain[turns >= 40]) and np.allclose(f[turns < 0.7], plain[turns < 0.7] / 8)
    between = (turns < 32) & (turns > 1)
    assert between.any() and ((f < plain) & (f > plain / 8))[between].all()
    assert np.allclose(oa.stretched(64, 10000.0, 1.0, 4096, 1.0, 32.0), plain)


@pytest.mark.parametrize("dim,theta,factor,original", [(64, 10000.0, 32.0, 4096), (192, 5.0e6, 8.0, 4096), (32, 10000.0, 2.5, 100), (16, 10000.0, 4.0, 3)])
def test_stretched_of_the_package(dim, theta, factor, original):
    from mimo_stream import stretched
    assert np.allclose(stretched(dim, theta, factor, original).numpy(), oa.stretched(dim, theta, factor, original, 1.0, 32.0), rtol=1e-13)
