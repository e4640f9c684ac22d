"""CPU pins of oracle.attention: tiny cases worked out by hand or by another formula."""
import numpy as np
import pytest

from oracle import attention as oa


def test_step_takes_and_returns_pages():
    table = np.zeros((3, 4), np.int64)
    table[0, :2] = [7, 3]
    table[1, :1] = [5]
    free = np.array([9, 8, 6, 0, 0])
    starts, lens, slots, pos, n_free, tab, fr = oa.step([17, 16, 0], [18, 17, 1], table, free, 3, 16, 4)
    assert starts.tolist() == [0, 1, 2, 3] and pos.tolist() == [17, 16, 0, 0]
    assert tab[1, 1] == 6 and tab[2, 0] == 8 and n_free == 1
    assert slots.tolist() == [3 * 16 + 1, 6 * 16, 8 * 16, -1]
    # the way back leaves the stack as it was
    _, _, s2, _, n2, _, fr2 = oa.step([18, 17, 1], [17, 16, 0], tab, fr, n_free, 16, 1)
    assert n2 == 3 and fr2[:3].tolist() == [9, 8, 6] and s2.tolist() == [-1]


def test_rotation_keeps_length_and_is_relative(rng):
    x, y = rng.standard_normal((1, 1, 8)), rng.standard_normal((1, 1, 8))
    def dot(p, q):
        return float((oa.rotate(x, [p], 8, 100.0) * oa.rotate(y, [q], 8, 100.0)).sum())
    assert abs(dot(5, 2) - dot(1005, 1002)) < 1e-9
    assert np.allclose(np.linalg.norm(oa.rotate(x, [77], 4, 100.0)), np.linalg.norm(x))
    assert np.array_equal(oa.rotate(x, [77], 4, 100.0)[..., 4:], x[..., 4:])


@pytest.mark.parametrize("window,sinks,p,want", [(0, 0, 2, [0, 1, 2]), (2, 0, 4, [3, 4]), (2, 1, 4, [0, 3, 4]), (2, 9, 4, [0, 1, 2, 3, 4]),
                                                 (1, 0, 0, [0])])
def test_visible(window, sinks, p, want):
    assert np.flatnonzero(oa.visible(p, 6, window, sinks)).tolist() == want


def test_attend_uniform_scores_and_sink_logit(rng):
    v = rng.standard_normal((2, 1, 2, 4))
    k = np.zeros((2, 1, 2, 4))
    q = rng.standard_normal((2, 3, 4))
    out, _ = oa.attend(q, k, v, [0, 2], [3], [[1, 0]], 1.0)
    rows = np.concatenate([v[1, 0], v[0, 0]])
    assert np.allclose(out[0], rows[:2].mean(0)) and np.allclose(out[1], rows[:3].mean(0))
    out, _ = oa.attend(q, k, v, [0, 2], [3], [[1, 0]], 1.0, sink_logits=np.log([1.0, 2.0, 3.0]))
    for h in range(3):
        assert np.allclose(out[1, h], rows[:3].sum(0) / (3 + h + 1))
