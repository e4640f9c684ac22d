"""append's rotary argument that is not a plain Rotary: what has a dim and turns, and classes derived from Rotary."""
import copy
import math
import pickle
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from mimo_stream import KVCache, Rotary, StepPlan, append
from mimo_stream.attention import _turns_of

CPU = torch.device("cpu")


class Stretched(Rotary):
    """Every frequency divided by a factor, set after the fact."""
    def __init__(self, dim, factor, device="cuda"):
        super().__init__(dim, device=device)
        self.factor = factor
        self.turns = self.turns / factor


class Plain(Rotary):
    def __init__(self, dim, device="cuda"):
        self.dim = dim
        self.turns = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim) / (2.0 * math.pi)


def test_what_a_call_is_given():
    r = Rotary(32, device="cpu", interleaved=True, magnitude=0.5)
    assert _turns_of(r, CPU, 64)[0] is r._struct
    for other in (SimpleNamespace(dim=32, turns=r.turns), Plain(32, "cpu")):
        s, turns = _turns_of(other, CPU, 64)
        assert (s.dim, s.interleaved, s.magnitude, s.turns) == (32, 0, 1.0, turns.data_ptr()) and torch.equal(turns, r.turns)
    s, _ = _turns_of(SimpleNamespace(dim=32, turns=r.turns, interleaved=True, magnitude=0.5), CPU, 64)
    assert (s.interleaved, s.magnitude) == (1, 0.5)
    s, turns = _turns_of(Stretched(32, 4.0, "cpu"), CPU, 64)
    assert s.turns == turns.data_ptr() and torch.equal(turns, r.turns / 4.0)


@pytest.mark.parametrize("dim,turns,match", [(80, torch.zeros(40, dtype=torch.float64), "dimension"), (-16, torch.zeros(8, dtype=torch.float64), "dimension"),
                                             (32, torch.zeros(15, dtype=torch.float64), "turns"), (32, torch.zeros(16), "turns"),
                                             (32, torch.zeros(32, dtype=torch.float64)[::2], "turns"), (32, torch.zeros(16, dtype=torch.float64, device="meta"), "meta")])
def test_what_is_refused(dim, turns, match):
    with pytest.raises(ValueError, match=match):
        _turns_of(SimpleNamespace(dim=dim, turns=turns), CPU, 64)


@pytest.mark.parametrize("again", [copy.copy, copy.deepcopy, lambda r: pickle.loads(pickle.dumps(r))])
def test_a_derived_one_is_copied_whole(again):
    r = again(Stretched(32, 4.0, "cpu"))
    assert r.factor == 4.0 and r.dim == 32 and torch.equal(r.turns, Rotary(32, device="cpu").turns / 4.0)


class Worked(Rotary):
    """Has no numbers of its own: they are worked out from a factor."""
    def __init__(self, factor):
        self.factor = factor
    dim = property(lambda self: 32)
    turns = property(lambda self: Rotary(32, device="cpu").turns / self.factor)


@pytest.mark.parametrize("again", [copy.copy, copy.deepcopy, lambda r: pickle.loads(pickle.dumps(r))])
def test_a_derived_one_without_numbers_is_copied(again):
    r = again(Worked(2.0))
    s, turns = _turns_of(r, CPU, 64)
    assert r.factor == 2.0 and s.turns == turns.data_ptr() and torch.equal(turns, Rotary(32, device="cpu").turns / 2.0)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "blocks"])
def test_append_takes_them(rng, kind):
    N, heads, D = 9, 2, 64
    q, k, v = (torch.from_numpy(rng.standard_normal((N, heads, D)).astype(np.float32)).to(torch.bfloat16).cuda() for _ in range(3))
    slots = torch.arange(N, dtype=torch.int32, device="cuda")
    freq = torch.as_tensor(10000.0 ** (-torch.arange(0, 32, 2, dtype=torch.float64) / 32))

    def result(rotary):
        cache = KVCache(1, 16, heads, D, D) if kind == "bf16" else KVCache(1, 16, heads, D, D, dtype=torch.float8_e4m3fn, block_scales=True)
        return append(cache, StepPlan(slots=slots, positions=slots + 100), k, v, q=q, rotary=rotary), cache.k.view(torch.uint8)
    plain, as_made = Rotary(32), Rotary.__new__(Rotary)
    as_made.__setstate__({"dim": 32, "turns": Plain(32).turns})
    side = Rotary(32, interleaved=True, magnitude=1.5)
    for rotary, same in ((SimpleNamespace(dim=32, turns=plain.turns), plain), (Plain(32), as_made),
                         (Stretched(32, 4.0), Rotary(32, frequencies=freq / 4.0)), (SimpleNamespace(dim=32, turns=side.turns, interleaved=True, magnitude=1.5), side)):
        got, want = result(rotary), result(same)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
