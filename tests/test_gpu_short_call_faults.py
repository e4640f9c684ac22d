"""The short host path where it cannot serve: tensors that have no memory of their own (inside of torch.vmap) are an error, and the
process goes on; without the module of the short path every call goes the long way."""
import numpy as np
import pytest
import torch

from mimo_stream import KVCache, PageTable, StepPlan, _lib, append, attend, read

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def _state():
    cache, pt = KVCache(4, 16, 2, 64, 64), PageTable(2, 2, 4, 16)
    plan = pt.step(i32([3, 2]), 5)
    q, k, v = (torch.ones(5, h, 64, dtype=BF, device="cuda") for h in (4, 2, 2))
    append(cache, plan, k, v)
    return cache, plan, q, k, v, attend(q, cache, plan)


def _twice(t):
    return torch.stack((t, t))


@pytest.mark.parametrize("what", ["slots", "positions", "k", "q"])
def test_append(what):
    cache, plan, q, k, v, _ = _state()

    def call(x):
        given = dict(slots=plan.slots, positions=plan.positions, k=k, q=q)
        given[what] = x
        return append(cache, StepPlan(slots=given["slots"], positions=given["positions"]), given["k"], v, q=given["q"])
    with pytest.raises(RuntimeError, match="data pointer|storage"):
        torch.vmap(call)(_twice(dict(slots=plan.slots, positions=plan.positions, k=k, q=q)[what]))
    assert torch.equal(append(cache, plan, k, v, q=q), q)


def test_read():
    cache, plan, _, k, _, _ = _state()
    with pytest.raises(RuntimeError, match="data pointer|storage"):
        torch.vmap(lambda x: read(cache, x))(_twice(plan.slots))
    assert torch.equal(read(cache, plan.slots)[0], k)


@pytest.mark.parametrize("what", ["starts", "lens", "table", "q"])
def test_attend(what):
    cache, plan, q, _, _, want = _state()
    given = dict(starts=plan.starts, lens=plan.lens, table=plan.table, q=q)

    def call(x):
        g = dict(given, **{what: x})
        return attend(g["q"], cache, StepPlan(starts=g["starts"], lens=g["lens"], table=g["table"], max_new=3))
    with pytest.raises(RuntimeError, match="data pointer|storage"):
        torch.vmap(call)(_twice(given[what]))
    assert torch.equal(attend(q, cache, plan), want)


def test_without_the_module(monkeypatch):
    *_, want = _state()

    def missing():
        raise RuntimeError("mimo_stream/_calls.so is not built")
    monkeypatch.setattr(_lib, "calls", missing)
    with pytest.warns(RuntimeWarning, match="_calls.so is not built"):
        cache, plan, q, k, _, got = _state()
    assert cache._call is None and torch.equal(got, want) and torch.equal(read(cache, plan.slots)[0], k)
