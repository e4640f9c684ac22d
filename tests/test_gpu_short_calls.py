"""append, read and attend through the short host path (csrc/calls.cpp) and the long one: the ordinary call takes the short
one, any other form the long one, and both give the same bits and raise the same refusals."""
import numpy as np
import pytest
import torch

from mimo_stream import KVCache, PageTable, Rotary, StepPlan, _lib, append, attend, attention, read

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
E4M3 = torch.float8_e4m3fn
HEADS, KV, DK, DV, PAGE = 6, 2, 192, 128, 16


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def _cache(kind):
    if kind == "bf16":
        return KVCache(8, PAGE, KV, DK, DV)
    return KVCache(8, PAGE, KV, DK, DV, dtype=E4M3, **(dict(block_scales=True) if kind == "blocks" else dict(k_scale=0.1, v_scale=0.2)))


def _rows(rng, N):
    return (torch.from_numpy(rng.standard_normal((N, h, d)).astype(np.float32)).to(BF).cuda() for h, d in ((HEADS, DK), (KV, DK), (KV, DV)))


def _pass(cache, pt, rng, long_way=False, **kw):
    if long_way:
        cache._call = None
    plan = pt.step(i32([20, 37]), 57)
    q, k, v = _rows(rng, 57)
    q = append(cache, plan, k, v, q=q, rotary=Rotary(64))
    out = attend(q, cache, plan, **kw)
    back = read(cache, plan.slots)
    plan.check()
    return q, out, *back


@pytest.mark.parametrize("kind", ["bf16", "heads", "blocks"])
@pytest.mark.parametrize("kw", [{}, dict(scale=0.05, window=20, sink_tokens=3)])
def test_both_ways_agree(kind, kw):
    got = [_pass(_cache(kind), PageTable(2, 4, 8, PAGE), np.random.default_rng(1), long_way, **kw) for long_way in (False, True)]
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_the_ordinary_call_takes_the_short_way(monkeypatch, rng):
    cache, pt = _cache("blocks"), PageTable(2, 4, 8, PAGE)
    _pass(cache, pt, rng)                                  # the stream's workspace is there now
    plan = pt.step(i32([21, 38]), 2)
    q, k, v = _rows(rng, 2)

    def long_way(name):
        raise AssertionError(f"{name} by the long way")
    monkeypatch.setattr(attention, "_entry", long_way)
    logits = torch.zeros(HEADS, device="cuda")
    q = append(cache, plan, k, v, q=q, rotary=Rotary(64, interleaved=True))
    assert append(cache, plan, k, v) is None
    out = torch.empty(2, HEADS, DV, dtype=BF, device="cuda")
    assert attend(q, cache, plan, out=out, sink_logits=logits) is out
    attend(q, cache, plan, scale=0.1, window=5, sink_tokens=1)
    read(cache, plan.slots, status=plan.status)


def test_other_forms_take_the_long_way(rng):
    """fp32 rows, rows of no alignment, int scale: converted as before, and as bf16 gives them."""
    cache, pt = _cache("heads"), PageTable(2, 4, 8, PAGE)
    _pass(cache, pt, rng)
    plan = pt.step(i32([21, 38]), 2)
    q, k, v = _rows(rng, 2)
    want = append(cache, plan, k, v, q=q)
    held = cache.k.view(torch.uint8).clone()
    odd = torch.zeros(2 * HEADS * DK + 1, dtype=BF, device="cuda")[1:].view(2, HEADS, DK).copy_(q)
    for form in (q.float(), odd, torch.nn.Parameter(q), q.transpose(0, 1).contiguous().transpose(0, 1)):
        assert torch.equal(append(cache, plan, k.float(), v, q=form), want)
    assert torch.equal(cache.k.view(torch.uint8), held)
    ref = attend(want, cache, plan, scale=1.0)
    assert torch.equal(attend(want.float(), cache, plan, scale=1), ref) and torch.equal(attend(want, cache, plan, scale=np.float32(1.0)), ref)
    assert torch.equal(attend(want, cache, plan, scale=1.0, sink_logits=torch.full((HEADS,), -1e30, dtype=torch.float64, device="cuda")), ref)


def test_refusals_are_the_same(rng):
    cache, pt = _cache("blocks"), PageTable(2, 4, 8, PAGE)
    _pass(cache, pt, rng)
    plan = pt.step(i32([21, 38]), 2)
    q, k, v = _rows(rng, 2)
    other = _cache("blocks")
    calls = [("slots", lambda: append(cache, StepPlan(slots=plan.slots.long(), positions=plan.positions), k, v)),
             ("slots", lambda: append(cache, StepPlan(positions=plan.positions), k, v)),
             ("tokens of k", lambda: append(cache, plan, k, v[:1])),
             ("k: need", lambda: append(cache, plan, v, v)),
             ("pages of 32", lambda: append(cache, StepPlan(slots=plan.slots, positions=plan.positions, page_size=32), k, v)),
             ("rotary dimension", lambda: append(cache, plan, k, v, rotary=Rotary(256))),
             ("rotary on cpu", lambda: append(cache, plan, k, v, rotary=Rotary(64, device="cpu"))),
             ("on cpu", lambda: append(cache, plan, k.cpu(), v)),
             ("status", lambda: append(cache, StepPlan(slots=plan.slots, positions=plan.positions, status=torch.zeros(2, dtype=torch.int32, device="cuda")), k, v)),
             ("overlap", lambda: attend(q, cache, plan, out=_over(q))),
             ("heads", lambda: attend(q[:, :3].contiguous(), cache, plan)),
             ("window", lambda: attend(q, cache, plan, window=-1)),
             ("window", lambda: attend(q, cache, plan, window=(1 << 32) + 5)),
             ("finite", lambda: attend(q, cache, plan, scale=float("nan"))),
             ("out", lambda: attend(q, cache, plan, out=torch.empty(2, HEADS, DK, dtype=BF, device="cuda"))),
             ("page table", lambda: attend(q, cache, StepPlan(starts=plan.starts, lens=plan.lens))),
             ("starts", lambda: attend(q, cache, StepPlan(starts=plan.starts[:2].contiguous(), lens=plan.lens, table=plan.table))),
             ("sink_logits", lambda: attend(q, cache, plan, sink_logits=torch.zeros(5, device="cuda"))),
             ("slots", lambda: read(cache, plan.slots.long())),
             ("slots", lambda: read(cache, plan.slots.cpu())),
             ("status", lambda: read(cache, plan.slots, status=torch.zeros(1, device="cuda")))]
    for match, call in calls:
        with pytest.raises(ValueError, match=match):
            call()
    before = cache._call
    cache._call = None
    for match, call in calls:
        with pytest.raises(ValueError, match=match):
            call()
    cache._call = before
    assert not other.k.float().any()


def _over(q):
    """An output in q's own memory."""
    return q.view(-1)[:2 * HEADS * DV].view(2, HEADS, DV)


def test_the_short_module_refuses_what_is_not_its_own():
    calls = _lib.calls()
    cache = _cache("bf16")
    assert calls.read(object(), 0, 0, i32([1]), None) is NotImplemented
    assert calls.read(cache._call, 1 << 70, 0, i32([1]), None) is NotImplemented
    assert calls.read(cache._call, 3, 0, i32([1]), None) is NotImplemented      # another current device
    assert calls.read(cache._call, 0, 0, None, None) is NotImplemented
    with pytest.raises(TypeError):
        calls.read(cache._call)
    with pytest.raises(TypeError):
        calls.cache("no address", 0)
