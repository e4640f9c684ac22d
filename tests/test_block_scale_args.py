"""Refusals of the cache with block scales, of the rotary forms and of read, without a GPU."""
import copy
import ctypes
import math
import os
import pickle

import pytest
import torch

from mimo_stream import KVCache, PageTable, Rotary, StepPlan, _lib, append, attend, read, stretched

pytestmark = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="libmimo_moe.so not built")

E4M3 = torch.float8_e4m3fn
BF = torch.bfloat16


def test_block_scaled_cache_arguments():
    c = KVCache(3, 32, 2, 64, 64, dtype=E4M3, block_scales=True, device="cpu")
    assert c.block_scales and c.k_scale.shape == (3, 2, 2) and c.k_scale.dtype == torch.uint8 and c.k.dtype == E4M3
    again = KVCache.of(c.k, c.v, c.k_scale, c.v_scale.view(torch.float8_e8m0fnu))
    assert again.block_scales and again.v_scale.data_ptr() == c.v_scale.data_ptr()
    assert not KVCache(3, 32, 2, 64, 64, dtype=E4M3, k_scale=1.0, v_scale=1.0, device="cpu").block_scales
    with pytest.raises(ValueError):
        KVCache(3, 32, 2, 64, 64, block_scales=True, device="cpu")             # bf16
    with pytest.raises(ValueError, match="makes its own"):
        KVCache(3, 32, 2, 64, 64, dtype=E4M3, k_scale=1.0, v_scale=1.0, block_scales=True, device="cpu")
    for page in (8, 0, 24):
        with pytest.raises(ValueError):
            KVCache(3, page, 2, 64, 64, dtype=E4M3, block_scales=True, device="cpu")
    with pytest.raises(ValueError, match="two kinds"):
        KVCache.of(c.k, c.v, c.k_scale, 1.0)
    with pytest.raises(ValueError, match="overlap"):
        KVCache.of(c.k, c.v, c.k_scale, c.k_scale)
    for bad in (c.k_scale[:, :, :1], c.k_scale.float(), c.k_scale.transpose(0, 1), torch.zeros(13, dtype=torch.uint8)[1:].view(3, 2, 2)):
        with pytest.raises(ValueError, match="block scales"):
            KVCache.of(c.k, c.v, bad, c.v_scale)


def test_rotary_forms_arguments():
    r = Rotary(64, device="cpu", interleaved=True, frequencies=stretched(64, 10000.0, 4.0, 4096), magnitude=1.25)
    assert r.interleaved and r.magnitude == 1.25 and r.turns.shape == (32,) and r.turns.dtype == torch.float64
    assert torch.equal(Rotary(32, device="cpu").turns, Rotary(32, device="cpu", frequencies=stretched(32, 10000.0, 1.0, 4096)).turns)
    for bad in (torch.ones(31), [1.0] * 33, [math.nan] * 32, [math.inf] + [1.0] * 31):
        with pytest.raises(ValueError, match="frequencies"):
            Rotary(64, device="cpu", frequencies=bad)
    for bad in (math.nan, math.inf, 1e300):
        with pytest.raises(ValueError, match="magnitude"):
            Rotary(64, device="cpu", magnitude=bad)
    with pytest.raises(AttributeError):
        r.turns = torch.zeros(32)


@pytest.mark.parametrize("bad", [dict(dim=0), dict(dim=15), dict(theta=1.0), dict(factor=0.0), dict(original=0), dict(few=0.0), dict(few=32.0),
                                 dict(factor=math.nan)])
def test_stretched_arguments(bad):
    with pytest.raises(ValueError):
        stretched(**{**dict(dim=64, theta=10000.0, factor=2.0, original=4096), **bad})


@pytest.mark.parametrize("again", [copy.copy, copy.deepcopy, lambda r: pickle.loads(pickle.dumps(r))])
def test_rotary_is_copied_and_saved(again):
    r = Rotary(64, 5000.0, device="cpu", interleaved=True, magnitude=0.75)
    c = again(r)
    assert (c.dim, c.interleaved, c.magnitude) == (64, True, 0.75) and torch.equal(c.turns, r.turns)
    s = c._struct                                          # what the kernels are given: the copy's own numbers
    assert (s.turns, s.dim, s.interleaved, s.magnitude) == (c.turns.data_ptr(), 64, 1, 0.75) and c._at == ctypes.addressof(s)
    before = Rotary.__new__(Rotary)                        # saved when there was one form
    before.__setstate__({"dim": 64, "turns": r.turns})
    assert (before.dim, before.interleaved, before.magnitude) == (64, False, 1.0)


@pytest.mark.parametrize("name,value", [("dim", 32), ("interleaved", True), ("magnitude", 2.0), ("turns", torch.zeros(32))])
def test_rotary_is_fixed(name, value):
    with pytest.raises(AttributeError):                    # and not a change that the kernels would not see
        setattr(Rotary(64, device="cpu"), name, value)


def test_slots_of_a_request():
    pt = PageTable(2, 3, 8, 16, device="cpu")
    pt.table.copy_(torch.tensor([[0, 0, 0], [5, 2, 7]], dtype=torch.int32))
    assert pt.slots(1, 48).tolist() == [5 * 16 + i for i in range(16)] + [2 * 16 + i for i in range(16)] + [7 * 16 + i for i in range(16)]
    assert pt.slots(1, 33, 15).tolist() == [95] + list(range(32, 48)) + [112] and pt.slots(0, 0).tolist() == []
    assert pt.slots(1, 3).dtype == torch.int32
    for bad in ((2, 1), (-1, 1), (0, 49), (0, 3, 4), (0, 3, -1)):
        with pytest.raises(ValueError):
            pt.slots(*bad)


def test_cpu_tensors_are_refused():
    c = KVCache(3, 16, 2, 64, 64, dtype=E4M3, block_scales=True, device="cpu")
    one = torch.zeros(1, dtype=torch.int32)
    plan = StepPlan(starts=torch.zeros(2, dtype=torch.int32), lens=one, table=one[None], slots=one, positions=one)
    x = torch.zeros(1, 2, 64, dtype=BF)
    for call in (lambda: append(c, plan, x, x), lambda: attend(x, c, plan), lambda: read(c, one)):
        with pytest.raises(ValueError, match="device tensors"):
            call()


# ---- the C entries check on the host before any HIP call
HOST = ctypes.create_string_buffer(1 << 16)
ADDR = (ctypes.addressof(HOST) + 255) // 256 * 256
OUT = ADDR + 32768


def _kv(**kw):
    f = dict(k=ADDR, v=ADDR, k_scale=ADDR, v_scale=ADDR + 16, dtype=2, n_pages=2, page_size=16, kv_heads=2, k_dim=64, v_dim=64)
    f.update(kw)
    return _lib.MimoKvCache(*(f[n] for n, _ in _lib.MimoKvCache._fields_))


def _append(cache=None, rotary=(ADDR, 16, 0, 1.0), **kw):
    f = dict(q=ADDR, qs=128, heads=2, k=ADDR, ks=128, v=ADDR, vs=128, N=1, positions=ADDR, slots=ADDR, cache=cache or _kv(),
             rotary=None if rotary is None else _lib.MimoRotary(*rotary), q_out=OUT, status=None, stream=None)
    f.update(kw)
    return _lib.load().mimo_cache_append_rotary(*f.values())


@pytest.mark.parametrize("bad,code", [(dict(rotary=(None, 16, 0, 1.0)), "ARG"), (dict(rotary=(ADDR, 24, 0, 1.0)), "SHAPE"), (dict(rotary=(ADDR, 80, 1, 1.0)), "SHAPE"),
                                      (dict(rotary=(ADDR, 16, 2, 1.0)), "ARG"), (dict(rotary=(ADDR, 16, 0, math.nan)), "ARG"), (dict(rotary=(ADDR, 16, 1, math.inf)), "ARG"),
                                      (dict(N=-1), "SHAPE"), (dict(N=(1 << 23) - 16), "SHAPE"), (dict(k=None), "ARG"), (dict(q_out=None), "ARG"),
                                      (dict(vs=132), "ALIGN"), (dict(q_out=ADDR), "ARG")])
def test_append_refusals(bad, code):
    assert _append(**bad) == getattr(_lib, "ERR_" + code)


BAD_CACHES = [(dict(k_scale=None), "ARG"), (dict(v_scale=None), "ARG"), (dict(dtype=3), "ARG"), (dict(dtype=-1), "ARG"), (dict(k_scale=ADDR + 4), "ALIGN"),
              (dict(v_scale=ADDR + 1), "ALIGN"), (dict(v_scale=ADDR), "ARG"), (dict(v_scale=ADDR + 16, n_pages=9), "ARG"), (dict(page_size=8), "SHAPE"), (dict(v_dim=128), "SHAPE"), (dict(k=None), "ARG")]


def _read(cache=None, **kw):
    f = dict(cache=cache or _kv(), slots=ADDR, N=1, k=OUT, v=OUT + 1024, status=None, stream=None)
    f.update(kw)
    return _lib.load().mimo_cache_read(*f.values())


@pytest.mark.parametrize("bad,code", [(dict(slots=None), "ARG"), (dict(k=None), "ARG"), (dict(v=None), "ARG"), (dict(N=-1), "SHAPE"), (dict(N=1 << 24), "SHAPE"),
                                      (dict(k=OUT + 8), "ALIGN"), (dict(v=OUT + 2), "ALIGN"), (dict(k=ADDR), "ARG"), (dict(v=ADDR + 4080), "ARG"),
                                      (dict(v=OUT + 240), "ARG"), (dict(slots=OUT + 16), "ARG")])
def test_read_refusals(bad, code):
    assert _read(**bad) == getattr(_lib, "ERR_" + code)


@pytest.mark.parametrize("dtype", [_lib.KV_E4M3, _lib.KV_E4M3_BLOCKS])
@pytest.mark.parametrize("scales", [dict(k_scale=OUT), dict(v_scale=OUT), dict(k_scale=OUT + 1024 + 240), dict(v_scale=OUT + 1024)])
def test_read_refuses_outputs_over_scales(dtype, scales):
    assert _read(_kv(dtype=dtype, **scales)) == _lib.ERR_ARG


@pytest.mark.parametrize("bad,code", BAD_CACHES)
def test_cache_refusals(bad, code):
    assert _append(_kv(**bad)) == getattr(_lib, "ERR_" + code)
    assert _read(_kv(**bad)) == getattr(_lib, "ERR_" + code)


def test_empty_calls_need_no_gpu():
    assert _append(N=0) == 0 and _append(N=0, rotary=None) == 0 and _read(N=0) == 0


def test_what_a_slot_failure_may_be():
    """A plan whose slots are all inside the cache, but not together, is not told that one is outside alone."""
    plan = StepPlan(status=torch.tensor([_lib.ERR_SLOT], dtype=torch.int32))
    for part in ("outside the cache", "a slot written twice", "that others part"):
        with pytest.raises(ValueError, match=part):
            plan.check("append")
