"""Refusals of the paged-cache operators that need no GPU: wrong shapes, types and devices never reach a launch."""
import ctypes
import os

import pytest
import torch

from mimo_stream import AttentionLayer, KVCache, PageTable, Rotary, StepPlan, _lib, append, attend

pytestmark = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="libmimo_moe.so not built")

BF = torch.bfloat16


def _cache(**kw):
    return KVCache(3, 16, 2, 64, 64, device="cpu", **kw)


def test_page_table_arguments():
    for bad in (dict(page_size=8), dict(page_size=48), dict(page_size=2048), dict(max_seqs=0), dict(max_pages=0), dict(n_pages=0)):
        with pytest.raises(ValueError):
            PageTable(**{**dict(max_seqs=2, max_pages=4, n_pages=8, page_size=16, device="cpu"), **bad})
    pt = PageTable(2, 4, 8, 16, device="cpu")
    assert pt.n_free.item() == 8 and sorted(pt.free.tolist()) == list(range(8))
    with pytest.raises(ValueError, match="device tensors"):
        pt.step(torch.zeros(2, dtype=torch.int32), 1)


def test_cache_arguments():
    with pytest.raises(ValueError):
        KVCache(3, 16, 2, 64, 128, device="cpu")
    with pytest.raises(ValueError):
        KVCache(3, 24, 2, 64, 64, device="cpu")
    with pytest.raises(ValueError):
        KVCache(3, 16, 2, 64, 64, dtype=torch.float16, device="cpu")
    with pytest.raises(ValueError, match="scale"):
        KVCache(3, 16, 2, 64, 64, dtype=torch.float8_e4m3fn, device="cpu")
    with pytest.raises(ValueError, match="scales"):
        _cache(k_scale=1.0, v_scale=1.0)
    c = KVCache(3, 16, 2, 64, 64, dtype=torch.float8_e4m3fn, k_scale=0.5, v_scale=[0.25, 1.0], device="cpu")
    assert c.k.dtype == torch.float8_e4m3fn and c.k_scale.tolist() == [0.5, 0.5] and c.v_scale.tolist() == [0.25, 1.0]
    k = torch.zeros(3, 2, 16, 64, dtype=BF)
    with pytest.raises(ValueError):
        KVCache.of(k, torch.zeros(3, 2, 32, 64, dtype=BF))
    with pytest.raises(ValueError, match="contiguous"):
        KVCache.of(k.transpose(1, 2).contiguous().transpose(1, 2), k)


def test_rotary_arguments():
    for dim in (0, 8, 24, 272):
        with pytest.raises(ValueError):
            Rotary(dim, device="cpu")
    with pytest.raises(ValueError):
        Rotary(64, theta=0.0, device="cpu")


def test_cpu_tensors_are_refused():
    c = _cache()
    plan = StepPlan(starts=torch.zeros(2, dtype=torch.int32), lens=torch.zeros(1, dtype=torch.int32),
                    table=torch.zeros(1, 1, dtype=torch.int32), slots=torch.zeros(1, dtype=torch.int32),
                    positions=torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="device tensors"):
        append(c, plan, torch.zeros(1, 2, 64, dtype=BF), torch.zeros(1, 2, 64, dtype=BF))
    with pytest.raises(ValueError, match="device tensors"):
        attend(torch.zeros(1, 2, 64, dtype=BF), c, plan)


def test_a_plan_of_other_pages_is_refused():
    c = _cache()
    plan = StepPlan(starts=torch.zeros(2, dtype=torch.int32), lens=torch.zeros(1, dtype=torch.int32),
                    table=torch.zeros(1, 1, dtype=torch.int32), slots=torch.zeros(1, dtype=torch.int32),
                    positions=torch.zeros(1, dtype=torch.int32), page_size=32)
    x = torch.zeros(1, 2, 64, dtype=BF)
    for call in (lambda: append(c, plan, x, x), lambda: attend(x, c, plan)):
        with pytest.raises(ValueError, match="pages of 32 tokens"):
            call()
    plan.page_size = 16                                  # the cache's: the next refusal is the CPU tensor's
    with pytest.raises(ValueError, match="device tensors"):
        attend(x, c, plan)


def test_numbers_past_32_bits_are_refused():
    """2^32 + 5 would reach the library as 5."""
    c = _cache()
    plan = StepPlan()
    x = torch.zeros(1, 2, 64, dtype=BF)
    for bad in (-1, 1 << 31, (1 << 32) + 5, -(1 << 32)):
        with pytest.raises(ValueError, match="window"):
            attend(x, c, plan, window=bad)
        with pytest.raises(ValueError, match="sink_tokens"):
            attend(x, c, plan, window=3, sink_tokens=bad)
    pt = PageTable(1, 4, 8, 16, device="cpu")
    target = torch.zeros(1, dtype=torch.int32)
    for bad in (-1, (1 << 20) + 1, (1 << 32) + 5):
        with pytest.raises(ValueError, match="n_tokens"):
            pt.step(target, bad)
    for bad in (-1, 1 << 31, 1 << 32, -(1 << 32)):
        with pytest.raises(ValueError, match="max_new"):
            pt.step(target, 4, max_new=bad)
    with pytest.raises(ValueError, match="slots"):
        PageTable(1, 4, (1 << 32) + 8, 16, device="cpu")


def test_layer_weights_leave_their_graph():
    """Parameters of a module may be given as they are: the layer shares their memory and builds no graph over them."""
    c = _cache()
    norm, qkv, o = (torch.nn.Parameter(torch.ones(shape, dtype=BF)) for shape in ((32,), (2 * 64 * 3, 32), (32, 128)))
    sinks = torch.nn.Parameter(torch.zeros(2))
    layer = AttentionLayer(norm, 1e-5, qkv, o, 2, c, sink_logits=sinks)
    for kept, given in ((layer.norm_weight, norm), (layer.qkv_weight, qkv), (layer.o_weight, o), (layer.sink_logits, sinks)):
        assert not kept.requires_grad and kept.data_ptr() == given.data_ptr()


# ---- the C entries check on the host before any HIP call
HOST = ctypes.create_string_buffer(4096)
ADDR = (ctypes.addressof(HOST) + 255) // 256 * 256
OUT = ADDR + 1024                                        # outputs that overlap no input


def _kv(**kw):
    f = dict(k=ADDR, v=ADDR, k_scale=None, v_scale=None, dtype=0, n_pages=4, page_size=16, kv_heads=2, k_dim=64, v_dim=64)
    f.update(kw)
    return _lib.MimoKvCache(*(f[n] for n, _ in _lib.MimoKvCache._fields_))


BAD_CACHES = [(dict(k=None), "ARG"), (dict(dtype=2), "ARG"), (dict(dtype=1), "ARG"), (dict(k_dim=96), "SHAPE"), (dict(v_dim=128), "SHAPE"),
              (dict(page_size=8), "SHAPE"), (dict(page_size=100), "SHAPE"), (dict(kv_heads=0), "SHAPE"), (dict(n_pages=0), "SHAPE"),
              (dict(n_pages=1 << 28), "SHAPE"), (dict(v=ADDR + 2), "ALIGN")]


def _step(**kw):
    f = dict(lens=ADDR, target=ADDR, B=1, table=ADDR, max_pages=1, free=ADDR, n_free=ADDR, n_pages=1, page_size=16, N=1, max_new=1,
             lens_out=ADDR + 64, n_free_out=ADDR + 64, starts=ADDR, slots=ADDR, positions=ADDR, cl=None, cn=None, status=ADDR, stream=None)
    f.update(kw)
    return _lib.load().mimo_cache_step(*f.values())


@pytest.mark.parametrize("bad,code", [(dict(lens=None), "ARG"), (dict(status=None), "ARG"), (dict(slots=None), "ARG"), (dict(B=0), "SHAPE"),
                                      (dict(B=4097), "SHAPE"), (dict(N=-1), "SHAPE"), (dict(N=(1 << 20) + 1), "SHAPE"),
                                      (dict(max_new=-1), "SHAPE"), (dict(page_size=17), "SHAPE"), (dict(n_pages=1 << 28), "SHAPE"),
                                      (dict(lens_out=ADDR), "ARG"), (dict(cl=ADDR), "ARG"), (dict(max_pages=1 << 28), "SHAPE")])
def test_step_refusals(bad, code):
    assert _step(**bad) == getattr(_lib, "ERR_" + code)


def _append(cache=None, **kw):
    f = dict(q=ADDR, qs=128, heads=2, k=ADDR, ks=128, v=ADDR, vs=128, N=1, positions=ADDR, slots=ADDR, cache=cache or _kv(), dim=16,
             turns=ADDR, q_out=OUT, status=None, stream=None)
    f.update(kw)
    return _lib.load().mimo_cache_append(*f.values())


@pytest.mark.parametrize("bad,code", [(dict(k=None), "ARG"), (dict(q_out=None), "ARG"), (dict(turns=None), "ARG"), (dict(dim=24), "SHAPE"),
                                      (dict(dim=80), "SHAPE"), (dict(N=-1), "SHAPE"), (dict(ks=120), "SHAPE"), (dict(vs=132), "ALIGN"),
                                      (dict(q=ADDR + 8), "ALIGN"), (dict(heads=0), "SHAPE"),
                                      (dict(q_out=ADDR), "ARG"), (dict(q=OUT, k=OUT + 256, q_out=OUT + 256), "ARG"), (dict(v=OUT + 240), "ARG")])
def test_append_refusals(bad, code):
    assert _append(**bad) == getattr(_lib, "ERR_" + code)


def _attend(cache=None, **kw):
    f = dict(q=ADDR, qs=128, N=1, heads=2, cache=cache or _kv(), B=1, starts=ADDR, lens=ADDR, table=ADDR, max_pages=1, max_new=1, scale=1.0,
             window=0, sinks=0, logits=None, out=OUT, status=None, ws=ADDR, bytes=1 << 40, stream=None)
    f.update(kw)
    return _lib.load().mimo_cache_attend(*f.values())


@pytest.mark.parametrize("bad,code", [(dict(q=None), "ARG"), (dict(table=None), "ARG"), (dict(heads=3), "SHAPE"), (dict(heads=0), "SHAPE"),
                                      (dict(N=-1), "SHAPE"), (dict(B=0), "SHAPE"), (dict(max_pages=0), "SHAPE"), (dict(window=-1), "SHAPE"),
                                      (dict(sinks=-1), "SHAPE"), (dict(scale=float("nan")), "ARG"), (dict(scale=float("inf")), "ARG"),
                                      (dict(qs=64), "SHAPE"), (dict(out=OUT + 8), "ALIGN"), (dict(ws=None), "WORKSPACE"),
                                      (dict(bytes=0), "WORKSPACE"), (dict(out=ADDR), "ARG"), (dict(out=ADDR + 240), "ARG"), (dict(B=(1 << 20) + 1), "SHAPE"),
                                      (dict(max_pages=1 << 27), "SHAPE"), (dict(N=(1 << 20) + 1), "SHAPE")])
def test_attend_refusals(bad, code):
    assert _attend(**bad) == getattr(_lib, "ERR_" + code)


FAR = 1 << 44                                            # far from every input


@pytest.mark.parametrize("kv,dims,B,max_pages", [(128, (128, 128), 1, 64), (1024, (64, 64), 1, 64), (64, (64, 64), 1 << 20, 1)])
def test_attend_refuses_more_blocks_than_a_launch_has(kv, dims, B, max_pages):
    """Rows to join, or row tiles over requests, past 2^24 blocks of 256 threads: refused before anything is queued."""
    N, cache = 1 << 20, _kv(kv_heads=kv, k_dim=dims[0], v_dim=dims[1], page_size=1024)
    heads = min(1024, 16 * kv) if B > 1 else kv
    rc = _attend(cache, N=N, heads=heads, qs=heads * dims[0], B=B, max_pages=max_pages, max_new=N, out=FAR)
    assert rc == _lib.ERR_SHAPE and b"row" in _lib.load().mimo_last_error()


def test_append_refuses_more_tokens_than_a_launch_has_blocks():
    assert _append(N=1 << 24, q_out=FAR) == _lib.ERR_SHAPE and b"2^24" in _lib.load().mimo_last_error()


@pytest.mark.parametrize("bad,code", BAD_CACHES)
def test_cache_refusals(bad, code):
    assert _append(_kv(**bad)) == getattr(_lib, "ERR_" + code)
    assert _attend(_kv(**bad)) == getattr(_lib, "ERR_" + code)


def test_empty_calls_need_no_gpu():
    assert _append(N=0) == 0 and _attend(N=0) == 0


def test_attend_workspace_never_falls():
    size = _lib.load().mimo_cache_attend_workspace_size
    for heads, kv, dv in ((64, 4, 128), (5, 5, 64), (64, 1, 128)):
        last = 0
        for n in list(range(1, 70)) + [127, 128, 129, 1000, 4096, 65536]:
            need = size(n, heads, kv, dv)
            assert need >= last
            last = need
