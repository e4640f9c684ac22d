"""The attention half of a decoder layer (AttentionLayer) alone, and with the MoE half (MoELayer), over steps of a paged cache."""
import numpy as np
import pytest
import torch

from helpers import rand_bf16, to_dev_bf16
from mimo_stream import AttentionLayer, KVCache, MoEBlock, MoELayer, PageTable, Rotary, Router, _lib, append, attend, pools

pytestmark = pytest.mark.gpu

H, HEADS, KV, DK, DV, PAGE = 512, 8, 2, 192, 128, 16


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def _layer(rng, window=0, sinks=0, logits=False, pages=64):
    cache = KVCache(pages, PAGE, KV, DK, DV)
    rows = HEADS * DK + KV * (DK + DV)
    return AttentionLayer(to_dev_bf16(rand_bf16(rng, (H,), 0.1) + 1.0), 1e-5, to_dev_bf16(rand_bf16(rng, (rows, H), H ** -0.5)),
                          to_dev_bf16(rand_bf16(rng, (H, HEADS * DV), (HEADS * DV) ** -0.5)), HEADS, cache, rotary=Rotary(64),
                          window=window, sink_tokens=sinks,
                          sink_logits=torch.from_numpy(rng.standard_normal(HEADS).astype(np.float32)) if logits else None)


def _moe(rng, seed=3):
    bank = pools.random_bank(8, seed=seed, hidden=H, inter=512)
    router = Router(H, 8, 2)
    router.weight.copy_(to_dev_bf16(rand_bf16(rng, (8, H), 0.02)))
    return MoELayer(MoEBlock(router, bank), to_dev_bf16(rand_bf16(rng, (H,), 0.1) + 1.0), 1e-5)


@pytest.mark.parametrize("window,sinks,logits", [(0, 0, False), (24, 2, True)])
def test_layer_is_its_pieces(rng, window, sinks, logits):
    """Bit for bit norm, projections, append, attend and residual, over steps of chunks and single tokens."""
    layer = _layer(rng, window, sinks, logits)
    pt = PageTable(2, 8, 64, PAGE)
    total = np.zeros(2, np.int64)
    for new in ([40, 7], [1, 1], [3, 20]):
        total = total + new
        N = int(sum(new))
        x = to_dev_bf16(rand_bf16(rng, (N, H)))
        plan = pt.step(i32(total), N)
        h = layer(x, plan)
        plan.check()
        # the cache rows are written again, with the same values
        r = torch.empty_like(x)
        _lib.call("mimo_rmsnorm", _lib.ptr(x), N, H, _lib.ptr(layer.norm_weight), 1e-5, _lib.ptr(r), _lib.stream_ptr(x.device))
        q, k, v = torch.matmul(r, layer.qkv_weight.T).split(layer.split, 1)
        q = append(layer.cache, plan, k.unflatten(1, (KV, DK)), v.unflatten(1, (KV, DV)), q=q.unflatten(1, (HEADS, DK)), rotary=layer.rotary)
        o = attend(q, layer.cache, plan, window=window, sink_tokens=sinks, sink_logits=layer.sink_logits)
        y = torch.matmul(o.flatten(1), layer.o_weight.T)
        want = torch.empty_like(x)
        _lib.call("mimo_residual_add", _lib.ptr(x), _lib.ptr(y), x.numel(), _lib.ptr(want), _lib.stream_ptr(x.device))
        assert torch.equal(h, want)


def test_decoder_layers_chunked_and_in_a_graph(rng):
    """Two decoder layers (attention and MoE halves), prompts in chunks and then tokens one by one from a captured graph: every
    replay equals the eager step of a second copy of the state bit for bit."""
    attn = [_layer(rng), _layer(rng, window=24, sinks=2, logits=True)]
    moe = [_moe(rng, 3), _moe(rng, 4)]
    B = 3
    prompt = to_dev_bf16(rand_bf16(rng, (60, H)))
    xs = [to_dev_bf16(rand_bf16(rng, (B, H))) for _ in range(5)]

    def forward(pt, x, target, max_new):
        plan = pt.step(target, x.shape[0], max_new=max_new)
        for a, m in zip(attn, moe):
            x = m(a(x, plan))
        return x, plan

    def prefill(pt):
        for target, rows in ([30, 9, 0], slice(0, 39)), ([40, 9, 11], slice(39, 60)):
            forward(pt, prompt[rows], i32(target), 30)[1].check()

    pt = PageTable(B, 16, 64, PAGE)
    prefill(pt)
    want = []
    for x in xs:
        out, plan = forward(pt, x, pt.lens + 1, 1)
        plan.check()
        want.append(out.clone())
    pt = PageTable(B, 16, 64, PAGE)                      # the same pages again: the caches are written anew
    prefill(pt)
    x = xs[0].clone()
    lens = pt.lens.clone()
    forward(pt, x, pt.lens + 1, 1)                       # warms the library GEMMs; then taken back
    pt.step(lens, 0).check()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, plan = forward(pt, x, pt.lens + 1, 1)
    for i, xi in enumerate(xs):
        x.copy_(xi)
        g.replay()
        torch.cuda.synchronize()
        assert plan.status.item() == 0 and torch.equal(out, want[i]), i
        _ = prompt @ prompt.T                            # eager work between replays


def test_layer_refusals(rng):
    layer = _layer(rng)
    pt = PageTable(1, 4, 8, PAGE)
    plan = pt.step(i32([2]), 2)
    x = to_dev_bf16(rand_bf16(rng, (2, H)))
    with pytest.raises(ValueError):
        layer(x[:, :256], plan)
    with pytest.raises(ValueError):
        layer(x.cpu(), plan)
    with pytest.raises(ValueError):
        layer(x[:1], plan)                               # the plan is for two rows
    assert layer(x[:0], plan).shape == (0, H)
    w = layer
    for bad in (dict(heads=3), dict(heads=4), dict(o_weight=w.o_weight.T), dict(eps=-1.0), dict(sink_logits=torch.zeros(3))):
        kw = dict(norm_weight=w.norm_weight, eps=1e-5, qkv_weight=w.qkv_weight, o_weight=w.o_weight, heads=HEADS, cache=w.cache)
        kw.update(bad)
        with pytest.raises(ValueError):
            AttentionLayer(**kw)
