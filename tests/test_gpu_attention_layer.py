"""The attention half of a decoder layer (AttentionLayer) alone, and with the MoE half (MoELayer), over steps of a paged cache."""
import numpy as np
import pytest
import torch

from helpers import rand_bf16, to_dev_bf16
from mimo_stream import AttentionLayer, KVCache, MoEBlock, MoELayer, PageTable, Rotary, Router, _lib, append, attend, pools
from oracle import attention as oa, layer as ol, mxfp4 as oq

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


def _one_of(rng, rows, cols, keep):
    """[rows, cols] with +-1 or +-0.5 at one place of each kept row: products with it are exact."""
    w = np.zeros((rows, cols), np.float32)
    at = np.flatnonzero(keep)
    w[at, rng.integers(0, cols, len(at))] = rng.choice([1.0, -1.0, 0.5, -0.5], len(at))
    return w


@pytest.mark.parametrize("window,sinks,logits", [(0, 0, False), (24, 2, True)])
def test_layer_matches_oracle(rng, window, sinks, logits):
    """The layer over steps of chunks and single tokens against attention over each whole sequence in 64 bits.

    The projections' weights have one value in a row, so q, k and v before the rotation, and y from o, are exact; q and k
    have 12 dimensions, 8 of them rotated.  A rotated value is off by e = 2^-20 (|a| + |b|) + 2^-8 |x| (its 32-bit pair and its
    rounding), a score therefore by d = scale sum(e_q |k| + |q| e_k + e_q e_k), a weight relative to the others by a factor of
    at most exp(2 d), d the row's largest; then attend's own 2^-8 |o| + (2^-8 + 2^-11) of the weighted mean of |v|, and the
    rounding of h, 2^-8 of it."""
    rot, theta, eps = 64, 10000.0, 1e-5
    used = np.zeros(DK, bool)
    used[[0, 1, 9, 20, 32, 33, 41, 52, 64, 70, 100, 191]] = True
    wq = _one_of(rng, HEADS * DK, H, np.tile(used, HEADS))
    wk, wv = _one_of(rng, KV * DK, H, np.tile(used, KV)), _one_of(rng, KV * DV, H, np.ones(KV * DV, bool))
    wo = _one_of(rng, H, HEADS * DV, np.ones(H, bool))
    norm = rand_bf16(rng, (H,), 0.1) + np.float32(1.0)
    norm = oq.round_bf16(norm)
    logit = rng.standard_normal(HEADS).astype(np.float32) if logits else None
    layer = AttentionLayer(to_dev_bf16(norm), eps, to_dev_bf16(np.concatenate([wq, wk, wv])), to_dev_bf16(wo), HEADS,
                           KVCache(64, PAGE, KV, DK, DV), rotary=Rotary(rot, theta), window=window, sink_tokens=sinks,
                           sink_logits=None if logit is None else torch.from_numpy(logit))
    pt = PageTable(2, 8, 64, PAGE)
    total, xs, hs = np.zeros(2, np.int64), [[], []], [[], []]
    for new in ([40, 7], [1, 1], [3, 20], [0, 1], [1, 1]):
        total = total + new
        x = rand_bf16(rng, (int(sum(new)), H))
        plan = pt.step(i32(total), len(x))
        h = layer(to_dev_bf16(x), plan).float().cpu().numpy().astype(np.float64)
        plan.check()
        for b, rows in enumerate((slice(0, new[0]), slice(new[0], None))):
            xs[b].append(x[rows]), hs[b].append(h[rows])
    for x, h in zip(xs, hs):
        x, h = np.concatenate(x), np.concatenate(h)
        L, at = len(x), np.arange(len(x))
        r = oq.bf16_bits_to_f32(ol.rmsnorm(oq.f32_to_bf16_bits(x), oq.f32_to_bf16_bits(norm), eps)).astype(np.float64)
        q0, k0, v = (r @ w.T.astype(np.float64) for w in (wq, wk, wv))
        q0, k0, v = q0.reshape(L, HEADS, DK), k0.reshape(L, KV, DK), v.reshape(L, KV, DV)
        q, k = oa.rotate(q0, at, rot, theta), oa.rotate(k0, at, rot, theta)

        def off(x0, x1):
            e = np.zeros_like(x1)
            pair = np.abs(x0[..., :rot // 2]) + np.abs(x0[..., rot // 2:rot])
            e[..., :rot] = 2.0 ** -20 * np.concatenate([pair, pair], -1) + 2.0 ** -8 * np.abs(x1[..., :rot])
            return e
        eq, ek = off(q0, q), off(k0, k)
        page = 1 << int(np.ceil(np.log2(L)))
        kp, vp = np.zeros((1, KV, page, DK)), np.zeros((1, KV, page, DV))
        kp[0, :, :L], vp[0, :, :L] = k.transpose(1, 0, 2), v.transpose(1, 0, 2)
        o, size = oa.attend(q, kp, vp, [0, L], [L], [[0]], DK ** -0.5, window, sinks, logit)
        seen = np.stack([oa.visible(p, L, window, sinks) for p in range(L)])
        G = HEADS // KV
        d = np.zeros((L, HEADS, 1))
        for n in range(HEADS):
            a, b, ea, eb = q[:, n], k[:, n // G], eq[:, n], ek[:, n // G]
            err = DK ** -0.5 * (ea @ np.abs(b).T + np.abs(a) @ eb.T + ea @ eb.T)
            d[:, n, 0] = np.where(seen, err, 0.0).max(axis=1)
        eo = np.expm1(2 * d) * size + 2.0 ** -8 * np.abs(o) + (2.0 ** -8 + 2.0 ** -11) * np.exp(2 * d) * size
        wide = wo.astype(np.float64).T
        want, e = x + o.reshape(L, -1) @ wide, eo.reshape(L, -1) @ np.abs(wide)
        tol = e + 2.0 ** -8 * (np.abs(want) + e)
        assert (np.abs(h - want) <= tol).all()
        kp[0, :, :L] = k0.transpose(1, 0, 2)             # what the tolerance tells apart: a layer that does not rotate
        o, _ = oa.attend(q0, kp, vp, [0, L], [L], [[0]], DK ** -0.5, window, sinks, logit)
        assert (np.abs(x + o.reshape(L, -1) @ wide - want) > tol).any()


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
