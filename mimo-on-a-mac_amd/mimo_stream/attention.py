"""The core of a decoder layer's attention half, over a paged K/V cache shared by many requests.

  PageTable.step(target)       request lengths -> page tables, slots and positions of the new tokens, on the device
  append(cache, plan, k, v, q) rotary positions on q and k, K and V written to their slots (bf16 or E4M3)
  attend(q, cache, plan)       attention of the new tokens over the cache: causal, grouped heads, sliding window, first
                               tokens that stay visible, sink logits

The reference's Attention (engine/mimo_stream/mimo_v2.py:66-150: full and sliding-window layers, sinks, partial RoPE)
runs on one request's KVCache / RotatingKVCache (engine/mimo_stream/model.py:169-170).  Here one step serves a whole
batch: requests decoding one token and requests with a chunk of new tokens, in one call each.  Lengths and tables stay on
the device, nothing synchronises, and every call can be captured into a HIP graph; a step's one plan serves every layer.
"""
import math
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib

E4M3 = torch.float8_e4m3fn

STATUS_MESSAGES = {_lib.ERR_PAGES: "fewer free pages than the step needs",
                   _lib.ERR_SHAPE: "request lengths outside the page table, the step's rows or max_new",
                   _lib.ERR_SLOT: "a page or slot outside the cache"}


def _device(device):
    device = torch.device(device)
    return torch.device("cuda", torch.cuda.current_device()) if device.type == "cuda" and device.index is None else device


def _same_device(dev, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{name} on {t.device}, expected {dev}")


def _int32(t, dev, shape, name):
    """The int32 device tensor that a kernel reads or writes in place: checked, never converted."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or not t.is_contiguous() or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: need a contiguous int32 tensor of shape {tuple(shape)}")
    _same_device(dev, **{name: t})
    return t


@dataclass
class StepPlan:
    """What one step's calls share.  append needs slots and positions; attend starts, lens, table and max_new.

    starts [B + 1]: request b's new tokens are rows starts[b] .. starts[b + 1] - 1; lens [B]: lengths with them; slots,
    positions [N] of the rows (-1 and 0 behind the last); table [B, max_pages]; n_free [1]; status [1]: the step's device
    status, to which append and attend add theirs."""
    starts: Optional[torch.Tensor] = None
    lens: Optional[torch.Tensor] = None
    slots: Optional[torch.Tensor] = None
    positions: Optional[torch.Tensor] = None
    table: Optional[torch.Tensor] = None
    max_new: Optional[int] = None
    n_free: Optional[torch.Tensor] = None
    status: Optional[torch.Tensor] = None

    def check(self, what="step"):
        """Raise ValueError if the step, or an append or attend of its plan, found a failure (synchronises)."""
        code = 0 if self.status is None else int(self.status.item())
        if code != _lib.MIMO_OK:
            raise ValueError(f"{what}: {STATUS_MESSAGES.get(code, 'device error')} (code {code})")


class PageTable:
    """Lengths, page tables and the free pages of up to max_seqs requests, on the device.

    One PageTable serves every layer whose caches have its pages.  All state is plain tensors: lens int32 [max_seqs], table
    int32 [max_seqs, max_pages], free int32 [n_pages] (a stack), n_free int32 [1]."""

    def __init__(self, max_seqs, max_pages, n_pages, page_size, device="cuda"):
        dev = _device(device)
        if max_seqs < 1 or max_pages < 1 or n_pages < 1:
            raise ValueError("need at least one request, one page per request and one page")
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two from 16 to 1024")
        self.page_size = int(page_size)
        self.n_pages = int(n_pages)
        self.lens = torch.zeros(max_seqs, dtype=torch.int32, device=dev)
        self.table = torch.zeros((max_seqs, max_pages), dtype=torch.int32, device=dev)
        self.free = torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device=dev)     # page 0 is taken first
        self.n_free = torch.full((1,), n_pages, dtype=torch.int32, device=dev)

    def step(self, target, n_tokens, max_new=None, commit=True):
        """Bring every request to target[b] tokens (int32 [max_seqs]; 0 ends a request, fewer takes tokens back).

        n_tokens: rows of the step, at least the sum of new tokens (more: the rows behind are padding); max_new: at most
        this many new tokens on one request (default n_tokens).  With commit=False the page table keeps its lengths and
        free pages, and the step can be dropped or made again.  Returns a StepPlan; a failure (too few free pages, lengths
        out of range) leaves the state as it was and is in plan.status (plan.check() raises)."""
        dev = self.lens.device
        B, width = self.table.shape
        _lib.require_cuda(self.lens)
        target = _int32(target, dev, (B,), "target")
        n_tokens = int(n_tokens)
        if n_tokens < 0:
            raise ValueError("n_tokens must be >= 0")
        max_new = n_tokens if max_new is None else int(max_new)
        with torch.cuda.device(dev):
            out = torch.empty(2 * B + 3 + 2 * n_tokens, dtype=torch.int32, device=dev)
            lens, n_free, status, starts, slots, positions = out.split([B, 1, 1, B + 1, n_tokens, n_tokens])
            _lib.call("mimo_cache_step", _lib.ptr(self.lens), _lib.ptr(target), B, _lib.ptr(self.table), width,
                      _lib.ptr(self.free), _lib.ptr(self.n_free), self.n_pages, self.page_size, n_tokens, max_new,
                      _lib.ptr(lens), _lib.ptr(n_free), _lib.ptr(starts), _lib.ptr(slots), _lib.ptr(positions),
                      _lib.ptr(self.lens if commit else None), _lib.ptr(self.n_free if commit else None), _lib.ptr(status),
                      _lib.stream_ptr(dev))
        return StepPlan(starts=starts, lens=lens, slots=slots, positions=positions, table=self.table, max_new=max_new,
                        n_free=n_free, status=status)


class KVCache:
    """One layer's K/V pages: k [n_pages, kv_heads, page_size, k_dim] and v [..., v_dim], bf16 or float8_e4m3fn with one
    fp32 scale per K/V head (a stored value stands for value * scale).  Head dimensions 64/64, 128/128 or 192/128."""

    def __init__(self, n_pages, page_size, kv_heads, k_dim, v_dim, dtype=torch.bfloat16, k_scale=None, v_scale=None,
                 device="cuda"):
        dev = _device(device)
        self._bind(torch.zeros((n_pages, kv_heads, page_size, k_dim), dtype=torch.uint8 if dtype == E4M3 else dtype, device=dev),
                   torch.zeros((n_pages, kv_heads, page_size, v_dim), dtype=torch.uint8 if dtype == E4M3 else dtype, device=dev),
                   k_scale, v_scale, dtype)

    @classmethod
    def of(cls, k, v, k_scale=None, v_scale=None):
        """A cache over existing page tensors (not copied)."""
        self = cls.__new__(cls)
        self._bind(k, v, k_scale, v_scale, k.dtype)
        return self

    def _bind(self, k, v, k_scale, v_scale, dtype):
        if dtype not in (torch.bfloat16, E4M3):
            raise ValueError("a K/V cache holds bfloat16 or float8_e4m3fn")
        if k.dtype == torch.uint8:
            k, v = k.view(dtype), v.view(dtype)
        if k.dim() != 4 or v.dim() != 4 or k.shape[:3] != v.shape[:3] or v.dtype != dtype:
            raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must be [pages, kv_heads, page_size, dim] of one type")
        if not k.is_contiguous() or not v.is_contiguous():
            raise ValueError("cache pages must be contiguous")
        n_pages, heads, page, k_dim = k.shape
        if page < 16 or page > 1024 or page & (page - 1):
            raise ValueError("page_size must be a power of two from 16 to 1024")
        if (k_dim, v.shape[3]) not in ((64, 64), (128, 128), (192, 128)):
            raise ValueError(f"head dimensions {k_dim} / {v.shape[3]}: 64/64, 128/128 and 192/128 are supported")
        if dtype == E4M3:
            if k_scale is None or v_scale is None:
                raise ValueError("an E4M3 cache needs k_scale and v_scale")
            k_scale, v_scale = (torch.as_tensor(s, dtype=torch.float32, device=k.device).expand(heads).contiguous()
                                for s in (k_scale, v_scale))
        elif k_scale is not None or v_scale is not None:
            raise ValueError("scales belong to an E4M3 cache")
        self.k, self.v, self.k_scale, self.v_scale, self.dtype = k, v, k_scale, v_scale, dtype
        self.kv_heads, self.k_dim, self.v_dim, self.page_size, self.n_pages = heads, k_dim, v.shape[3], page, n_pages

    def struct(self):
        return _lib.MimoKvCache(_lib.ptr(self.k), _lib.ptr(self.v), _lib.ptr(self.k_scale), _lib.ptr(self.v_scale),
                                1 if self.dtype == E4M3 else 0, self.n_pages, self.page_size, self.kv_heads, self.k_dim,
                                self.v_dim)


class Rotary:
    """Rotary positions on the first `dim` dimensions of a head (a multiple of 16), pairs (i, i + dim / 2), frequencies
    theta ** (-2 i / dim); kept as fp64 turns per position, so that far positions keep their fraction."""

    def __init__(self, dim, theta=10000.0, device="cuda"):
        if dim < 16 or dim % 16 or dim > 256:
            raise ValueError("the rotary dimension must be a multiple of 16 up to 256")
        if not theta > 0.0:
            raise ValueError("theta must be positive")
        self.dim = int(dim)
        i = torch.arange(0, dim, 2, dtype=torch.float64)
        self.turns = (float(theta) ** (-i / dim) / (2.0 * math.pi)).to(_device(device))


def _rows(x, dev, heads, dim, name):
    """x as bf16 rows the kernels can read: [N, heads, dim] with contiguous, 16-byte aligned tokens at any distance."""
    if not isinstance(x, torch.Tensor) or x.dim() != 3 or x.shape[2] != dim or (heads is not None and x.shape[1] != heads):
        raise ValueError(f"{name}: need [tokens, {'heads' if heads is None else heads}, {dim}]"
                         + (f", got {tuple(x.shape)}" if isinstance(x, torch.Tensor) else ""))
    _lib.require_cuda(x)
    _same_device(dev, **{name: x})
    x = x.to(torch.bfloat16)
    if x.stride(2) != 1 or x.stride(1) != dim or x.stride(0) % 8 or x.stride(0) < x.shape[1] * dim or x.data_ptr() % 16:
        x = x.contiguous()
        if x.data_ptr() % 16:
            x = x.clone()
    return x


def append(cache, plan, k, v, q=None, rotary=None):
    """Write the new tokens' k [N, kv_heads, k_dim] and v [N, kv_heads, v_dim] to plan.slots (rows with slot -1 are left
    out), k rotated to plan.positions; returns q [N, heads, k_dim] rotated likewise (None without q).  q, k and v may be
    views of one projection's rows."""
    dev = cache.k.device
    _lib.require_cuda(cache.k)
    k = _rows(k, dev, cache.kv_heads, cache.k_dim, "k")
    v = _rows(v, dev, cache.kv_heads, cache.v_dim, "v")
    N = k.shape[0]
    if v.shape[0] != N:
        raise ValueError(f"{N} tokens of k, {v.shape[0]} of v")
    slots = _int32(plan.slots, dev, (N,), "plan.slots")
    positions = _int32(plan.positions, dev, (N,), "plan.positions")
    _same_device(dev, status=plan.status)
    dim = 0
    if rotary is not None:
        dim = rotary.dim
        if dim > cache.k_dim:
            raise ValueError(f"rotary dimension {dim} past the head's {cache.k_dim}")
        _same_device(dev, rotary=rotary.turns)
    out, heads = None, 0
    if q is not None:
        q = _rows(q, dev, None, cache.k_dim, "q")
        if q.shape[0] != N:
            raise ValueError(f"{N} tokens of k, {q.shape[0]} of q")
        heads = q.shape[1]
        out = torch.empty((N, heads, cache.k_dim), dtype=torch.bfloat16, device=dev)
    if N == 0:
        return out
    with torch.cuda.device(dev):
        _lib.call("mimo_cache_append", _lib.ptr(q), 0 if q is None else q.stride(0), heads, _lib.ptr(k), k.stride(0),
                  _lib.ptr(v), v.stride(0), N, _lib.ptr(positions), _lib.ptr(slots), cache.struct(), dim,
                  _lib.ptr(None if rotary is None else rotary.turns), _lib.ptr(out), _lib.ptr(plan.status),
                  _lib.stream_ptr(dev))
    return out


def _workspace(nbytes, dev):
    """A workspace of this call's own in a captured graph (two graphs never share one), else the stream's cached one."""
    if torch.cuda.is_current_stream_capturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=dev)
    return _lib.workspace(nbytes, dev, "attend")


def attend(q, cache, plan, scale=None, window=0, sink_tokens=0, sink_logits=None, out=None):
    """Attention of the new tokens q [N, heads, k_dim] over the cache, which holds their keys and values already (append).

    A token at position p sees its request's keys j <= p; with window > 0 those with p - j < window, and the first
    sink_tokens.  scale defaults to k_dim ** -0.5.  sink_logits fp32 [heads]: a logit that joins each row's softmax without
    a value.  Returns bf16 [N, heads, v_dim] (out, if given: contiguous bf16); rows of no request are 0."""
    dev = cache.k.device
    _lib.require_cuda(cache.k)
    q = _rows(q, dev, None, cache.k_dim, "q")
    N, heads = q.shape[:2]
    if heads < 1 or heads % cache.kv_heads:
        raise ValueError(f"{heads} heads on {cache.kv_heads} K/V heads")
    if plan.table is None or plan.table.dim() != 2:
        raise ValueError("the plan has no page table")
    B, width = plan.table.shape
    table = _int32(plan.table, dev, (B, width), "plan.table")
    starts = _int32(plan.starts, dev, (B + 1,), "plan.starts")
    lens = _int32(plan.lens, dev, (B,), "plan.lens")
    _same_device(dev, status=plan.status)
    if window < 0 or sink_tokens < 0:
        raise ValueError("window and sink_tokens must be >= 0")
    if sink_logits is not None:
        if tuple(sink_logits.shape) != (heads,):
            raise ValueError(f"sink_logits of shape {tuple(sink_logits.shape)} for {heads} heads")
        _same_device(dev, sink_logits=sink_logits)
        sink_logits = sink_logits.to(torch.float32).contiguous()
    shape = (N, heads, cache.v_dim)
    if out is None:
        out = torch.empty(shape, dtype=torch.bfloat16, device=dev)
    elif out.dtype != torch.bfloat16 or tuple(out.shape) != shape or not out.is_contiguous() or out.device != dev:
        raise ValueError(f"out: need a contiguous bf16 tensor of shape {shape} on {dev}")
    if N == 0:
        return out
    scale = cache.k_dim ** -0.5 if scale is None else float(scale)
    max_new = N if plan.max_new is None else min(N, int(plan.max_new))
    with torch.cuda.device(dev):
        nbytes = _lib.load().mimo_cache_attend_workspace_size(N, heads, cache.kv_heads, cache.v_dim)
        ws = _workspace(nbytes, dev)
        _lib.call("mimo_cache_attend", _lib.ptr(q), q.stride(0), N, heads, cache.struct(), B, _lib.ptr(starts), _lib.ptr(lens),
                  _lib.ptr(table), width, max_new, scale, int(window), int(sink_tokens), _lib.ptr(sink_logits), _lib.ptr(out),
                  _lib.ptr(plan.status), _lib.ptr(ws), ws.numel(), _lib.stream_ptr(dev))
    return out
