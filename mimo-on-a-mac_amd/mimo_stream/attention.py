"""The core of a decoder layer's attention half, over a paged K/V cache shared by many requests.

  PageTable.step(target)       request lengths -> page tables, slots and positions of the new tokens, on the device
  append(cache, plan, k, v, q) rotary positions on q and k, K and V written to their slots (bf16 or E4M3)
  read(cache, slots)           cached tokens back as bf16 rows
  attend(q, cache, plan)       attention of the new tokens over the cache: causal, grouped heads, sliding window, first
                               tokens that stay visible, sink logits

The reference's Attention (engine/mimo_stream/mimo_v2.py:66-150: full and sliding-window layers, sinks, partial RoPE)
runs on one request's KVCache / RotatingKVCache (engine/mimo_stream/model.py:169-170).  Here one step serves a whole
batch: requests decoding one token and requests with a chunk of new tokens, in one call each.  Lengths and tables stay on
the device, nothing synchronises, and every call can be captured into a HIP graph; a step's one plan serves every layer.
For inference: no output carries a gradient.
"""
import ctypes
import functools
import math
import warnings
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib

E4M3 = torch.float8_e4m3fn
E8M0 = torch.float8_e8m0fnu
BF16 = torch.bfloat16
INT32 = torch.int32

STATUS_MESSAGES = {_lib.ERR_PAGES: "fewer free pages than the step needs",
                   _lib.ERR_SHAPE: "request lengths or starts outside the page table, the rows or max_new",
                   _lib.ERR_SLOT: "a page or slot outside the cache, or, with block scales, a slot written twice or rows of a block of "
                                  "16 slots that others part"}

# A decode step makes one step call and two calls per layer, each of a few microseconds on the GPU: what they do on the host
# is kept short.  append, read and attend hand a call to _lib.calls() first, which takes it in its ordinary form (csrc/calls.cpp)
# and answers NotImplemented for any other: then what stands here checks and converts the arguments one by one.
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_capturing = torch.cuda.is_current_stream_capturing


INT32_MAX = 0x7FFFFFFF                                   # ctypes takes the low bits of larger numbers without a word


def _taken(code, name):
    """What a short path answered, if it made the call; a code of the library's raises."""
    if type(code) is int:
        _lib.check(code, name)
    return code


def _device(device):
    device = torch.device(device)
    return torch.device("cuda", torch.cuda.current_device()) if device.type == "cuda" and device.index is None else device


@functools.lru_cache(maxsize=None)
def _entry(name):
    return getattr(_lib.load(), name)


def _gpu(dev):
    if dev.type != "cuda":
        raise ValueError("libmimo_moe works on device tensors; got a CPU tensor")
    return dev.index


def _int32(t, dev, shape, name):
    """Address of the int32 device tensor that a kernel reads or writes in place: checked, never converted."""
    if not (isinstance(t, torch.Tensor) and t.dtype is INT32 and t.device == dev and t.shape == shape and t.is_contiguous()):
        raise ValueError(f"{name}: need a contiguous int32 tensor of shape {tuple(shape)} on {dev}")
    return t.data_ptr()


def _same_pages(plan, cache):
    if plan.page_size is not None and plan.page_size != cache.page_size:
        raise ValueError(f"a plan of pages of {plan.page_size} tokens for a cache whose pages hold {cache.page_size}")


def _status(plan, dev):
    return None if plan.status is None else _int32(plan.status, dev, (1,), "plan.status")


@dataclass
class StepPlan:
    """What one step's calls share.  append needs slots and positions; attend starts, lens, table and max_new.

    starts [B + 1]: request b's new tokens are rows starts[b] .. starts[b + 1] - 1; lens [B]: lengths with them; slots,
    positions [N] of the rows (-1 and 0 behind the last); table [B, max_pages]; n_free [1]; status [1]: the step's device
    status, to which append and attend add theirs; page_size: of the slots and the table (None: not compared with the cache's)."""
    starts: Optional[torch.Tensor] = None
    lens: Optional[torch.Tensor] = None
    slots: Optional[torch.Tensor] = None
    positions: Optional[torch.Tensor] = None
    table: Optional[torch.Tensor] = None
    max_new: Optional[int] = None
    n_free: Optional[torch.Tensor] = None
    status: Optional[torch.Tensor] = None
    page_size: Optional[int] = None

    def check(self, what="step"):
        """Raise ValueError if the step, or an append or attend of its plan, found a failure (synchronises)."""
        code = 0 if self.status is None else int(self.status.item())
        if code != _lib.MIMO_OK:
            raise ValueError(f"{what}: {STATUS_MESSAGES.get(code, 'device error')} (code {code})")


class PageTable:
    """Lengths, page tables and the free pages of up to max_seqs requests, on the device.

    One PageTable serves every layer whose caches have its pages.  The state is int32 tensors, changed in place only: lens
    [max_seqs], table [max_seqs, max_pages], free [n_pages] (a stack), n_free [1]."""

    def __init__(self, max_seqs, max_pages, n_pages, page_size, device="cuda"):
        dev = _device(device)
        if max_seqs < 1 or max_pages < 1 or n_pages < 1:
            raise ValueError("need at least one request, one page per request and one page")
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two from 16 to 1024")
        if n_pages * page_size > INT32_MAX:
            raise ValueError(f"{n_pages} pages of {page_size} (at most 2^31 - 1 slots)")
        self.page_size = int(page_size)
        self.n_pages = int(n_pages)
        self._lens = torch.zeros(max_seqs, dtype=INT32, device=dev)
        self._table = torch.zeros((max_seqs, max_pages), dtype=INT32, device=dev)
        self._free = torch.arange(n_pages - 1, -1, -1, dtype=INT32, device=dev)     # page 0 is taken first
        self._n_free = torch.full((1,), n_pages, dtype=INT32, device=dev)

    lens = property(lambda self: self._lens)
    table = property(lambda self: self._table)
    free = property(lambda self: self._free)
    n_free = property(lambda self: self._n_free)

    def step(self, target, n_tokens, max_new=None, commit=True):
        """Bring every request to target[b] tokens (int32 [max_seqs]; 0 ends a request, fewer takes tokens back).

        n_tokens: rows of the step, at least the sum of new tokens (more: the rows behind are padding); max_new: at most
        this many new tokens on one request (default n_tokens).  With commit=False the page table keeps its lengths and
        free pages, and the step can be dropped or made again; after an append only if it gave no pages back (a request's
        pages that end in a step are the first that others take in it, and then hold their tokens).  In a cache with block
        scales an appended token leaves a trace even if its step is dropped or it is taken back: where it raised the scale of
        a block of 16 slots that older tokens share, these stay rounded to that scale's steps, and later tokens of the block
        get it too (KVCache).  Returns a StepPlan; a failure (too few free pages, lengths out of range) leaves the state as
        it was and is in plan.status (plan.check() raises)."""
        if not 0 <= n_tokens <= 1 << 20 or (max_new is not None and not 0 <= max_new <= INT32_MAX):
            raise ValueError(f"n_tokens must be from 0 to 2^20 and max_new from 0 to 2^31 - 1 (got {n_tokens}, {max_new})")
        dev = self._lens.device
        index = _gpu(dev)
        if _current_device() != index:
            with torch.cuda.device(dev):
                return self.step(target, n_tokens, max_new, commit)
        B, width = self._table.shape
        at_target = _int32(target, dev, (B,), "target")
        n_tokens = int(n_tokens)
        max_new = n_tokens if max_new is None else int(max_new)
        out = torch.empty(2 * B + 3 + 2 * n_tokens, dtype=INT32, device=dev)
        lens, n_free, status, starts, slots, positions = out.split_with_sizes((B, 1, 1, B + 1, n_tokens, n_tokens))
        at = out.data_ptr()
        at_starts = at + 4 * B + 8
        at_slots = at_starts + 4 * B + 4
        state, count = self._lens.data_ptr(), self._n_free.data_ptr()
        rc = _entry("mimo_cache_step")(
            state, at_target, B, self._table.data_ptr(), width, self._free.data_ptr(), count, self.n_pages, self.page_size,
            n_tokens, max_new, at, at + 4 * B, at_starts, at_slots, at_slots + 4 * n_tokens, state if commit else None,
            count if commit else None, at + 4 * B + 4, _raw_stream(index))
        if rc:
            _lib.check(rc, "mimo_cache_step")
        return StepPlan(starts, lens, slots, positions, self._table, max_new, n_free, status, self.page_size)

    def slots(self, request, stop, start=0):
        """int32 slots of a request's tokens start .. stop - 1, as its page table has them now (read takes them).  The request's
        length is on the device and is not looked at: tokens past it have slots of no meaning."""
        B, width = self._table.shape
        if not (0 <= request < B and 0 <= start <= stop <= width * self.page_size):
            raise ValueError(f"tokens {start} to {stop} of request {request}: {B} requests of up to {width * self.page_size} tokens")
        at = torch.arange(start, stop, dtype=INT32, device=self._table.device)
        return self._table[request][at // self.page_size] * self.page_size + at % self.page_size


def _block_scales(s, dev, shape):
    """Block scales as the bytes that append writes in place: checked, never converted."""
    if s.dtype == E8M0:
        s = s.view(torch.uint8)
    if s.dtype != torch.uint8 or s.device != dev or s.shape != shape or not s.is_contiguous() or s.data_ptr() % 16:
        raise ValueError(f"block scales: need contiguous, 16-byte aligned bytes of shape {shape} on {dev}, got {s.dtype} "
                         f"{tuple(s.shape)} on {s.device}")
    return s


class KVCache:
    """One layer's K/V pages: k [n_pages, kv_heads, page_size, k_dim] and v [..., v_dim].  Head dimensions 64/64, 128/128 or
    192/128.  Of three kinds:

    bf16;
    float8_e4m3fn with one fp32 scale per K/V head, k_scale and v_scale (a stored value stands for value * scale), which a
    user has to know beforehand: what is past 448 scales saturates;
    float8_e4m3fn with block_scales: k_scale and v_scale are bytes [n_pages, kv_heads, page_size / 16], and a value of a slot
    stands for value * 2 ** (byte - 127).  append sets a block's byte by the values that it writes (mimo_stream.append); a
    byte only grows until the block begins anew.  So what a request reads may depend on tokens that were rejected: a draft
    whose values raised its block's byte has rounded the older tokens' values below 2 ** -6 of the new scale to 2 ** -9 of it,
    and its byte stays when its step is dropped or its tokens are taken back, for the tokens that take their place as well.
    A request whose length is taken back to the block's first slot, or before it, writes the block anew."""

    def __init__(self, n_pages, page_size, kv_heads, k_dim, v_dim, dtype=torch.bfloat16, k_scale=None, v_scale=None,
                 device="cuda", block_scales=False):
        dev = _device(device)
        if block_scales:
            if k_scale is not None or v_scale is not None:
                raise ValueError("a cache with block scales makes its own (KVCache.of takes existing ones)")
            k_scale, v_scale = (torch.full((n_pages, kv_heads, max(page_size, 0) // 16), 127, dtype=torch.uint8, device=dev)
                                for _ in range(2))
        self._bind(torch.zeros((n_pages, kv_heads, page_size, k_dim), dtype=torch.uint8 if dtype == E4M3 else dtype, device=dev),
                   torch.zeros((n_pages, kv_heads, page_size, v_dim), dtype=torch.uint8 if dtype == E4M3 else dtype, device=dev),
                   k_scale, v_scale, dtype)

    @classmethod
    def of(cls, k, v, k_scale=None, v_scale=None):
        """A cache over existing page tensors (not copied).  Scales of three dimensions, uint8 or float8_e8m0fnu, are block
        scales: bytes 1 to 246, and not copied either."""
        self = cls.__new__(cls)
        self._bind(k, v, k_scale, v_scale, k.dtype)
        return self

    def _bind(self, k, v, k_scale, v_scale, dtype):
        if dtype not in (torch.bfloat16, E4M3):
            raise ValueError("a K/V cache holds bfloat16 or float8_e4m3fn")
        if k.dtype == torch.uint8:
            k, v = k.view(dtype), v.view(dtype)
        if k.device != v.device:
            raise ValueError(f"k on {k.device}, v on {v.device}")
        if k.dim() != 4 or v.dim() != 4 or k.shape[:3] != v.shape[:3] or v.dtype != dtype:
            raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must be [pages, kv_heads, page_size, dim] of one type")
        if not k.is_contiguous() or not v.is_contiguous():
            raise ValueError("cache pages must be contiguous")
        n_pages, heads, page, k_dim = k.shape
        if page < 16 or page > 1024 or page & (page - 1):
            raise ValueError("page_size must be a power of two from 16 to 1024")
        if (k_dim, v.shape[3]) not in ((64, 64), (128, 128), (192, 128)):
            raise ValueError(f"head dimensions {k_dim} / {v.shape[3]}: 64/64, 128/128 and 192/128 are supported")
        kind = _lib.KV_BF16
        if dtype == E4M3:
            if k_scale is None or v_scale is None:
                raise ValueError("an E4M3 cache needs k_scale and v_scale")
            blocks = [isinstance(s, torch.Tensor) and s.dim() == 3 for s in (k_scale, v_scale)]
            if blocks[0] != blocks[1]:
                raise ValueError("k_scale and v_scale of two kinds")
            if blocks[0]:
                k_scale, v_scale = (_block_scales(s, k.device, (n_pages, heads, page // 16)) for s in (k_scale, v_scale))
                if abs(k_scale.data_ptr() - v_scale.data_ptr()) < k_scale.numel():
                    raise ValueError("k_scale and v_scale overlap: a block scale belongs to K or to V")
                kind = _lib.KV_E4M3_BLOCKS
            else:
                k_scale, v_scale = (torch.as_tensor(s, dtype=torch.float32, device=k.device).expand(heads).contiguous()
                                    for s in (k_scale, v_scale))
                kind = _lib.KV_E4M3
        elif k_scale is not None or v_scale is not None:
            raise ValueError("scales belong to an E4M3 cache")
        self._tensors = (k, v, k_scale, v_scale)             # fixed: the struct holds their addresses
        self.dtype, self.device = dtype, k.device
        self.kv_heads, self.k_dim, self.v_dim, self.page_size, self.n_pages = heads, k_dim, v.shape[3], page, n_pages
        self.block_scales = kind == _lib.KV_E4M3_BLOCKS
        self._struct = _lib.MimoKvCache(*(_lib.ptr(t) for t in self._tensors), kind, n_pages, page, heads, k_dim, v.shape[3])
        self._calls = self._call = None
        if k.device.type == "cuda":
            try:
                self._calls = _lib.calls()
                self._call = self._calls.cache(ctypes.addressof(self._struct), k.device.index)
            except RuntimeError as e:                        # the long way serves every call, with 3 to 5 us more on the host
                warnings.warn(f"{e}; append, read and attend take longer on the host", RuntimeWarning, stacklevel=3)

    k = property(lambda self: self._tensors[0])
    v = property(lambda self: self._tensors[1])
    k_scale = property(lambda self: self._tensors[2])
    v_scale = property(lambda self: self._tensors[3])


def stretched(dim, theta, factor, original, few=1.0, many=32.0):
    """Frequencies fp64 [dim / 2] for contexts `factor` times as long as the `original` length that theta ** (-2 i / dim) was
    trained at: a pair that turns at least `many` times over the original length keeps its frequency, one of at most `few`
    turns has it divided by factor, and those between are blended in proportion to i, from the last whole pair number of
    `many` turns (0 at least) to the first of `few` (dim - 1 at most, past the last pair: where even that one turns more than
    `few` times, none is divided by the whole factor)."""
    if dim < 2 or dim % 2 or not 1.0 < theta < math.inf or not 0.0 < factor < math.inf or not 0 < original < math.inf or not 0.0 < few < many < math.inf:
        raise ValueError(f"need an even dim, theta > 1, factor > 0, original > 0 and 0 < few < many, all finite (got {dim}, {theta}, "
                         f"{factor}, {original}, {few}, {many})")
    i = torch.arange(dim // 2, dtype=torch.float64)
    freq = float(theta) ** (-2.0 * i / dim)
    # pair i turns original theta ** (-2 i / dim) / 2 pi times
    first, last = (0.5 * dim * math.log(original / (2.0 * math.pi * turns)) / math.log(theta) for turns in (many, few))
    first, last = max(math.floor(first), 0), min(math.ceil(last), dim - 1)
    slow = ((i - first) / max(last - first, 1)).clamp(0.0, 1.0)
    slow[i >= last] = 1.0                                    # pair 0 as well, where it has few turns already
    return freq * (1.0 - slow * (1.0 - 1.0 / factor))


def _rotary_number(name):
    """One of a Rotary's numbers: fixed, since its struct holds them.  A class derived from it may set its own, which a call then takes
    as they are (append)."""
    def change(self, value):
        if type(self) is Rotary:
            raise AttributeError(f"a Rotary's {name} is fixed")
        self.__dict__["_" + name] = value

    def value(self):
        try:
            return self.__dict__["_" + name]
        except KeyError:
            raise AttributeError(name) from None
    return property(value, change)


class Rotary:
    """Rotary positions on the first `dim` dimensions of a head (a multiple of 16): pairs (i, i + dim / 2), or (2 i, 2 i + 1) if
    interleaved; frequencies theta ** (-2 i / dim), or the dim / 2 given ones (stretched makes them for long contexts), kept
    as fp64 turns per position, so that far positions keep their fraction.  Rotated values are taken times magnitude."""

    def __init__(self, dim, theta=10000.0, device="cuda", interleaved=False, frequencies=None, magnitude=1.0):
        if dim < 16 or dim % 16 or dim > 256:
            raise ValueError("the rotary dimension must be a multiple of 16 up to 256")
        if not theta > 0.0:
            raise ValueError("theta must be positive")
        magnitude = float(magnitude)
        if not math.isfinite(magnitude) or abs(magnitude) > 3.4e38:
            raise ValueError("magnitude must be a finite fp32")
        if frequencies is None:
            frequencies = float(theta) ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
        else:
            frequencies = torch.as_tensor(frequencies).detach().to(device="cpu", dtype=torch.float64)
            if frequencies.shape != (dim // 2,) or not bool(torch.isfinite(frequencies).all()):
                raise ValueError(f"frequencies: need {dim // 2} finite numbers, got shape {tuple(frequencies.shape)}")
        self._bind((frequencies / (2.0 * math.pi)).to(_device(device)), int(dim), bool(interleaved), magnitude)

    def _bind(self, turns, dim, interleaved, magnitude):
        self._turns, self._dim, self._interleaved, self._magnitude = turns, dim, interleaved, magnitude
        self._struct = _lib.MimoRotary(turns.data_ptr(), dim, interleaved, magnitude)
        self._at = ctypes.addressof(self._struct)
        self._index = turns.device.index if turns.is_cuda else -1

    turns, dim, interleaved, magnitude = (_rotary_number(name) for name in ("turns", "dim", "interleaved", "magnitude"))

    # a copied or saved Rotary is its numbers; the struct, which holds an address, is made anew
    def __getstate__(self):
        own = ("_turns", "_dim", "_interleaved", "_magnitude")
        state = {name: value for name, value in self.__dict__.items() if name not in own + ("_struct", "_at", "_index")}
        return {**state, **{name[1:]: self.__dict__[name] for name in own if name in self.__dict__}}

    def __setstate__(self, state):
        state = dict(state)
        if "turns" in state and "dim" in state:              # a derived class may work them out instead
            self._bind(state.pop("turns"), state.pop("dim"), state.pop("interleaved", False), state.pop("magnitude", 1.0))
        self.__dict__.update(state)


def _turns_of(rotary, dev, k_dim):
    """(struct mimo_rotary, turns to be held until the call is queued): a Rotary's own, or of whatever else has dim and turns (fp64,
    the first dim / 2 of them) and may have interleaved and magnitude."""
    dim, turns = rotary.dim, rotary.turns
    if not 0 <= dim <= k_dim:
        raise ValueError(f"rotary dimension {dim} past the head's {k_dim}")
    if turns.device != dev:
        raise ValueError(f"rotary on {turns.device}, expected {dev}")
    if type(rotary) is Rotary:
        return rotary._struct, turns
    if turns.dtype != torch.float64 or turns.numel() < dim // 2 or not turns.is_contiguous():
        raise ValueError(f"rotary turns: need contiguous float64 [{dim // 2}], got {turns.dtype} {tuple(turns.shape)}")
    side, magnitude = getattr(rotary, "interleaved", False), getattr(rotary, "magnitude", 1.0)
    return _lib.MimoRotary(turns.data_ptr(), int(dim), bool(side), float(magnitude)), turns


def _rows(x, dev, heads, dim, name):
    """(x, address, elements between tokens): x as bf16 rows the kernels can read, [N, heads, dim] with contiguous, 16-byte
    aligned tokens at any distance; copied when it is not."""
    shape = x.shape
    if len(shape) != 3 or shape[2] != dim or (heads is not None and shape[1] != heads):
        raise ValueError(f"{name}: need [tokens, {'heads' if heads is None else heads}, {dim}], got {tuple(shape)}")
    if x.device != dev:
        raise ValueError(f"{name} on {x.device}, expected {dev}")
    if x.dtype is not BF16:
        x = x.to(BF16)
    s0, s1, s2 = x.stride()
    row = shape[1] * dim
    at = x.data_ptr()
    if shape[0] <= 1:
        s0 = row                                             # one token: any distance will do
    if s2 != 1 or (s1 != dim and shape[1] != 1) or s0 % 8 or s0 < row or at % 16:
        x = x.clone(memory_format=torch.contiguous_format)
        s0, at = row, x.data_ptr()
    return x, at, s0


def append(cache, plan, k, v, q=None, rotary=None):
    """Write the new tokens' k [N, kv_heads, k_dim] and v [N, kv_heads, v_dim] to plan.slots (rows with slot -1 are left
    out), k rotated to plan.positions; returns q [N, heads, k_dim] rotated likewise (None without q).  q, k and v may be
    views of one projection's rows; other types than bf16 are rounded to it first.  Slots are distinct.  rotary is a Rotary, or
    has a dim and fp64 turns [dim / 2] on the cache's device, as one has (interleaved and magnitude if they are not False and 1).

    Into a cache with block scales, the rows of one block of 16 slots follow one another, as in the plan of a step, with no
    other row between them, not even one that is left out (a block whose rows do not has undefined contents, and plan.check()
    raises where 15 or fewer rows lie between).  A call that writes a block's first slot begins the block anew; in another the
    scale of each head grows where the new values need it, and what the block holds is kept: exactly, but for values below
    2 ** -6 of the new scale, which are rounded to 2 ** -9 of it.  Values past 448 * 2 ** 119 saturate, infinities among
    them."""
    if cache._call is not None and (rotary is None or (type(rotary) is Rotary and rotary._dim <= cache.k_dim)):
        done = cache._calls.append(cache._call, _current_device(), _raw_stream(cache.device.index), plan.slots, plan.positions, plan.status,
                                   plan.page_size, k, v, q, 0 if rotary is None else rotary._at, -1 if rotary is None else rotary._index)
        if done is not NotImplemented:
            return _taken(done, "mimo_cache_append")
    _same_pages(plan, cache)
    dev = cache.device
    index = _gpu(dev)
    if _current_device() != index:
        with torch.cuda.device(dev):
            return append(cache, plan, k, v, q, rotary)
    k, at_k, k_stride = _rows(k, dev, cache.kv_heads, cache.k_dim, "k")
    v, at_v, v_stride = _rows(v, dev, cache.kv_heads, cache.v_dim, "v")
    N = k.shape[0]
    if v.shape[0] != N:
        raise ValueError(f"{N} tokens of k, {v.shape[0]} of v")
    at_slots = _int32(plan.slots, dev, (N,), "plan.slots")
    at_positions = _int32(plan.positions, dev, (N,), "plan.positions")
    turn, turns = (None, None) if rotary is None else _turns_of(rotary, dev, cache.k_dim)
    out, at_q, at_out, q_stride, heads = None, None, None, 0, 0
    if q is not None:
        q, at_q, q_stride = _rows(q, dev, None, cache.k_dim, "q")
        if q.shape[0] != N:
            raise ValueError(f"{N} tokens of k, {q.shape[0]} of q")
        heads = q.shape[1]
        out = torch.empty((N, heads, cache.k_dim), dtype=BF16, device=dev)
        at_out = out.data_ptr()
    status = _status(plan, dev)
    if N:
        rc = _entry("mimo_cache_append_rotary")(
            at_q, q_stride, heads, at_k, k_stride, at_v, v_stride, N, at_positions, at_slots, cache._struct, turn, at_out, status,
            _raw_stream(index))
        if rc:
            _lib.check(rc, "mimo_cache_append")
    return out


def read(cache, slots, out=None, status=None):
    """Cached tokens as rows: (k [N, kv_heads, k_dim], v [N, kv_heads, v_dim]) in bf16 of int32 slots [N] (a plan's, or
    PageTable.slots; in any order, any slot any number of times), stored values times their scales (in 32 bits, rounded to
    bf16); rows of slot -1 are 0.  Keys are as append left them, rotated.  out: two contiguous bf16 tensors to write; status:
    int32 [1] that receives a failure (a slot past the cache, whose row is 0) as plan.status does."""
    if cache._call is not None and out is None:
        done = cache._calls.read(cache._call, _current_device(), _raw_stream(cache.device.index), slots, status)
        if done is not NotImplemented:
            return _taken(done, "mimo_cache_read")
    dev = cache.device
    index = _gpu(dev)
    if _current_device() != index:
        with torch.cuda.device(dev):
            return read(cache, slots, out, status)
    N = slots.numel() if isinstance(slots, torch.Tensor) else 0
    at_slots = _int32(slots, dev, (N,), "slots")
    shapes = (N, cache.kv_heads, cache.k_dim), (N, cache.kv_heads, cache.v_dim)
    if out is None:
        k, v = (torch.empty(shape, dtype=BF16, device=dev) for shape in shapes)
    else:
        k, v = out
        for x, shape in zip((k, v), shapes):
            if x.dtype is not BF16 or x.shape != shape or not x.is_contiguous() or x.device != dev or x.data_ptr() % 16:
                raise ValueError(f"out: need a contiguous, 16-byte aligned bf16 tensor of shape {shape} on {dev}")
    at_status = None if status is None else _int32(status, dev, (1,), "status")
    if N:
        rc = _entry("mimo_cache_read")(cache._struct, at_slots, N, k.data_ptr(), v.data_ptr(), at_status, _raw_stream(index))
        if rc:
            _lib.check(rc, "mimo_cache_read")
    return k, v


@functools.lru_cache(maxsize=1024)
def _workspace_size(N, heads, kv_heads, v_dim):
    return _entry("mimo_cache_attend_workspace_size")(N, heads, kv_heads, v_dim)


def _workspace(nbytes, dev, stream):
    """A workspace of this call's own in a captured graph (two graphs never share one), else the stream's cached one."""
    if torch.cuda.is_current_stream_capturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=dev)
    ws = _lib._ws.get((dev.index, stream, "attend"))
    return ws if ws is not None and ws.numel() >= nbytes else _lib.workspace(nbytes, dev, "attend")


def attend(q, cache, plan, scale=None, window=0, sink_tokens=0, sink_logits=None, out=None):
    """Attention of the new tokens q [N, heads, k_dim] over the cache, which holds their keys and values already (append).

    A token at position p sees its request's keys j <= p; with window > 0 those with p - j < window, and the first
    sink_tokens.  scale defaults to k_dim ** -0.5.  q of another type than bf16 is rounded to it first.  In a call whose
    requests have up to 32 rows each (new tokens x heads / kv_heads, by plan.max_new) the softmax weights keep 17 bits in the
    product with v, else 8: a decoding request beside a chunk differs by that rounding.  sink_logits fp32 [heads]: a logit
    that joins each row's softmax without a value.  Returns bf16 [N, heads, v_dim] (out, if given: contiguous bf16); rows of
    no request are 0."""
    if cache._call is not None and not _capturing():
        index = cache.device.index
        stream = _raw_stream(index)
        ws = _lib._ws.get((index, stream, "attend"))
        if ws is not None:
            done = cache._calls.attend(cache._call, _current_device(), stream, q, plan.starts, plan.lens, plan.table, plan.max_new,
                                       plan.status, plan.page_size, scale, window, sink_tokens, sink_logits, out, ws)
            if done is not NotImplemented:
                return _taken(done, "mimo_cache_attend")
    if not (0 <= window <= INT32_MAX and 0 <= sink_tokens <= INT32_MAX):
        raise ValueError(f"window and sink_tokens must be from 0 to 2^31 - 1 (got {window}, {sink_tokens})")
    _same_pages(plan, cache)
    dev = cache.device
    index = _gpu(dev)
    if _current_device() != index:
        with torch.cuda.device(dev):
            return attend(q, cache, plan, scale, window, sink_tokens, sink_logits, out)
    q, at_q, q_stride = _rows(q, dev, None, cache.k_dim, "q")
    N, heads, _ = q.shape
    if heads < 1 or heads % cache.kv_heads:
        raise ValueError(f"{heads} heads on {cache.kv_heads} K/V heads")
    if plan.table is None or plan.table.dim() != 2:
        raise ValueError("the plan has no page table")
    B, width = plan.table.shape
    at_table = _int32(plan.table, dev, (B, width), "plan.table")
    at_starts = _int32(plan.starts, dev, (B + 1,), "plan.starts")
    at_lens = _int32(plan.lens, dev, (B,), "plan.lens")
    at_logits = None
    if sink_logits is not None:
        if sink_logits.shape != (heads,) or sink_logits.device != dev:
            raise ValueError(f"sink_logits of shape {tuple(sink_logits.shape)} on {sink_logits.device} for {heads} heads on {dev}")
        sink_logits = sink_logits.to(torch.float32).contiguous()
        at_logits = sink_logits.data_ptr()
    shape = (N, heads, cache.v_dim)
    if out is None:
        out = torch.empty(shape, dtype=BF16, device=dev)
    elif out.dtype is not BF16 or out.shape != shape or not out.is_contiguous() or out.device != dev or out.data_ptr() % 16:
        raise ValueError(f"out: need a contiguous, 16-byte aligned bf16 tensor of shape {shape} on {dev}")
    status = _status(plan, dev)
    if N == 0:
        return out
    stream = _raw_stream(index)
    ws = _workspace(_workspace_size(N, heads, cache.kv_heads, cache.v_dim), dev, stream)
    rc = _entry("mimo_cache_attend")(
        at_q, q_stride, N, heads, cache._struct, B, at_starts, at_lens, at_table, width,
        N if plan.max_new is None else max(-1, min(N, int(plan.max_new))), cache.k_dim ** -0.5 if scale is None else float(scale),
        int(window), int(sink_tokens), at_logits, out.data_ptr(), status, ws.data_ptr(), ws.numel(), stream)
    if rc:
        _lib.check(rc, "mimo_cache_attend")
    return out


class AttentionLayer:
    """The attention half of a decoder layer (engine/mimo_stream/model.py:296-298 around mimo_v2.py:110-150):

        r = input_layernorm(x);  q, k, v = r Wq, r Wk, r Wv;  h = x + attend(q, cache) Wo

    norm_weight bf16 [hidden] and eps as in MoELayer; qkv_weight bf16 [heads k_dim + kv_heads (k_dim + v_dim), hidden]
    (q rows, then k, then v), o_weight bf16 [hidden, heads v_dim]; cache: the layer's KVCache; rotary, window, sink_tokens,
    sink_logits and scale as in append and attend.  The two projections are library GEMMs, the rest the library's kernels.
    MoELayer takes its output: h = moe_layer(attention_layer(x, plan)), one plan for all layers of a step.  For inference: the
    weights are taken without their gradients' graph."""

    def __init__(self, norm_weight, eps, qkv_weight, o_weight, heads, cache, rotary=None, window=0, sink_tokens=0,
                 sink_logits=None, scale=None):
        dev = cache.device
        self.cache, self.heads, self.rotary, self.scale = cache, int(heads), rotary, scale
        self.window, self.sink_tokens = int(window), int(sink_tokens)
        self.norm_weight, self.qkv_weight, self.o_weight = (
            torch.as_tensor(w).detach().to(device=dev, dtype=BF16).contiguous() for w in (norm_weight, qkv_weight, o_weight))
        self.sink_logits = None if sink_logits is None else torch.as_tensor(sink_logits).detach().to(device=dev, dtype=torch.float32).contiguous()
        self.eps = float(eps)
        if not self.eps >= 0.0:
            raise ValueError("eps must be a non-negative number")
        self.hidden = self.norm_weight.numel()
        self.split = (self.heads * cache.k_dim, cache.kv_heads * cache.k_dim, cache.kv_heads * cache.v_dim)
        if self.heads < 1 or self.heads % cache.kv_heads:
            raise ValueError(f"{heads} heads on {cache.kv_heads} K/V heads")
        for name, w, shape in (("norm_weight", self.norm_weight, (self.hidden,)),
                               ("qkv_weight", self.qkv_weight, (sum(self.split), self.hidden)),
                               ("o_weight", self.o_weight, (self.hidden, self.heads * cache.v_dim))):
            if tuple(w.shape) != shape:
                raise ValueError(f"{name} of shape {tuple(w.shape)}, expected {shape}")
        if self.sink_logits is not None and tuple(self.sink_logits.shape) != (self.heads,):
            raise ValueError(f"sink_logits of shape {tuple(self.sink_logits.shape)} for {heads} heads")

    def __call__(self, x, plan):
        """h for x bf16 [N, hidden], the rows of the step that made plan."""
        dev = self.cache.device
        index = _gpu(dev)
        if x.device != dev or x.dim() != 2 or x.shape[1] != self.hidden:
            raise ValueError(f"x: need [tokens, {self.hidden}] on {dev}, got {tuple(x.shape)} on {x.device}")
        if _current_device() != index:
            with torch.cuda.device(dev):
                return self(x, plan)
        x = x.to(BF16).contiguous()
        if x.data_ptr() % 16:
            x = x.clone()
        h = torch.empty_like(x)
        N = x.shape[0]
        if N == 0:
            return h
        r = torch.empty_like(x)
        _lib.call("mimo_rmsnorm", _lib.ptr(x), N, self.hidden, _lib.ptr(self.norm_weight), self.eps, _lib.ptr(r), _lib.stream_ptr(dev))
        c = self.cache
        q, k, v = torch.matmul(r, self.qkv_weight.T).split_with_sizes(self.split, 1)
        q = append(c, plan, k.unflatten(1, (c.kv_heads, c.k_dim)), v.unflatten(1, (c.kv_heads, c.v_dim)),
                   q=q.unflatten(1, (self.heads, c.k_dim)), rotary=self.rotary)
        o = attend(q, c, plan, self.scale, self.window, self.sink_tokens, self.sink_logits)
        y = torch.matmul(o.flatten(1), self.o_weight.T)
        _lib.call("mimo_residual_add", _lib.ptr(x), _lib.ptr(y), x.numel(), _lib.ptr(h), _lib.stream_ptr(dev))
        return h
