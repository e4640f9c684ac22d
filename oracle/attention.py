"""The attention half's operators over a paged K/V cache, restated in numpy and 64 bits: page tables and slots of a step,
rotary positions, and attention with causal order, sliding window, visible first tokens and sink logits (the semantics of
the reference's Attention, engine/mimo_stream/mimo_v2.py:66-150)."""
import numpy as np


def pages(n, page):
    return -(-n // page)


def step(lens, target, table, free, n_free, page, n_tokens):
    """(starts, lens, slots, positions, n_free, table, free) after a step; table and free are copies."""
    table, free = np.array(table), np.array(free)
    stack = list(free[:n_free])
    released = [table[b, j] for b, (x, y) in enumerate(zip(lens, target)) for j in range(pages(y, page), pages(x, page))]
    stack += released[::-1]
    starts, slots, positions = [0], [], []
    for b, (x, y) in enumerate(zip(lens, target)):
        for j in range(pages(x, page), pages(y, page)):
            table[b, j] = stack.pop()
        for p in range(x, y):
            slots.append(int(table[b, p // page]) * page + p % page)
            positions.append(p)
        starts.append(len(slots))
    for i in range(n_free, len(stack)):
        free[i] = stack[i]
    pad = n_tokens - len(slots)
    return (np.array(starts), np.array(target), np.array(slots + [-1] * pad, dtype=np.int64),
            np.array(positions + [0] * pad, dtype=np.int64), len(stack), table, free)


def rotate(x, positions, dim, theta):
    """x [N, heads, D] float64 with its first dim dimensions rotated, pairs (i, i + dim / 2)."""
    x = np.array(x, dtype=np.float64)
    half = dim // 2
    angle = np.asarray(positions, dtype=np.float64)[:, None] * theta ** (-2.0 * np.arange(half) / dim)
    c, s = np.cos(angle)[:, None, :], np.sin(angle)[:, None, :]
    a, b = x[..., :half].copy(), x[..., half:dim].copy()
    x[..., :half], x[..., half:dim] = a * c - b * s, b * c + a * s
    return x


def visible(p, length, window, sinks):
    """Which keys j < length the token at position p sees."""
    j = np.arange(length)
    seen = j <= p
    if window:
        seen &= (p - j < window) | (j < sinks)
    return seen


def attend(q, k_pages, v_pages, starts, lens, table, scale, window=0, sinks=0, sink_logits=None):
    """q [N, heads, Dk], pages [P, kv_heads, page, D], all float64.  Returns the output [N, heads, Dv] and the weighted mean
    of |v| (the size that rounding the weights acts on), both 0 for rows of no request."""
    N, heads, _ = q.shape
    _, kv_heads, page, dv = v_pages.shape
    out = np.zeros((N, heads, dv))
    size = np.zeros((N, heads, dv))
    G = heads // kv_heads
    for b in range(len(lens)):
        length, n = int(lens[b]), int(starts[b + 1] - starts[b])
        if n == 0:
            continue
        rows = slice(int(starts[b]), int(starts[b + 1]))
        ids = np.asarray(table[b][:pages(length, page)], dtype=np.int64)
        seen = np.stack([visible(length - n + i, length, window, sinks) for i in range(n)])[:, None, :]
        used = seen.any(axis=(0, 1))                       # keys no row sees are not touched: they may hold anything
        for g in range(kv_heads):
            K = np.where(used[:, None], k_pages[ids, g].reshape(-1, k_pages.shape[3])[:length], 0.0)
            V = np.where(used[:, None], v_pages[ids, g].reshape(-1, dv)[:length], 0.0)
            with np.errstate(invalid="ignore", over="ignore"):
                s = np.where(seen, scale * (q[rows, g * G:(g + 1) * G] @ K.T), -np.inf)
            top = s.max(axis=-1, keepdims=True)
            sink = None if sink_logits is None else np.asarray(sink_logits, dtype=np.float64)[None, g * G:(g + 1) * G, None]
            if sink is not None:
                top = np.maximum(top, sink)
            with np.errstate(invalid="ignore"):
                w = np.where(seen & (s != -np.inf), np.exp(s - np.where(top == -np.inf, 0.0, top)), 0.0)
                total = w.sum(axis=-1, keepdims=True)
                if sink is not None:
                    total = total + np.where(top == -np.inf, 0.0, np.exp(sink - np.where(top == -np.inf, 0.0, top)))
                bad = ~np.isfinite(V).all(axis=1)          # a weight of 0 keeps a row clear of another row's NaN value
                o = w[..., ~bad] @ V[~bad]
                z = w[..., ~bad] @ np.abs(V[~bad])
                for j in np.flatnonzero(bad):
                    o += np.where(seen[..., j, None], w[..., j, None] * V[j], 0.0)
            out[rows, g * G:(g + 1) * G] = np.where(total == 0.0, 0.0, o / np.where(total == 0.0, 1.0, total))
            size[rows, g * G:(g + 1) * G] = np.where(total == 0.0, 0.0, z / np.where(total == 0.0, 1.0, total))
    return out, size


def turn(x, positions, frequencies, interleaved=False, magnitude=1.0):
    """x [N, heads, D] float64 with its first 2 len(frequencies) dimensions rotated in pairs (i, i + len) or (2 i, 2 i + 1)."""
    x = np.array(x, dtype=np.float64)
    half = len(frequencies)
    angle = np.asarray(positions, dtype=np.float64)[:, None, None] * np.asarray(frequencies, dtype=np.float64)
    c, s = magnitude * np.cos(angle), magnitude * np.sin(angle)
    at = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = x[..., at[0]].copy(), x[..., at[1]].copy()
    x[..., at[0]], x[..., at[1]] = a * c - b * s, b * c + a * s
    return x


def stretched(dim, theta, factor, original, few, many):
    """Frequencies of a context stretched by factor, pair by pair: those that turn `many` times over the original length or
    more are kept, those of up to `few` divided by factor, and pair numbers between are blended in proportion."""
    freq = [theta ** (-2.0 * i / dim) for i in range(dim // 2)]

    def pair_of(turns):                                    # the real pair number whose frequency makes that many turns
        return dim * np.log(original / (2 * np.pi * turns)) / (2 * np.log(theta))
    lo, hi = max(int(np.floor(pair_of(many))), 0), min(int(np.ceil(pair_of(few))), dim - 1)
    out = []
    for i, f in enumerate(freq):
        share = 1.0 if i >= hi else 0.0 if i <= lo else (i - lo) / (hi - lo)
        out.append((1 - share) * f + share * f / factor)
    return np.array(out)


SCALE_ROWS = 16
SCALE_TOP = 246


def block_byte(most):
    """The smallest byte s of 1 .. 246 with most <= 448 * 2 ** (s - 127) (246 if none is large enough)."""
    for s in range(1, SCALE_TOP):
        if most <= 448.0 * 2.0 ** (s - 127):
            return s
    return SCALE_TOP


def block_write(held, byte, x, slots, page):
    """What a cache with block scales holds after x [N, heads, D] (float64; NaN and infinities among it) went to its slots: its
    values divided by their block's scale, before any rounding, and the bytes.  held [pages, heads, page, D] are the codes'
    values before, byte [pages, heads, page / 16]."""
    held, byte = np.array(held, dtype=np.float64), np.array(byte, dtype=np.int64)
    n = 0
    while n < len(slots):
        if slots[n] < 0:
            n += 1
            continue
        rows = [n]
        while n + 1 < len(slots) and slots[n + 1] >= 0 and slots[n + 1] // SCALE_ROWS == slots[n] // SCALE_ROWS:
            n += 1
            rows.append(n)
        n += 1
        p, block = slots[rows[0]] // page, slots[rows[0]] % page // SCALE_ROWS
        span = slice(SCALE_ROWS * block, SCALE_ROWS * (block + 1))
        for h in range(held.shape[1]):
            values = np.abs(x[rows, h])
            need = block_byte(values[np.isfinite(values)].max(initial=0.0))
            if not any(slots[r] % SCALE_ROWS == 0 for r in rows):
                old = int(byte[p, h, block])
                need = max(need, old)
                held[p, h, span] *= 2.0 ** (old - need)
            byte[p, h, block] = need
            for r in rows:
                held[p, h, slots[r] % page] = np.clip(x[r, h] * 2.0 ** (127 - need), -448.0, 448.0)
    return held, byte


def block_values(codes, byte):
    """Values [pages, heads, page, D] that codes (as float64) and bytes stand for."""
    return codes * np.repeat(2.0 ** (np.asarray(byte, dtype=np.float64) - 127.0), SCALE_ROWS, axis=2)[..., None]
