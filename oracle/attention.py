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
