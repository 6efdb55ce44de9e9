"""CPU restatement in 64 bits of the frame-cache operators (block tables and slots, rotary rows into pages, attention
of new frames over pages), one sequence and one row at a time, for the tests."""

from __future__ import annotations

import numpy as np

NO_PAGES, TABLE_FULL, ROWS_FULL, BAD_LENGTH = 1, 2, 4, 8


def plan(cached, new, page, free, table, max_rows):
    """(table, cu, total, slots, positions, taken, flags) as lists and arrays of whole numbers."""
    table, free = np.array(table), list(free)
    cu, total, flags, wanted = [0], [], 0, 0
    slots, positions = np.full(max_rows, -1, np.int64), np.zeros(max_rows, np.int64)
    for i, (c, n) in enumerate(zip(cached, new)):
        if c < 0 or n < 0 or c + n > 1 << 30:
            flags, c, n = flags | BAD_LENGTH, 0, 0
        held, need = -(-c // page), -(-(c + n) // page)
        if need > table.shape[1]:
            flags |= TABLE_FULL
        for column in range(held, need):
            got = free[wanted] if wanted < len(free) else -1
            wanted += 1
            if column < table.shape[1]:
                table[i, column] = got
        for k in range(n):
            row = cu[-1] + k
            if row < max_rows:
                p = c + k
                positions[row] = p
                if p // page < table.shape[1] and table[i, p // page] >= 0:
                    slots[row] = table[i, p // page] * page + p % page
        cu.append(cu[-1] + n)
        total.append(c + n)
    if wanted > len(free):
        flags |= NO_PAGES
    if cu[-1] > max_rows:
        flags |= ROWS_FULL
    return table, cu, total, slots, positions, min(wanted, len(free)), flags


def rotate(x, positions, freqs):
    """(rows, heads, 64) float64, pairs (2j, 2j + 1) turned by position * freq_j; also sum(|x0| + |x1|) per element."""
    a = np.asarray(positions, np.float64)[:, None] * np.asarray(freqs, np.float64)[None]
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    x0, x1 = x[..., 0::2], x[..., 1::2]
    y, size = np.empty_like(x), np.empty_like(x)
    y[..., 0::2], y[..., 1::2] = x0 * c - x1 * s, x1 * c + x0 * s
    size[..., 0::2] = size[..., 1::2] = np.abs(x0) + np.abs(x1)
    return y, size


def visible(total, n, i, causal, window):
    """Keys [lo, hi) that new frame i of n sees in a sequence of `total` frames."""
    pos = total - n + i
    hi = min(total, max(0, pos + 1)) if causal else total
    lo = max(0, pos - window + 1) if window else 0
    return min(lo, hi), hi


def attention(q, k, v, table, cu, total, page, causal, window, scale, gates=None):
    """float64 arrays q (rows, heads, 64), k and v (pages, cache heads, page, 64). Returns the result (rows, heads,
    64), the same with |v| in the place of v (what rounding of the weights scales with) and the number of keys of
    each row; rows of no sequence are zero."""
    rows, heads, _ = q.shape
    kv = k.shape[1]
    group = heads // kv
    out, size, keys = np.zeros_like(q), np.zeros_like(q), np.zeros(rows, np.int64)
    for i, t in enumerate(total):
        n = cu[i + 1] - cu[i]
        if n == 0:
            continue
        pages = [table[i][c] for c in range(-(-t // page))]
        ks = k[pages].transpose(1, 0, 2, 3).reshape(kv, -1, 64)[:, :t]
        vs = v[pages].transpose(1, 0, 2, 3).reshape(kv, -1, 64)[:, :t]
        for f in range(n):
            lo, hi = visible(t, n, f, causal, window)
            row = cu[i] + f
            keys[row] = hi - lo
            if lo == hi:
                continue
            s = np.einsum("kgd,kjd->kgj", q[row].reshape(kv, group, 64), ks[:, lo:hi]) * scale
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            out[row] = np.einsum("kgj,kjd->kgd", p, vs[:, lo:hi]).reshape(heads, 64)
            size[row] = np.einsum("kgj,kjd->kgd", p, np.abs(vs[:, lo:hi])).reshape(heads, 64)
    if gates is not None:
        out, size = out * gates[..., None], size * np.abs(gates[..., None])
    return out, size, keys
