"""Paged attention and its parts in 64 bits with numpy, and the rounding errors that the library's
types allow: what tests/test_gpu_paged.py holds the kernels to."""
import numpy as np

U32 = 2.0 ** -24   # half a step of f32, relative
U16 = 2.0 ** -11   # of f16


def positions(table, ps, pages, b, h, n):
    """Rows 0 .. n - 1 of sequence b's KV head h, float64 [n, D]."""
    j = np.arange(n)
    return pages[table[b, j // ps], h, j % ps].astype(np.float64)


def attend(q, k, v, limit, scale):
    """One query over rows 0 .. limit - 1 of k and v: (out, what one rounding per step may move)."""
    D = k.shape[1]
    if limit <= 0:
        return np.zeros(D), np.zeros(D), np.zeros(D)
    q, k, v = q.astype(np.float64), k[:limit], v[:limit]
    x = k @ q * scale
    p = np.exp(x - x.max())
    p /= p.sum()
    # a score: D products and sums, the scale, and a query held in two parts of 11 bits (2^-22);
    # the exponential and its difference from the maximum: 16 steps
    e = ((D + 16) * U32 + 2.0 ** -22) * abs(scale) * (np.abs(k) @ np.abs(q)).max() + 16 * U32 + np.abs(x - x.max()).max() * U32
    near = p @ np.abs(v)
    return p @ v, near * (2 * e + (limit + 64) * U32), near


def attention(q, k_pages, v_pages, table, lens, cu, ps, scale, q16):
    """out [rows, heads, D] and the absolute error allowed at each; rows of no sequence are NaN."""
    rows, heads, D = q.shape
    G = heads // k_pages.shape[1]
    out, tol = np.full(q.shape, np.nan), np.zeros(q.shape)
    for b in range(len(lens)):
        n = cu[b + 1] - cu[b]
        for h in range(heads):
            if not n:
                continue
            k, v = positions(table, ps, k_pages, b, h // G, lens[b]), positions(table, ps, v_pages, b, h // G, lens[b])
            for i in range(n):
                o, t, near = attend(q[cu[b] + i, h], k, v, lens[b] - n + i + 1, scale)
                # f16 rows: weights and result rounded to f16, half a step each (twice over, and
                # f16's smallest steps below its normal numbers)
                out[cu[b] + i, h], tol[cu[b] + i, h] = o, t + (U16 * (near + np.abs(o)) + 2.0 ** -24 * (near + 1) if q16 else 0)
    return out, tol
