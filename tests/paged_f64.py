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
    """Queries [n, D] over rows 0 .. limit[i] - 1 of k and v: out, the error that one rounding per
    step may make, and sum_j p_j |v_j|."""
    D = k.shape[1]
    seen = np.arange(len(k))[None] < limit[:, None]
    some = limit > 0
    q = q.astype(np.float64)
    x = np.where(seen, q @ k.T * scale, -np.inf)
    size = np.where(seen, np.abs(q) @ np.abs(k).T, 0.0)
    top = np.where(some, np.max(x, axis=1, initial=-np.inf), 0.0)
    p = np.exp(x - top[:, None])
    p /= np.where(some, p.sum(1), 1.0)[:, None]
    # a score: D products and sums, the scale, and a query held in two parts of 11 bits (2^-22);
    # the exponential and its difference from the maximum: 16 steps
    far = np.max(np.where(seen, top[:, None] - x, 0.0), axis=1, initial=0.0)
    e = ((D + 16) * U32 + 2.0 ** -22) * abs(scale) * size.max(1, initial=0.0) + 16 * U32 + far * U32
    near = p @ np.abs(v)
    return p @ v, near * (2 * e + (np.maximum(limit, 0) + 64) * U32)[:, None], near


def attention(q, k_pages, v_pages, table, lens, cu, ps, scale, q16):
    """out [rows, heads, D] and the absolute error allowed at each; rows of no sequence are NaN."""
    rows, heads, D = q.shape
    G = heads // k_pages.shape[1]
    out, tol = np.full(q.shape, np.nan), np.zeros(q.shape)
    for b in range(len(lens)):
        n = cu[b + 1] - cu[b]
        for h in range(heads if n else 0):
            k, v = positions(table, ps, k_pages, b, h // G, lens[b]), positions(table, ps, v_pages, b, h // G, lens[b])
            at = slice(cu[b], cu[b + 1])
            o, t, near = attend(q[at, h], k, v, lens[b] - n + 1 + np.arange(n), scale)
            # f16 rows: weights and result rounded to f16, half a step each, and f16's smallest steps
            # below its normal numbers
            out[at, h], tol[at, h] = o, t + (U16 * (near + np.abs(o)) + 2.0 ** -24 * (near + 1) if q16 else 0)
    return out, tol
