"""Attention among the rows of one window in 64 bits, with bounds that follow from the formula alone.  Test infrastructure only.

u = 2^-24 is half a step of FP32 relative to a value, 2^-11 that of FP16.
"""
import numpy as np

U = 2.0 ** -24


def one_window(qkv, cells, heads, kv_heads, dim, slopes=None, cell=(1.0, 1.0, 1.0), cap=0.0, scale=1.0, queries=None):
    """qkv [rows, (heads + 2 kv_heads) dim], cells [rows, 3] integers -> output [rows, heads * dim], bound of the same shape;  of `queries` alone, if
    there are any.

    A score t = scale q.k: within (dim + 2) u scale sum|q_d k_d| of itself; the cap, whose slope is at most 1, adds 8 u cap.  The difference
    of two cells is an integer below 2^24, exact in FP32; times the cells' size (u), squared (doubles that) with three products and
    two sums (u each at most, all terms positive), a root (halves it, 2 u of its own) and the slope (3 u with what it is held in): 8 u of
    slope * distance.  Less the maximum and to the base 2: three roundings of at most |t| + |max|.  With e the largest such error of a row, a
    weight is within 2 e + 8 u of itself relative to the others (exponential 4 u); sums of L terms within L u each, numerator and denominator,
    a running sum's rescaling 8 u for each block of 16 keys that raises the maximum.
    FP16: a weight is rounded to 11 bits, 2^-11 relative or, of the smallest, 2^-39 of the largest one, in numerator and denominator."""
    half = qkv.dtype == np.float16
    x = qkv.astype(np.float64)
    rows = len(x)
    of = np.arange(rows) if queries is None else np.asarray(queries)
    out, bound = np.zeros((len(of), heads * dim)), np.zeros((len(of), heads * dim))
    if slopes is not None:
        diff = (cells[of][:, None].astype(np.int64) - cells[None].astype(np.int64)) * np.asarray(cell, np.float32).astype(np.float64)
        far = np.sqrt((diff ** 2).sum(2))
    for h in range(heads):
        g = h // (heads // kv_heads)
        q, k, v = (x[:, i * dim:(i + 1) * dim] for i in (h, heads + g, heads + kv_heads + g))
        q = q[of]
        t = scale * (q @ k.T)
        e = (dim + 2) * U * abs(scale) * (np.abs(q) @ np.abs(k).T)
        if cap:
            t = cap * np.tanh(t / cap)
            e = e + 8 * U * cap
        if slopes is not None:
            s = float(np.float32(slopes[h]))
            t = t - s * far
            e = e + 8 * U * abs(s) * far
        top = t.max(1, keepdims=True)
        p = np.exp(t - top)
        total = p.sum(1, keepdims=True)
        # (an error of a score that weighs nothing moves nothing: those within 60 of the largest one count)
        e = np.where(t >= top - 60, e + 3 * U * (np.abs(t) + np.abs(top)), 0).max(1, keepdims=True)
        o, a = (p @ v) / total, (p @ np.abs(v)) / total
        rel = 2 * e + 8 * U + 2 * rows * U + 8 * U * (rows / 16 + 1) + (2.0 ** -10 if half else 0.0)
        tol = (a + np.abs(o)) * rel
        if half:
            tol = tol + rows * 2.0 ** -39 / total * (np.abs(v).max(0) + np.abs(o)) + np.abs(o) * 2.0 ** -11 + 2.0 ** -25
        else:
            tol = tol + np.abs(o) * 4 * U
        out[:, h * dim:(h + 1) * dim], bound[:, h * dim:(h + 1) * dim] = o, tol
    return out, bound


def windows(qkv, cells, window, heads, kv_heads, dim, most=1000, seed=0, **kw):
    """The same for rows of several windows: rows that are checked, output, bound.  Of a window of more than `most` rows, 150 are."""
    _, which = np.unique(cells // np.array(window), axis=0, return_inverse=True)
    which = which.reshape(-1)
    rows, outs, bounds = [], [], []
    for w in range(which.max() + 1):
        at = np.nonzero(which == w)[0]
        some = None
        if len(at) > most:
            some = np.unique(np.concatenate([[0, len(at) - 1], np.random.default_rng(seed).integers(len(at), size=150)]))
        o, b = one_window(qkv[at], cells[at], heads, kv_heads, dim, queries=some, **kw)
        rows.append(at if some is None else at[some])
        outs.append(o)
        bounds.append(b)
    return np.concatenate(rows), np.concatenate(outs), np.concatenate(bounds)
