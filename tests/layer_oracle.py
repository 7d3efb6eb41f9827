"""The layers of a transformer block over voxel features, restated in 64 bits with numpy, and the bounds that their outputs are
held to.  Test infrastructure only.

Units: u = 2^-24 is half a step of FP32 relative to a value, 2^-11 that of FP16 (2^-25 its smallest half step); a sum of n
FP32 terms in any order is within n * u of the sum of their magnitudes.
"""
import numpy as np

U = 2.0 ** -24


# --- e4m3: sign, four bits of exponent (bias 7), three of mantissa, no infinities; 0x7f and 0xff are NaN
def e4m3_values():
    v = np.zeros(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        v[c] = np.nan if c & 0x7f == 0x7f else -x if c & 0x80 else x
    return v


VALUES = e4m3_values()


def to_e4m3(x):
    """Codes of the e4m3 nearest to x (64 bits), ties to the even mantissa, beyond 448 the largest."""
    a = np.abs(np.asarray(x, np.float64))
    e = np.maximum(np.frexp(np.where(a > 0, a, 1.0))[1] - 1, -6).astype(np.int64)
    r = np.rint(np.ldexp(np.where(np.isfinite(a), a, 0.0), 3 - e)).astype(np.int64)  # eighths of 2^e
    code = np.minimum(np.where(a < 2.0 ** -6, r, (e + 7) * 8 + r - 8), 0x7e)
    return np.where(np.isnan(x), 0x7f, code | np.where(np.signbit(x), 0x80, 0)).astype(np.uint8)


def near_a_border(x):
    """Whether x is so near the middle of two e4m3 that its FP32 form, rounded to nearest, may lie on the other side."""
    a = np.abs(np.asarray(x, np.float64))
    e = np.maximum(np.frexp(np.where(a > 0, a, 1.0))[1] - 1, -6)
    r = np.ldexp(a, 3 - e)
    return np.abs(r - np.floor(r) - 0.5) <= 2 * U * r


def norm(feat, residual, gamma, eps):
    """-> quotient y / s (64 bits, not rounded), s, h;  h is the FP32 sum"""
    h = feat.astype(np.float32)
    if residual is not None:
        with np.errstate(over="ignore", invalid="ignore"):
            h = h + residual.astype(np.float32)
    d = h.astype(np.float64)
    with np.errstate(all="ignore"):
        y = d / np.sqrt((d * d).mean(1, keepdims=True) + eps) * gamma.astype(np.float64)
        s = np.maximum(np.abs(y).max(1, keepdims=True) / 448.0, 2.0 ** -100)
        return y / s, s, h


def norm_scale_tolerance(channels):
    """Relative: sum of squares and mean (channels + 2 roundings, halved by the root), eps, root, reciprocal, product, quotient."""
    return ((channels + 2) / 2 + 8) * U


def linear(codes, row_scale, w, scale=None, shift=None, relu=False):
    """-> result, and the sum of the magnitudes that it is made of"""
    ws = np.maximum(np.abs(w).max(0) / np.float32(448.0), np.float32(2.0 ** -100)).astype(np.float32)
    wq = VALUES[to_e4m3((w / ws).astype(np.float32))]
    q, s = VALUES[codes], row_scale.astype(np.float64)
    by = ws.astype(np.float64) * (1.0 if scale is None else scale.astype(np.float64))
    add = 0.0 if shift is None else shift.astype(np.float64)
    y = (q @ wq) * s * by + add
    magnitude = (np.abs(q) @ np.abs(wq)) * np.abs(s * by) + np.abs(add)
    return (np.where(y < 0, 0.0, y) if relu else y), magnitude


def linear_tolerance(want, magnitude, cin, half):
    """cin products (exact) added in FP32, four roundings of the epilogue, one to the output's type."""
    return magnitude * (cin + 5) * U + (np.abs(want) * 2.0 ** -11 + 2.0 ** -25 if half else np.abs(want) * U)


def attention(qkv, coors, n, grid_zyx, window_zyx, shift_zyx, heads, kv_heads, dim, slopes, cell_zyx, cap, scale):
    """-> output [rows, heads * dim], bound on an FP32 or FP16 kernel's distance from it (of the same shape).  Rows outside the grid and
    beyond n: zeros.

    The bound.  A score t = scale * q.k is within e_t = (dim + 2) u * scale * sum|q_d k_d| of itself, which the cap's slope (at most 1)
    does not enlarge; the cap itself adds 8 u * cap (argument, exponential, quotient, product).  A voxel's place is taken from its
    window's first cell on and is within u of itself, so that a difference is within 2 u * extent of the window on that axis and a
    distance within 4 u * the extents' sum and, for squares, sums, root and product, 8 u of itself.  Taken to the base 2 and less the maximum, it is rounded three times
    more: 4 u * (|t| + |max|).  With e the largest such error of a row, a weight is within 2 e + 8 u of itself relative to the
    others (2^x within 4 u), the sum of L weights and that of L products within L u each, every rescaling of a running sum
    by 8 u more, L / 32 of them at most.  FP16: the weights are rounded to 11 bits, relative 2^-11 or 2^-25 of the largest weight.
    All of that multiplies sum p |v|, the 2^-25 L max|v|; the quotient and the output's rounding follow."""
    rows = len(qkv)
    half = qkv.dtype == np.float16
    x = qkv.astype(np.float64)
    out, bound = np.zeros((rows, heads * dim)), np.zeros((rows, heads * dim))
    c = coors[:n].astype(np.int64)
    grid = np.array(grid_zyx)
    inside = (c[:, 0] == 0) & (c[:, 1:] >= 0).all(1) & (c[:, 1:] < grid).all(1) if n else np.zeros(0, bool)
    win = (c[:, 1:] + np.array(shift_zyx)) // np.array(window_zyx)
    p_at = c[:, 1:] * np.array(cell_zyx, np.float32).astype(np.float64)
    extent = float((np.minimum(window_zyx, grid) * np.abs(np.array(cell_zyx, np.float64))).sum())
    at = np.nonzero(inside)[0]
    if not len(at):
        return out, bound
    _, which = np.unique(win[at], axis=0, return_inverse=True)
    for w in range(which.max() + 1):
        b = at[which.reshape(-1) == w]
        far = np.sqrt(((p_at[b][:, None] - p_at[b][None]) ** 2).sum(2))
        for h in range(heads):
            g = h // (heads // kv_heads)
            q = x[b, h * dim:(h + 1) * dim]
            k = x[b, (heads + g) * dim:(heads + g + 1) * dim]
            v = x[b, (heads + kv_heads + g) * dim:(heads + kv_heads + g + 1) * dim]
            with np.errstate(all="ignore"):
                t = scale * (q @ k.T)
                e = (dim + 2) * U * abs(scale) * (np.abs(q) @ np.abs(k).T)
                if cap:
                    t = cap * np.tanh(t / cap)
                    e = e + 8 * U * cap
                if slopes is not None:
                    t = t - float(slopes[h]) * far
                    e = e + abs(float(slopes[h])) * (8 * U * far + 4 * U * extent)
                e = (e + 4 * U * (np.abs(t) + np.abs(t.max(1, keepdims=True)))).max(1, keepdims=True)
                p = np.exp(t - t.max(1, keepdims=True))
                total = p.sum(1, keepdims=True)
                o = (p @ v) / total
                a = (p @ np.abs(v)) / total
                length = len(b)
                rel = 2 * e + 8 * U + 2 * length * U + 8 * U * (length / 32 + 1)
                if half:
                    rel = rel + 2.0 ** -11
                    tol = a * rel + length * 2.0 ** -25 * np.abs(v).max(0) / total + np.abs(o) * 2.0 ** -11 + 2.0 ** -25
                else:
                    tol = a * rel + np.abs(o) * 4 * U
            out[b, h * dim:(h + 1) * dim] = o
            bound[b, h * dim:(h + 1) * dim] = tol
    return out, bound
