"""VoxelAttention on the GPU where FP32 and FP16 run out of bits: against 64 bits, with bounds from the formula alone (attention_bounds.py)."""
import numpy as np
import pytest
import torch

import attention_bounds as A
from gpu_util import dev
from sessd3d import api

pytestmark = pytest.mark.gpu
HALF, FLOAT = torch.float16, torch.float32
# Rows of the tensor that holds a window: a few, those whose windows are listed, and so many that a workgroup takes two heads in FP16
CAPACITIES = [None, 6000, 100500]


def num(n):
    return dev(np.array([n], np.int32))


def attend(qkv, cells, grid_zyx, heads, kv_heads, dim, capacity=None, **kw):
    """One window as large as the grid; the tensor's rows behind the window's are NaN."""
    n = len(qkv)
    rows = max(n, capacity or n)
    x = np.full((rows, qkv.shape[1]), np.nan, qkv.dtype)
    coors = np.full((rows, 4), -1, np.int32)
    x[:n], coors[:n, 0], coors[:n, 1:] = qkv, 0, cells
    op = api.VoxelAttention(heads, kv_heads, dim, grid_zyx[::-1], grid_zyx[::-1], max_voxels=rows, **kw)
    got = op(dev(x), dev(coors), num(n))
    assert op.status() == 0
    return got.cpu().numpy()[:n].astype(np.float64)


def assert_within(got, want, tol):
    off = ~(np.abs(got - want) <= tol)
    assert not off.any(), (int(off.sum()), float(np.nanmax(np.abs(got - want))), float((np.abs(got - want) / tol)[off].max()))


@pytest.mark.parametrize("capacity", CAPACITIES)
@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("length,cell,slope", [(1600, 0.05, 40.0), (100000, 0.05, 20.0), (1 << 24, 0.3, 4.0), (1 << 24, 1e-3, 1e3)])
def test_distances_far_from_the_windows_first_cell(dtype, length, cell, slope, capacity):
    """Neighbours at the far end of a long window: their distance has the bits that it has anywhere else."""
    rng = np.random.default_rng(length)
    n, heads, dim = 300, 2, 16
    cells = np.zeros((n, 3), np.int64)
    cells[:, 2] = length - 1 - rng.choice(min(length, 900), n, replace=False)
    cells[:, 1] = rng.integers(0, 40, n)
    cells[:, 0] = rng.integers(0, 4, n)
    qkv = rng.standard_normal((n, 3 * heads * dim)).astype(np.float16 if dtype == HALF else np.float32)
    size = (2 * cell, cell, cell)  # z,y,x
    slopes = np.array([slope, slope / 7], np.float32)
    want, tol = A.one_window(qkv, cells, heads, heads, dim, slopes, size, scale=0.25)
    assert_within(attend(qkv, cells, (4, 40, length), heads, heads, dim, capacity, slopes=slopes, cell_size_xyz=size[::-1]), want, tol)


@pytest.mark.parametrize("capacity", CAPACITIES)
@pytest.mark.parametrize("dtype,exponent", [(t, e) for t in (HALF, FLOAT) for e in (20, 26, 29, 32, 35)] + [(FLOAT, 60)])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("n", [20, 60, 700])
def test_scores_of_any_size(dtype, exponent, bias, n, capacity):
    """Scores of some 2^exponent, apart by at least a thousandth of that: the largest one's key takes all, and scores that are the same share."""
    rng = np.random.default_rng(exponent)
    heads, dim, t = 2, 64, np.float16 if dtype == HALF else np.float32
    cells = np.stack(np.unravel_index(np.arange(n), (1, 28, 25)), 1)
    qkv = np.zeros((n, 3 * heads * dim), t)
    each = 2.0 ** ((exponent - 6) / 2)  # of 64 products, that of a query's value and a key's
    for h in range(heads):
        key = np.rint(rng.permutation(n) * (1000.0 / n)) + 1000.0   # (1000 .. 2000, of 11 bits: what they are times is a power of two)
        key[rng.integers(n, size=n // 4)] = key.max()
        sign = rng.choice([-1.0, 1.0], n)
        qkv[:, h * dim:(h + 1) * dim] = (sign * 2.0 ** np.floor(np.log2(each)))[:, None]
        qkv[:, (heads + h) * dim:(heads + h + 1) * dim] = (key * 2.0 ** (np.ceil(np.log2(each)) - 10))[:, None]
    qkv[:, 2 * heads * dim:] = rng.standard_normal((n, heads * dim))
    assert np.isfinite(qkv).all()
    slopes = [0.5, 0.25] if bias else None
    x = qkv.astype(np.float64)
    want = np.zeros((n, heads * dim))
    for h in range(heads):
        q, k, v = (x[:, i * dim:(i + 1) * dim] for i in (h, heads + h, 2 * heads + h))
        s = q @ k.T
        if bias:  # (in FP32 it is less than a step of the score, or decides between scores that are the same)
            far = np.sqrt(((cells[:, None] - cells[None]) ** 2).sum(2))
            s = (s.astype(np.float32) - np.float32(slopes[h]) * far.astype(np.float32)).astype(np.float64)
        p = np.exp(s - s.max(1, keepdims=True))
        want[:, h * dim:(h + 1) * dim] = (p @ v) / p.sum(1, keepdims=True)
    got = attend(qkv, cells, (1, 28, 25), heads, heads, dim, capacity, softmax_scale=1.0, slopes=slopes)
    assert np.isfinite(got).all()
    if not bias:  # equal weights of 1 or 2^14, and zeros
        tol = (2.0 ** -11 if dtype == HALF else 8 * A.U) * np.abs(x[:, 2 * heads * dim:]).max() + n * A.U
        assert_within(got, want, np.full(want.shape, tol))


@pytest.mark.parametrize("capacity", CAPACITIES)
@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 1, 16), (2, 2, 32), (2, 1, 64)])
@pytest.mark.parametrize("below", [9.0, 16.0, 17.25, 17.5, 20.0])
def test_what_many_small_weights_add_up_to(dtype, heads, kv_heads, dim, below, capacity):
    """One key takes nearly all, and thousands are `below` less than it, each of them below FP16's steps next to 1."""
    n = 4000
    cells = np.stack(np.unravel_index(np.arange(n), (4, 25, 40)), 1)
    qkv = np.zeros((n, (heads + 2 * kv_heads) * dim), np.float16 if dtype == HALF else np.float32)
    qkv[:, :heads * dim:dim] = 1.0
    qkv[77, heads * dim:(heads + kv_heads) * dim:dim] = below
    qkv[:, (heads + kv_heads) * dim:] = np.random.default_rng(0).uniform(0.5, 1.5, (n, kv_heads * dim))
    qkv[77, (heads + kv_heads) * dim:] = 0.0
    want, tol = A.one_window(qkv, cells, heads, kv_heads, dim, queries=[0])  # (all queries are the same)
    assert (tol <= want * 0.01 + 2.0 ** -24).all()
    assert_within(attend(qkv, cells, (4, 25, 40), heads, kv_heads, dim, capacity, softmax_scale=1.0), want, tol)
