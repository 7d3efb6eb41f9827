"""VoxelAttention on the GPU where a workgroup takes two heads: FP16 tensors of 200 000 rows times heads and more, with few rows that count."""
import numpy as np
import pytest
import torch

import attention_bounds as A
from gpu_util import DEV, dev
from sessd3d import api

pytestmark = pytest.mark.gpu
GRID = (9, 40, 50)
REGION = (9, 20, 25)  # where the voxels are


def run(n, heads, kv_heads, dim, window, region=REGION, seed=0, **kw):
    rng = np.random.default_rng([seed, n, heads, dim])
    rows = 200000 // heads + 7
    cells = np.stack(np.unravel_index(rng.choice(int(np.prod(region)), n, replace=False), region), 1)
    qkv = rng.standard_normal((n, (heads + 2 * kv_heads) * dim)).astype(np.float16)
    x = torch.full((rows, qkv.shape[1]), float("nan"), dtype=torch.float16, device=DEV)
    coors = torch.full((rows, 4), -1, dtype=torch.int32, device=DEV)
    x[:n], coors[:n, 0], coors[:n, 1:] = dev(qkv), 0, dev(cells.astype(np.int32))
    num = dev(np.array([n], np.int32))
    size = kw.pop("cell", (0.1, 0.05, 0.05))
    op = api.VoxelAttention(heads, kv_heads, dim, GRID[::-1], window[::-1], cell_size_xyz=size[::-1], max_voxels=rows, **kw)
    out = op(x, coors, num)
    assert op.status() == 0 and not out[n:].any()
    assert torch.equal(op(x, coors, num), out)
    scale = float(np.float32(kw["softmax_scale"])) if kw.get("softmax_scale") else 1 / np.sqrt(dim)
    at, want, tol = A.windows(qkv, cells, window, heads, kv_heads, dim, slopes=kw.get("slopes"), cell=size, cap=kw.get("cap", 0.0), scale=scale)
    got = out[:n].cpu().numpy()[at].astype(np.float64)
    off = ~(np.abs(got - want) <= tol)
    assert not off.any(), (int(off.sum()), float((np.abs(got - want) / tol)[off].max()))


# of 1 to 9, some 36, some 150, all rows
@pytest.mark.parametrize("window", [(1, 3, 3), (9, 2, 3), (9, 5, 5), (9, 40, 50)])
@pytest.mark.parametrize("dim", [8, 16, 24, 32, 40, 64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (3, 3), (5, 1), (6, 3), (8, 2), (6, 2)])
@pytest.mark.parametrize("bias", [False, True])
def test_heads_and_windows(window, dim, heads, kv_heads, bias):
    kw = dict(slopes=np.linspace(0.5, 3, heads).astype(np.float32), cap=20.0) if bias else {}
    run(3000, heads, kv_heads, dim, window, **kw)


@pytest.mark.parametrize("cap,scale", [(0.0, -0.4), (1000.0, 0.0), (5.0, 0.7)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (3, 3, 32)])
def test_caps_and_scales(cap, scale, heads, kv_heads, dim):
    run(2100, heads, kv_heads, dim, (9, 4, 25), cap=cap, softmax_scale=scale, slopes=[1.0, -0.5, 0.0, 3.0][:heads])


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 32, 33, 48, 49, 64, 65, 127, 128, 129, 200, 257])
@pytest.mark.parametrize("heads,kv_heads,dim", [(3, 3, 16), (4, 1, 64)])
def test_rows_of_one_window(n, heads, kv_heads, dim):
    """Either side of a tile, of a block of keys, of what is tiny, short and long."""
    run(n, heads, kv_heads, dim, GRID, slopes=np.ones(heads, np.float32))


@pytest.mark.parametrize("heads,kv_heads,dim,window", [(8, 4, 16, (9, 40, 50)), (7, 7, 32, (9, 40, 50)), (8, 2, 64, (9, 3, 4)), (9, 9, 16, (9, 3, 4)), (8, 8, 24, (9, 10, 10))])
def test_work_for_the_whole_card(heads, kv_heads, dim, window):
    """More than 1 024 pairs of an item of 64 queries and two heads, long items or short ones: workgroups with two heads, and an odd last one."""
    run(17000, heads, kv_heads, dim, window, region=GRID, slopes=np.linspace(0, 1, heads).astype(np.float32))
