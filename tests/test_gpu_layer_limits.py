"""RmsNorm, Linear8 and VoxelAttention on the GPU with as many rows and windows as they take, against plain torch in FP32 and 64 bits."""
import numpy as np
import pytest
import torch

from gpu_util import DEV, dev
from sessd3d import api

pytestmark = pytest.mark.gpu
MOST = 1 << 24


def num(n):
    return dev(np.array([n], np.int32))


def random_halves(rows, columns, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return torch.randn((rows, columns), generator=g, device=DEV).half()


def test_norm_and_linear_of_2_24_rows():
    c = 8
    x = random_halves(MOST, c, 0)
    n = MOST - 3
    q, s = api.RmsNorm(c, np.ones(c, np.float32), max_voxels=MOST)(x, num(n))
    y = x.double()
    y = y / torch.sqrt((y * y).mean(1, keepdim=True) + float(np.float32(1e-6)))
    scale = y.abs().amax(1, keepdim=True) / 448
    assert ((s[:n] - scale[:n]).abs() <= 16 * 2.0 ** -24 * scale[:n]).all() and not s[n:].any()
    # a value is within half a step of e4m3 (2^-4 of itself, 2^-10 below 2^-6) of the quotient
    off = (q[:n].float() - (y / scale)[:n]).abs()
    assert (off <= (y / scale)[:n].abs() * 2.0 ** -4 * (1 + 2.0 ** -20) + 2.0 ** -10).all() and not q[n:].float().any()
    del y, scale, off
    q16 = torch.cat([q, q], 1)
    del q, x
    w = np.random.default_rng(0).standard_normal((16, 8)).astype(np.float32)
    op = api.Linear8(16, 8, w, max_voxels=MOST)
    got = op(q16, s, num(n))
    ws = np.maximum(np.abs(w).max(0) / np.float32(448), np.float32(2.0 ** -100))
    wq = torch.from_numpy(w / ws).to(torch.float8_e4m3fn).double().to(DEV) * torch.from_numpy(ws).double().to(DEV)
    for at in range(0, MOST, 1 << 22):
        part = slice(at, min(at + (1 << 22), n))
        a, b = q16[part].double(), s[part].double()
        want, magnitude = (a @ wq) * b, (a.abs() @ wq.abs()) * b
        assert ((got[part] - want).abs() <= magnitude * 21 * 2.0 ** -24 + want.abs() * 2.0 ** -11 + 2.0 ** -25).all()
    assert not got[n:].any()


@pytest.mark.parametrize("window", [(1, 2, 2), (1, 8, 16)])
def test_attention_of_2_24_rows(window):
    """A grid without an empty cell, its rows in any order: 2^22 windows of four rows, and 2^17 of 128."""
    d, side = 8, 4096
    x = random_halves(MOST, 3 * d, 1)
    g = torch.Generator(device=DEV)
    g.manual_seed(2)
    cell = torch.randperm(MOST, generator=g, device=DEV)   # of a row
    coors = torch.zeros((MOST, 4), dtype=torch.int32, device=DEV)
    coors[:, 2], coors[:, 3] = cell // side, cell % side
    op = api.VoxelAttention(1, 1, d, (side, side, 1), window[::-1], slopes=[0.5], max_voxels=MOST)
    got = op(x, coors, num(MOST))
    assert op.status() == 0
    at = torch.empty(MOST, dtype=torch.int64, device=DEV)
    at[cell] = torch.arange(MOST, device=DEV)               # row of a cell
    h, w = window[1:]
    rows = at.reshape(side // h, h, side // w, w).permute(0, 2, 1, 3).reshape(-1, h * w)
    place = torch.stack([torch.arange(h * w, device=DEV) // w, torch.arange(h * w, device=DEV) % w], 1).float()
    far = ((place[:, None] - place[None]) ** 2).sum(2).sqrt()
    step = (1 << 22) // (h * w)
    for i in range(0, len(rows), step):
        part = rows[i:i + step]
        q, k, v = x[part].float().split(d, 2)
        p = torch.softmax((q[:, :, None] * k[:, None]).sum(3) * d ** -0.5 - 0.5 * far, 2)
        o, a = ((p[..., None] * t[:, None]).sum(2) for t in (v, v.abs()))
        # weights of 11 bits in numerator and denominator, scores below 32 within 2^-17, the output's rounding
        assert ((got[part].float() - o).abs() <= (a + o.abs()) * (2.0 ** -10 + 2.0 ** -16) + o.abs() * 2.0 ** -11 + 2.0 ** -25).all()
