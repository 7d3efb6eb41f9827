"""RmsNorm on the GPU where the squares of a row are at the end of FP32 or beyond it, against its 64-bit restatement (layer_oracle.py)."""
import numpy as np
import pytest
import torch

import layer_oracle as L
from gpu_util import dev
from sessd3d import api

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eps", [0.0, 1e-44, 1e-37, 1e-30, 1e-6])
@pytest.mark.parametrize("c", [1, 8, 40, 65, 256, 1000, 4096])
def test_small_rows_and_small_eps(c, eps):
    """Rows of 1e-12 down to the smallest FP32: what is not all zeros has its norm, whatever eps is."""
    rng = np.random.default_rng(c)
    sizes = 10.0 ** -np.arange(12, 45, dtype=np.float64)
    feat = (np.maximum(np.abs(rng.standard_normal((len(sizes), c))), 0.25) * rng.choice([-1, 1], (len(sizes), c)) * sizes[:, None]).astype(np.float32)
    feat = np.concatenate([feat, np.full((1, c), 1e-45, np.float32), np.zeros((1, c), np.float32)])
    feat[:, 0] = np.where(feat[:, 0] == 0, np.float32(1e-45), feat[:, 0])
    feat[-1] = 0
    gamma = rng.uniform(0.5, 1.5, c).astype(np.float32)
    rows = len(feat)
    q, s = api.RmsNorm(c, gamma, max_voxels=rows, eps=eps)(dev(feat), dev(np.array([rows], np.int32)))
    q, s = q.view(torch.uint8).cpu().numpy(), s.cpu().numpy().astype(np.float64)
    want, scale, _ = L.norm(feat, None, gamma, float(np.float32(eps)))
    some = slice(0, rows - 1 if eps == 0 else rows)   # (0 / 0 has no value)
    assert (np.abs(s - scale) <= L.norm_scale_tolerance(c) * scale)[some].all(), np.nanmax(np.abs(s / scale - 1)[some])
    off = (q != L.to_e4m3(want))[some]
    assert (L.near_a_border(want[some][off]) | (want[some][off] == 0)).all()
    if eps == 0:
        assert np.isnan(s[-1]).all() and ((q[-1] & 0x7f) == 0x7f).all()
