"""Linear8 on the GPU with so many rows that a wave takes several blocks of them, for every number of input channels that has a kernel of its own."""
import numpy as np
import pytest
import torch

import layer_oracle as L
from gpu_util import dev
from sessd3d import api

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cin,cout", [(64, 64), (48, 200), (128, 384), (112, 9), (192, 72), (256, 1024), (240, 33), (320, 96), (384, 200), (352, 130), (448, 72),
                                      (512, 128), (496, 1000), (1024, 256), (2048, 40)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_rows_of_several_rounds(cin, cout, dtype):
    columns = 32 if 256 < cin <= 512 else 64          # of a wave; 512 workgroups of four share the columns out and then the rows
    rows = int(2.6 * 16 * (2048 // -(-cout // columns)))
    n = rows - 21
    rng = np.random.default_rng(cin)
    q = rng.integers(0, 256, (rows, cin)).astype(np.uint8)
    q[(q & 0x7f) == 0x7f] = 0x11
    s = (2.0 ** rng.uniform(-8, -1, (rows, 1))).astype(np.float32)
    w = (rng.standard_normal((cin, cout)) / np.sqrt(cin)).astype(np.float32)
    scale, shift = rng.uniform(0.5, 1.5, cout).astype(np.float32), rng.uniform(-1, 1, cout).astype(np.float32)
    op = api.Linear8(cin, cout, w, max_voxels=rows)
    op.set_epilogue(scale, shift, relu=True)
    got = op(dev(q).view(torch.float8_e4m3fn), dev(s), dev(np.array([n], np.int32)), out_dtype=dtype).cpu().numpy().astype(np.float64)
    q[n:], s[n:] = 0, 0
    want, magnitude = L.linear(q, s, w, scale, shift, True)
    tol = L.linear_tolerance(want, magnitude, cin, dtype == torch.float16)
    ok = np.abs(got - want) <= tol
    if dtype == torch.float16:  # (those that FP16 may round to infinity)
        ok |= (want + tol >= 65504) & (got >= 65504 - 32)
    assert ok.all(), (int((~ok).sum()), np.argwhere(~ok)[:3])
