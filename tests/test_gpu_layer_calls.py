"""RmsNorm, Linear8 and VoxelAttention on the GPU: calls that meet other calls, other streams, graphs and what a plugin is told between them."""
import numpy as np
import pytest
import torch

from gpu_util import DEV, dev
from sessd3d import api

pytestmark = pytest.mark.gpu
HALF, FLOAT = torch.float16, torch.float32


def num(n):
    return dev(np.array([n], np.int32))


def linear_inputs(rows, cin, seed=0):
    rng = np.random.default_rng(seed)
    q = rng.integers(0, 256, (rows, cin)).astype(np.uint8)
    q[(q & 0x7f) == 0x7f] = 0x11
    return dev(q).view(torch.float8_e4m3fn), dev((2.0 ** rng.uniform(-6, -3, (rows, 1))).astype(np.float32))


@pytest.mark.parametrize("cin,cout", [(256, 1024), (1040, 200)])
def test_a_new_epilogue_waits_for_the_calls_that_have_the_old_one(cin, cout):
    rng = np.random.default_rng(1)
    rows = 40000
    q, s = linear_inputs(rows, cin)
    n = num(rows)
    op = api.Linear8(cin, cout, (rng.standard_normal((cin, cout)) / 16).astype(np.float32), max_voxels=rows)
    a, b = rng.uniform(0.5, 1.5, (2, cout)).astype(np.float32)
    old, new = (a, b, True), (-b, None, False)
    want = []
    for e in (new, old):
        op.set_epilogue(*e[:2], relu=e[2])
        want.append(op(q, s, n))
    assert not torch.equal(*want)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        queued = [op(q, s, n) for _ in range(12)]
        op.set_epilogue(new[0], new[1], relu=new[2])
        behind = op(q, s, n)
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[1]) for x in queued) and torch.equal(behind, want[0])


def test_a_captured_call_has_a_new_epilogue_as_a_whole():
    rng = np.random.default_rng(2)
    rows = 3000
    q, s = linear_inputs(rows, 64)
    op = api.Linear8(64, 192, rng.standard_normal((64, 192)).astype(np.float32), max_voxels=rows)
    out, n = torch.empty((rows, 192), dtype=HALF, device=DEV), num(2900)
    op.configure([q, s, n], [out])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        op.enqueue([q, s, n], [out], torch.cuda.current_stream())
    for relu, with_scale, with_shift in ((True, True, True), (False, False, True), (True, False, False), (False, True, False)):
        scale, shift = rng.uniform(-1.5, 1.5, (2, 192)).astype(np.float32)
        op.set_epilogue(scale if with_scale else None, shift if with_shift else None, relu=relu)
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        op.enqueue([q, s, n], [out])
        torch.cuda.synchronize()
        assert torch.equal(out, replayed) and bool((out < 0).any()) != relu
