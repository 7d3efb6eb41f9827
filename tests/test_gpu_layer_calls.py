"""RmsNorm, Linear8 and VoxelAttention on the GPU: calls that meet other calls, other streams, graphs and what a plugin is told between them."""
import numpy as np
import pytest
import torch

from gpu_util import DEV, dev
from sessd3d import api, ctypes_defs as D

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
        done = torch.cuda.Event()
        done.record()
        op.set_epilogue(new[0], new[1], relu=new[2])
        assert done.query()
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


def attention(rows, window=(4, 6, 6), heads=2, dim=16, **kw):
    return api.VoxelAttention(heads, heads, dim, (50, 40, 9), window[::-1], max_voxels=rows, **kw)


def attention_inputs(rows, heads=2, dim=16, seed=0, dtype=np.float16):
    rng = np.random.default_rng(seed)
    coors = np.zeros((rows, 4), np.int32)
    at = rng.choice(9 * 40 * 50, rows, replace=False)
    coors[:, 1], coors[:, 2], coors[:, 3] = at // 2000, at // 50 % 40, at % 50
    return dev(rng.standard_normal((rows, 3 * heads * dim)).astype(dtype)), dev(coors), num(rows)


@pytest.mark.parametrize("rows", [700, 5000])
def test_the_status_of_a_layer_on_shared_windows_is_that_of_those_windows(rows):
    x, c, n = attention_inputs(rows)
    first, second = attention(rows), attention(rows)
    with pytest.raises(api.SessdError, match="has not run"):
        second.status()
    first(x, c, n)
    second(x, c, n, windows_from=first)
    assert second.status() == 0
    bad = c.clone()
    bad[5, 1] = 9
    first(x, bad, n)
    second(x, bad, n, windows_from=first)
    assert second.status() == D.SESSD_STATUS_BAD_COORD
    second(x, c, n)          # alone again
    assert second.status() == 0 and first.status() == D.SESSD_STATUS_BAD_COORD
    ws = torch.empty_like(first.ws)
    out = torch.empty((rows, 32), dtype=HALF, device=DEV)
    second.enqueue([x, bad, n], [out], workspace=ws)
    assert second.status() == D.SESSD_STATUS_BAD_COORD
    with pytest.raises(api.SessdError, match="has not run"):
        second.clone().status()


@pytest.mark.parametrize("rows", [700, 5000])
def test_windows_of_a_call_that_was_refused_are_not_shared(rows):
    x, c, n = attention_inputs(rows)
    first, second, third = attention(rows), attention(rows), attention(rows)
    odd = torch.empty(x.numel() + 1, dtype=HALF, device=DEV)[1:].reshape(x.shape)
    with pytest.raises(api.SessdError, match="aligned"):
        first(odd, c, n)
    for layer in (first, first.clone()):
        with pytest.raises(api.SessdError, match="windows_from"):
            second(x, c, n, windows_from=layer)
    want = first(x, c, n)
    with pytest.raises(api.SessdError, match="windows_from"):
        second(x, c, n, windows_from=first.clone())
    with pytest.raises(api.SessdError, match="aligned"):
        second(odd, c, n, windows_from=first)
    with pytest.raises(api.SessdError, match="windows_from"):
        third(x, c, n, windows_from=second)
    # a sharer's windows can be shared, and so can those in a workspace of the caller's
    assert torch.equal(second(x, c, n, windows_from=first), want) and torch.equal(third(x, c, n, windows_from=second), want)
    ws, out = torch.empty_like(first.ws), torch.empty_like(want)
    y, d, m = attention_inputs(rows, seed=1)
    third.configure([y, d, m], [out])
    third.enqueue([y, d, m], [out], workspace=ws)
    first.ws.fill_(0x55)   # (what third's earlier calls went by)
    assert torch.equal(second(y, d, m, windows_from=third), out)


def test_layers_read_back_from_their_bytes_are_called_as_the_first_ones():
    rng = np.random.default_rng(0)
    rows = 300
    x, c, n = attention_inputs(rows)
    attn = attention(rows, slopes=[1.0, 0.5], cap=20.0, cell_size_xyz=(0.1, 0.1, 0.2))
    again = api.VoxelAttention.deserialize(attn.serialize())
    want = attn(x, c, n)
    assert torch.equal(again(x, c, n), want) and torch.equal(again(x, c, n, windows_from=attn), want)
    norm = api.RmsNorm(96, rng.uniform(0.5, 1.5, 96).astype(np.float32), max_voxels=rows)
    a, b = norm(x, n), api.RmsNorm.deserialize(norm.serialize())(x, n)
    assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(a, b))
    lin = api.Linear8(96, 40, rng.standard_normal((96, 40)).astype(np.float32), max_voxels=rows)
    lin.set_epilogue(None, rng.standard_normal(40).astype(np.float32), relu=True)
    assert torch.equal(api.Linear8.deserialize(lin.serialize())(*a, n), lin(*a, n))


def test_a_call_on_another_stream_takes_no_memory_of_the_current_one():
    """What was freed on the current stream may still be read there: outputs and workspaces of a call on another stream lie elsewhere."""
    rng = np.random.default_rng(0)
    rows = 5000
    x, c, n = attention_inputs(rows)
    q, s = linear_inputs(rows, 64)
    norm = api.RmsNorm(96, rng.uniform(0.5, 1.5, 96).astype(np.float32), max_voxels=rows)
    lin = api.Linear8(64, 160, rng.standard_normal((64, 160)).astype(np.float32), max_voxels=rows)
    side = torch.cuda.Stream()
    attn = attention(rows)
    want = norm(x, n, x) + (lin(q, s, n), attn(x, c, n))
    torch.cuda.synchronize()
    fresh = [attention(rows) for _ in range(2)]
    bytes_of = lambda t: t.untyped_storage().nbytes()  # noqa: E731
    freed = set()
    for t in [t for t in want + (attn.ws,) for _ in range(3)]:   # as large as what the calls below take
        block = torch.empty(bytes_of(t), dtype=torch.uint8, device=DEV)
        freed.add((block.data_ptr(), bytes_of(t)))
        del block
    side.wait_stream(torch.cuda.current_stream())
    got = norm(x, n, x, stream=side) + (lin(q, s, n, stream=side), fresh[0](x, c, n, stream=side))
    out = torch.empty_like(want[-1])
    fresh[1].configure([x, c, n], [out])
    fresh[1].enqueue([x, c, n], [out], side)
    for t in got + tuple(f.ws for f in fresh):
        a, b = t.data_ptr(), t.data_ptr() + bytes_of(t)
        assert not any(a < p + size and p < b for p, size in freed)
    assert torch.cuda.current_stream() != side
    side.synchronize()
    for a, b in zip(got + (out,), want + (want[-1],)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("rows", [1500, 6000])
def test_shared_windows_in_one_graph(rows):
    """A layer and a sharer of its windows, captured together and replayed on other frames."""
    x, c, n = attention_inputs(rows)
    first, second = attention(rows, slopes=[1.0, 2.0]), attention(rows, cap=20.0)
    eager = attention(rows, slopes=[1.0, 2.0]), attention(rows, cap=20.0)
    outs = [torch.empty((rows, 32), dtype=HALF, device=DEV) for _ in range(2)]
    first(x, c, n)
    second(x, c, n, windows_from=first)      # (workspace and descriptors are there)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        outs = first(x, c, n), second(x, c, n, windows_from=first)
    for k, m in enumerate((rows, 7, 0, rows - 5)):
        y, d, _ = attention_inputs(rows, seed=k)
        x.copy_(y)
        c.copy_(d)
        n.fill_(m)
        graph.replay()
        torch.cuda.synchronize()
        for got, op in zip(outs, eager):
            assert torch.equal(got, op(x, c, n))
        assert first.status() == second.status() == 0
