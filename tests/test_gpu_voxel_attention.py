"""VoxelAttention on the GPU against its 64-bit restatement (layer_oracle.py), and a run of the layers together."""
import numpy as np
import pytest
import torch

import layer_oracle as L
from gpu_util import DEV, dev
from sessd3d import api, backbone as B, ctypes_defs as D, frames as F

pytestmark = pytest.mark.gpu
HALF, FLOAT = torch.float16, torch.float32
GRID = (9, 40, 50)  # z,y,x


def num(n):
    return dev(np.array([n], np.int32))


def make(rows, heads, kv_heads, dim, dtype, seed=0, grid=GRID, distinct=True, spread=1.0):
    rng = np.random.default_rng([seed, rows, heads, dim])
    coors = np.zeros((rows, 4), np.int32)
    cells = int(np.prod(grid))
    at = rng.choice(cells, rows, replace=not distinct or rows > cells)
    coors[:, 1], rest = np.divmod(at, grid[1] * grid[2])
    coors[:, 2], coors[:, 3] = np.divmod(rest, grid[2])
    qkv = (rng.standard_normal((rows, (heads + 2 * kv_heads) * dim)) * spread).astype(np.float16 if dtype == HALF else np.float32)
    return qkv, coors


class Case:
    def __init__(self, heads, kv_heads, dim, window, shift=(0, 0, 0), slopes=None, cap=0.0, scale=0.0, cell=(0.1, 0.05, 0.05), grid=GRID):
        self.heads, self.kv, self.dim, self.grid, self.window, self.shift = heads, kv_heads, dim, grid, window, shift
        self.slopes = None if slopes is None else np.asarray(slopes, np.float32)
        self.cap, self.scale, self.cell = cap, scale, cell

    def op(self, rows):
        return api.VoxelAttention(self.heads, self.kv, self.dim, self.grid[::-1], self.window[::-1], shift_xyz=self.shift[::-1], slopes=self.slopes,
                                  cell_size_xyz=self.cell[::-1], cap=self.cap, softmax_scale=self.scale, max_voxels=rows)

    def check(self, got, qkv, coors, n):
        n = min(max(n, 0), len(qkv))
        scale = np.float32(self.scale) if self.scale else np.float32(1 / np.sqrt(self.dim))
        want, tol = L.attention(qkv, coors, n, self.grid, self.window, self.shift, self.heads, self.kv, self.dim, self.slopes, self.cell,
                                float(np.float32(self.cap)), float(scale))
        g = got.cpu().numpy().astype(np.float64)
        assert np.array_equal(np.isnan(g), np.isnan(want))
        off = np.abs(g - want) > tol
        assert not off.any(), (int(off.sum()), np.argwhere(off)[:3], float((np.abs(g - want) / tol)[off].max()))


MANY = 4200  # rows of a tensor whose windows are listed; those of smaller ones are looked up by the attention itself


def run(case, rows, n, dtype, **kw):
    """The rows as they are, and at the front of a large tensor."""
    qkv, coors = make(rows, case.heads, case.kv, case.dim, dtype, **kw)
    for more in (0, MANY):
        if more:
            n = min(max(n, 0), rows)
            qkv = np.concatenate([qkv, np.full((more, qkv.shape[1]), np.nan, qkv.dtype)])
            coors = np.concatenate([coors, np.full((more, 4), -1, np.int32)])
        op = case.op(rows + more)
        got = op(dev(qkv), dev(coors), num(n))
        case.check(got, qkv, coors, n)
        assert op.status() == 0
    return got


@pytest.mark.parametrize("dim", [8, 16, 24, 32, 40, 56, 64, 96, 120, 128])
@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (8, 2), (5, 1)])
def test_heads(dim, dtype, heads, kv_heads):
    run(Case(heads, kv_heads, dim, (9, 10, 10), slopes=np.linspace(0.5, 3, heads), cap=20.0), 500, 490, dtype)


@pytest.mark.parametrize("rows,n", [(1, 1), (1, 0), (2, 2), (15, 15), (16, 16), (17, 17), (31, 30), (33, 33), (64, 64), (65, 65), (129, 128), (700, 700),
                                    (300, 0), (300, -2), (300, 900), (3000, 2999)])
@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("window", [(1, 1, 1), (9, 40, 50), (2, 7, 6)])
def test_rows_and_windows(rows, n, dtype, window):
    run(Case(4, 2, 16, window, slopes=[1, 2, 3, 4]), rows, n, dtype)


@pytest.mark.parametrize("rows,n,window", [(5000, 5000, (2, 2, 2)), (6000, 5900, (21, 30, 44)), (9000, 9000, (1, 1, 1)), (4097, 4097, (3, 5, 4))])
@pytest.mark.parametrize("dtype", [HALF, FLOAT])
def test_grids_of_many_windows(rows, n, window, dtype):
    """Up to 2^22 windows, and window counts either side of what is counted in LDS."""
    grid = (21, 300, 220)
    run(Case(2, 2, 16, window, slopes=[1.0, 0.5], grid=grid), rows, n, dtype, grid=grid)


@pytest.mark.parametrize("shift", [(0, 0, 0), (1, 0, 0), (0, 3, 5), (2, 6, 6), (1, 1, 1)])
@pytest.mark.parametrize("dtype", [HALF, FLOAT])
def test_shifted_windows(shift, dtype):
    run(Case(2, 2, 32, (3, 7, 7), shift=shift, slopes=[1.0, 0.25]), 1500, 1500, dtype)


@pytest.mark.parametrize("cap,slopes,scale", [(0.0, None, 0.0), (5.0, None, 0.0), (0.0, [2.0, -1.0], 0.0), (50.0, [0.0, 0.3], 0.5), (1000.0, None, -0.3), (0.01, [30.0, 1.0], 4.0)])
@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("window", [(9, 40, 50), (9, 8, 8)])
def test_caps_slopes_scales(cap, slopes, scale, dtype, window):
    run(Case(2, 1, 64, window, cap=cap, slopes=slopes, scale=scale), 900, 900, dtype)


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
def test_large_scores(dtype):
    """Scores of some thousands: one key takes all, nothing overflows."""
    run(Case(2, 2, 32, (9, 40, 50)), 400, 400, dtype, spread=25.0)


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
def test_rows_that_name_one_voxel(dtype):
    run(Case(2, 2, 16, (2, 2, 2), slopes=[1, 1], grid=(4, 4, 4)), 700, 700, dtype, grid=(4, 4, 4), distinct=False)


def test_long_windows_of_ragged_lengths():
    rng = np.random.default_rng(1)
    # windows of 1 .. 2200 rows side by side, their rows interleaved
    lengths = [1, 2, 2200, 31, 32, 33, 640, 5, 1, 1025, 63, 64, 65, 127, 129]
    grid = (16, 16, 16 * len(lengths))
    cells = []
    for i, m in enumerate(lengths):
        at = rng.choice(4096, m, replace=False)
        cells.append(np.stack([at // 256, at // 16 % 16, at % 16 + 16 * i], 1))
    cells = rng.permutation(np.concatenate(cells))
    rows = len(cells) + 5
    for dtype in (HALF, FLOAT):
        case = Case(4, 4, 24, (16, 16, 16), slopes=[0.3, 0.2, 0.1, 0.0], cap=30.0, grid=grid)
        qkv, coors = make(rows, 4, 4, 24, dtype)
        coors[:len(cells), 1:] = cells
        op = case.op(rows)
        case.check(op(dev(qkv), dev(coors), num(len(cells))), qkv, coors, len(cells))


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("window", [(9, 2, 2), (9, 4, 5), (9, 20, 25)])
@pytest.mark.parametrize("rows", [1200, MANY])
def test_what_is_not_finite_stays_in_its_window(dtype, window, rows):
    case = Case(2, 1, 16, window, slopes=[1.0, 0.5], cap=10.0)
    qkv, coors = make(rows, 2, 1, 16, dtype)
    op = case.op(rows)
    clean = op(dev(qkv), dev(coors), num(1150))
    bad_rows = (3, 400, 777)
    for row, bad in zip(bad_rows, (np.nan, np.inf, -np.inf)):
        qkv[row] = bad
    qkv[1150:] = np.nan     # rows behind the last
    coors[1150:] = -7
    got = op(dev(qkv), dev(coors), num(1150))
    win = coors[:1150, 1:] // np.array(window)
    touched = np.zeros(rows, bool)
    for row in bad_rows:
        touched[:1150] |= (win == win[row]).all(1)
    assert touched.sum() < 1150
    assert torch.equal(got[dev(~touched)], clean[dev(~touched)])
    # in the window of the NaN every row has it among its keys; what inf leaves is the formula's affair
    mine = np.zeros(rows, bool)
    mine[:1150] = (win == win[3]).all(1)
    assert torch.isnan(got[dev(mine)]).all()


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("rows", [300, MANY])
def test_a_row_outside_the_grid_takes_part_in_nothing(dtype, rows):
    case = Case(2, 2, 16, (9, 40, 50))
    qkv, coors = make(rows, 2, 2, 16, dtype)
    coors[5] = (0, 9, 0, 0)
    coors[17] = (0, 0, -1, 3)
    coors[18] = (1, 0, 1, 3)
    coors[299] = (0, 2 ** 31 - 1, -2 ** 31, 50)
    qkv[[5, 17, 18, 299]] = np.nan
    op = case.op(rows)
    op.set_flags(D.SESSD_FLAG_SKIP_PAD_ROWS)
    got = op(dev(qkv), dev(coors), num(300))[:300]  # (the rows behind it are anything)
    case.check(got, qkv[:300], coors, 300)
    assert not got[[5, 17, 18, 299]].any() and op.status() == D.SESSD_STATUS_BAD_COORD
    coors[:, 0] = 3         # every row
    assert not op(dev(qkv), dev(coors), num(300))[:300].any()
    coors[:, 0] = 0
    coors[[5, 17, 299], 1:] = 1
    op(dev(np.nan_to_num(qkv)), dev(coors), num(300))
    assert op.status() == 0


@pytest.mark.parametrize("rows", [200, MANY])
def test_rows_behind_the_last_are_left_as_they_were(rows):
    case = Case(2, 2, 24, (9, 8, 8))
    qkv, coors = make(rows, 2, 2, 24, HALF)
    op = case.op(rows)
    op.set_flags(D.SESSD_FLAG_SKIP_PAD_ROWS)
    out = torch.full((rows, 48), 7.0, dtype=HALF, device=DEV)
    ins = [dev(qkv), dev(coors), num(131)]
    op.configure(ins, [out])
    op.enqueue(ins, [out])
    assert (out[131:] == 7).all()
    case.check(torch.cat([out[:131], out[131:] * 0]), qkv, coors, 131)
    op.set_flags(0)
    op.enqueue(ins, [out])
    assert not out[131:].any()


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("window", [(9, 5, 5), (9, 40, 50)])
@pytest.mark.parametrize("rows", [2500, 5000])
def test_the_same_bits_each_time_and_on_shared_windows(dtype, window, rows):
    case = Case(8, 4, 32, window, slopes=np.linspace(0, 2, 8), cap=25.0)
    qkv, coors = make(rows, 8, 4, 32, dtype)
    x, c, n = dev(qkv), dev(coors), num(rows - 100)
    first, second = case.op(rows), case.op(rows)
    a = first(x, c, n)
    for _ in range(3):
        assert torch.equal(first(x, c, n), a)
    assert torch.equal(second(x, c, n, windows_from=first), a)
    other = Case(2, 2, 16, window)    # another layer on the same windows
    qkv2, _ = make(rows, 2, 2, 16, dtype)
    assert torch.equal(other.op(rows)(dev(qkv2), c, n, windows_from=first), other.op(rows)(dev(qkv2), c, n))
    # a row's bits follow from its window's rows, wherever else rows lie: the rows of the other windows leave
    if window == (9, 5, 5):
        keep = (coors[:rows - 100, 3] // 5) % 2 == 0
        got = first(x, dev(np.where(np.concatenate([keep, np.ones(100, bool)])[:, None], coors, -1).astype(np.int32)), n)
        assert torch.equal(got[:rows - 100][dev(keep)], a[:rows - 100][dev(keep)])


@pytest.mark.parametrize("rows,window", [(900, (9, 6, 6)), (MANY, (9, 6, 6)), (MANY, (1, 1, 1))])
def test_shared_windows_go_by_the_rows_they_were_found_for(rows, window):
    """voxel_num and coors that another frame has overwritten by the time of the sharer's call."""
    case = Case(2, 2, 16, window, grid=(9, 80, 80))  # (57 600 windows of one cell: by tickets)
    qkv, coors = make(rows, 2, 2, 16, HALF, grid=(9, 80, 80))
    coors[7, 1] = 9  # outside
    first, second = case.op(rows), case.op(rows)
    for m in (500, 0):
        c, n = dev(coors), num(m)
        a = first(dev(qkv), c, n)
        case.check(a, qkv, coors, m)
        for other in (rows, 3, -5):
            n.fill_(other)
            c.fill_(-1 if other == 3 else 2)
            assert torch.equal(second(dev(qkv), c, n, windows_from=first), a)


def test_windows_of_another_kind_are_not_shared():
    case = Case(2, 2, 16, (9, 6, 6))
    qkv, coors = make(100, 2, 2, 16, HALF)
    x, c, n = dev(qkv), dev(coors), num(100)
    op = case.op(100)
    for first, rows in ((Case(2, 2, 16, (9, 6, 6)), 90), (Case(2, 2, 16, (9, 6, 7)), 100), (Case(2, 2, 16, (9, 6, 6), shift=(0, 1, 0)), 100),
                        (Case(2, 2, 16, (9, 6, 6), grid=(9, 40, 51)), 100)):
        other = first.op(rows)
        other(x[:rows], c[:rows], n)
        with pytest.raises(api.SessdError, match="windows_from"):
            op(x, c, n, windows_from=other)
    with pytest.raises(api.SessdError, match="windows_from"):  # (has not run)
        op(x, c, n, windows_from=case.op(100))


def test_order_of_rows_does_not_choose_neighbours():
    """The same voxels in another order: the same outputs up to the order of their sums."""
    case = Case(2, 2, 16, (9, 6, 6), slopes=[1, 2])
    qkv, coors = make(2000, 2, 2, 16, FLOAT)
    p = np.random.default_rng(3).permutation(2000)
    op = case.op(2000)
    a = op(dev(qkv), dev(coors), num(2000)).cpu().numpy()
    b = op(dev(qkv[p]), dev(coors[p]), num(2000)).cpu().numpy()
    case.check(dev(b), qkv[p], coors[p], 2000)
    assert np.abs(a[p] - b).max() < 1e-4


@pytest.mark.parametrize("rows", [600, MANY])
def test_dirty_workspace_and_outputs(rows):
    case = Case(2, 2, 16, (9, 6, 6), slopes=[1, 2])
    qkv, coors = make(rows, 2, 2, 16, HALF)
    op = case.op(rows)
    ins = [dev(qkv), dev(coors), num(555)]
    for fill in (0xff, 0x7f, 0x01):
        out = torch.full((rows, 32), float("nan"), dtype=HALF, device=DEV)
        op.configure(ins, [out])
        ws = torch.full((op.workspace_size(ins, [out]),), fill, dtype=torch.uint8, device=DEV)
        op.enqueue(ins, [out], workspace=ws)
        case.check(out, qkv, coors, 555)


@pytest.mark.parametrize("rows", [4000, 8000])
def test_two_calls_at_once(rows):
    """Two layers on two streams, each with a workspace of its own."""
    case = Case(4, 4, 16, (9, 8, 8), slopes=[1, 1, 2, 2])
    qkv, coors = make(rows, 4, 4, 16, HALF)
    qkv2, coors2 = make(rows, 4, 4, 16, HALF, seed=9)
    a, b = case.op(rows), case.op(rows)
    one, two = (dev(qkv), dev(coors), num(rows - 100)), (dev(qkv2), dev(coors2), num(rows))
    want = a(*one).clone(), b(*two).clone()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        with torch.cuda.stream(s):
            outs[0].append(a(*one))
        with torch.cuda.stream(t):
            outs[1].append(b(*two))
    torch.cuda.synchronize()
    for got, w in zip(outs, want):
        for g in got:
            assert torch.equal(g, w)


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("heads,kv_heads,dim", [(13, 13, 16), (24, 3, 32), (16, 16, 128), (2, 1, 128), (1, 1, 64)])
@pytest.mark.parametrize("window", [(9, 40, 50), (9, 9, 9)])
def test_few_rows_and_many_heads(dtype, heads, kv_heads, dim, window):
    """Rows times heads either side of where a query's keys are shared out among the waves."""
    rows = 2600
    qkv, coors = make(rows, heads, kv_heads, dim, dtype)
    case = Case(heads, kv_heads, dim, window, slopes=np.linspace(0, 1, heads))
    op = case.op(rows)
    got = op(dev(qkv), dev(coors), num(rows - 1))
    case.check(got, qkv, coors, rows - 1)
    assert torch.equal(op(dev(qkv), dev(coors), num(rows - 1)), got)


def test_rows_beyond_32_bit_offsets():
    """qkv of more than 2^31 elements: the windows of the last rows."""
    rows, heads, dim = 360000, 16, 128
    n = 64
    case = Case(heads, heads, dim, (1, 4, 4), grid=(1, 600, 600))
    x = torch.zeros((rows, 3 * heads * dim), dtype=HALF, device=DEV)
    tail = np.random.default_rng(0).standard_normal((n, 3 * heads * dim)).astype(np.float16)
    x[-n:] = dev(tail)
    coors = np.zeros((rows, 4), np.int32)
    coors[:, 2], coors[:, 3] = np.divmod(np.arange(rows), 600)
    # the last 64 rows fill four windows of a band of their own
    at = np.arange(rows - 600 * 4, rows).reshape(4, 600)[:, -16:].reshape(-1)
    rest = np.setdiff1d(np.arange(rows), at)
    coors = coors[np.concatenate([rest, at])]
    got = case.op(rows)(x, dev(coors), num(rows))
    case.check(got[-n:], tail, coors[-n:], n)
    assert not got[:-n].any()


@pytest.mark.parametrize("rows", [1500, MANY])
def test_under_a_graph(rows):
    case = Case(4, 2, 16, (9, 8, 8), slopes=[1, 1, 2, 2], cap=20.0)
    qkv, coors = make(rows, 4, 2, 16, HALF)
    x, c, n = dev(qkv), dev(coors), num(1400)
    op, eager_op = case.op(rows), case.op(rows)
    out = torch.empty((rows, 64), dtype=HALF, device=DEV)
    eager = torch.empty_like(out)
    ws = torch.empty(op.workspace_size([x, c, n], [out]), dtype=torch.uint8, device=DEV)
    for o in (op, eager_op):
        o.configure([x, c, n], [out])
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        op.enqueue([x, c, n], [out], side, workspace=ws)
    rng = np.random.default_rng(0)
    for k in range(4):
        m = (1400, rows, 3, 700)[k]
        p = rng.permutation(rows)
        x.copy_(dev(qkv[p]))
        c.copy_(dev(coors[p]))
        n.copy_(num(m))
        graph.replay()
        eager_op.enqueue([x, c, n], [eager])
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        case.check(out, qkv[p], coors[p], m)


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
def test_a_block_behind_the_convolutions(dtype):
    """Points -> voxels -> SubM layer -> norm, query / key / value, attention, norm, projection, norm with the residual, feed-forward part ->
    SubM layer: every layer of the block on the GPU's own rows of the layer before it, against its 64-bit restatement."""
    max_voxels = 3000
    grid_xyz = (1408, 1600, 41)
    pts = F.lidar_frame(2500, 4)
    vg = api.VoxelGenerator(max_voxels=max_voxels)
    buf = np.zeros((2600, 4), np.float32)
    buf[:len(pts)] = pts
    voxels, coors, n_dev = vg(dev(buf), num(len(pts)))
    rng = np.random.default_rng(0)
    c, heads, kv, dim = 64, 4, 2, 16
    stem = api.SubmConv3d(4, c, grid_xyz, (rng.standard_normal((27, 4, c)) * 0.2).astype(np.float32), max_voxels)
    feat = stem(voxels, coors, n_dev).to(dtype)
    n = int(n_dev.item())
    assert 1000 < n < max_voxels
    w = lambda i, o: (rng.standard_normal((i, o)) / np.sqrt(i)).astype(np.float32)  # noqa: E731
    gamma = lambda k: rng.uniform(0.5, 1.5, k).astype(np.float32)  # noqa: E731
    case = Case(heads, kv, dim, (41, 64, 64), shift=(0, 32, 32), slopes=[1.0, 0.5, 0.25, 0.1], cap=30.0, grid=grid_xyz[::-1])

    def norm(x, residual=None):
        g = gamma(x.shape[1])
        got = api.RmsNorm(x.shape[1], g, max_voxels=max_voxels)(x, n_dev, residual)
        a = lambda t: None if t is None else t.cpu().numpy()  # noqa: E731
        want, s, h = L.norm(a(x)[:n], None if residual is None else a(residual)[:n], g, 1e-6)
        codes = got[0].view(torch.uint8).cpu().numpy()[:n]
        off = codes != L.to_e4m3(want)
        assert (L.near_a_border(want[off]) | (want[off] == 0)).all()
        assert (np.abs(a(got[1])[:n] - s) <= L.norm_scale_tolerance(x.shape[1]) * s).all()
        if residual is not None:
            assert np.array_equal(a(got[2])[:n], h.astype(a(x).dtype))
        return got

    def linear(q, s, cout, relu=False):
        cin = q.shape[1]
        m = w(cin, cout)
        op = api.Linear8(cin, cout, m, max_voxels=max_voxels)
        shift = rng.uniform(-0.2, 0.2, cout).astype(np.float32)
        op.set_epilogue(None, shift, relu=relu)
        got = op(q, s, n_dev, out_dtype=dtype)
        want, magnitude = L.linear(q.view(torch.uint8).cpu().numpy()[:n], s.cpu().numpy()[:n], m, None, shift, relu)
        assert (np.abs(got.cpu().numpy()[:n] - want) <= L.linear_tolerance(want, magnitude, cin, dtype == HALF)).all()
        return got

    q, s = norm(feat)
    qkv = linear(q, s, (heads + 2 * kv) * dim)
    attn = case.op(max_voxels)
    a = attn(qkv, coors, n_dev)
    case.check(a, qkv.cpu().numpy(), coors.cpu().numpy(), n)
    assert attn.status() == 0
    o = linear(*norm(a), c)
    q, s, x = norm(o, feat)
    hidden = linear(q, s, 4 * c, relu=True)
    down = linear(*norm(hidden), c)
    q, s, x = norm(down, x)
    behind = api.SubmConv3d(c, 16, grid_xyz, (rng.standard_normal((27, c, 16)) * 0.05).astype(np.float32), max_voxels)(x, coors, n_dev)
    assert torch.isfinite(behind.float()).all() and behind[:n].float().abs().sum() > 0 and not x[n:].any()
