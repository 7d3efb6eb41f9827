"""RmsNorm and Linear8 on the GPU against their 64-bit restatements (layer_oracle.py)."""
import numpy as np
import pytest
import torch

import layer_oracle as L
from gpu_util import DEV, dev
from sessd3d import api, ctypes_defs as D

pytestmark = pytest.mark.gpu
HALF, FLOAT = torch.float16, torch.float32


def np_type(t):
    return np.float16 if t == HALF else np.float32


def num(n):
    return dev(np.array([n], np.int32))


def codes(t):
    return t.view(torch.uint8).cpu().numpy()


def assert_norm(got, feat, residual, gamma, eps, n):
    """Rows < n against the formula, the others zeros."""
    q, scale = codes(got[0]), got[1].cpu().numpy()
    want, s, h = L.norm(feat[:n], None if residual is None else residual[:n], gamma, eps)
    assert (q[n:] == 0).all() and (scale[n:] == 0).all()
    with np.errstate(invalid="ignore", over="ignore"):
        finite = np.isfinite(s[:, 0]) & np.isfinite(h).all(1) & (np.square(h).sum(1) < 3e38)
    assert np.isnan(scale[:n][~finite]).all() and ((q[:n][~finite] & 0x7f) == 0x7f).all()
    tol = L.norm_scale_tolerance(feat.shape[1])
    assert (np.abs(scale[:n][finite] - s[finite]) <= tol * s[finite]).all()
    off = (q[:n] != L.to_e4m3(want)) & finite[:, None]
    # (codes may differ where the quotient's FP32 form lies on a border of two values; zeros by their sign)
    assert (L.near_a_border(want[off]) | (want[off] == 0)).all(), (int(off.sum()), want[off][:4], L.VALUES[q[:n][off]][:4])
    if residual is not None:
        with np.errstate(over="ignore"):
            assert np.array_equal(got[2].cpu().numpy()[:n], h.astype(feat.dtype), equal_nan=True)
        assert not got[2][n:].any()


def norm_inputs(rng, rows, c, dtype, residual):
    t = np_type(dtype)
    feat = rng.standard_normal((rows, c)).astype(t)
    res = (rng.standard_normal((rows, c)) * 3).astype(t) if residual else None
    return feat, res, rng.uniform(0.5, 1.5, c).astype(np.float32) * rng.choice([-1, 1], c).astype(np.float32)


@pytest.mark.parametrize("c", [1, 5, 8, 16, 24, 32, 56, 64, 65, 96, 128, 200, 250, 256, 264, 512, 520, 1000, 1001, 1024, 2048, 4095, 4096])
@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_widths(c, dtype, residual):
    rng = np.random.default_rng(c)
    feat, res, gamma = norm_inputs(rng, 70, c, dtype, residual)
    op = api.RmsNorm(c, gamma, max_voxels=70, eps=1e-5)
    assert_norm(op(dev(feat), num(67), None if res is None else dev(res)), feat, res, gamma, 1e-5, 67)


@pytest.mark.parametrize("rows,n", [(1, 1), (1, 0), (3, 3), (64, 63), (257, 257), (300, 0), (300, 1000), (300, -5), (20000, 16825)])
@pytest.mark.parametrize("dtype", [HALF, FLOAT])
def test_norm_rows(rows, n, dtype):
    rng = np.random.default_rng(rows)
    feat, res, gamma = norm_inputs(rng, rows, 64, dtype, True)
    op = api.RmsNorm(64, gamma, max_voxels=rows)
    assert_norm(op(dev(feat), num(n), dev(res)), feat, res, gamma, 1e-6, min(max(n, 0), rows))


def test_norm_rows_of_zeros_small_large_and_not_finite():
    feat = np.zeros((12, 40), np.float32)
    feat[1, 3] = 1e-30
    feat[2] = 1e-20
    feat[3] = np.linspace(-1e15, 1e15, 40)
    feat[4, 7] = np.nan
    feat[5, 39] = np.inf
    feat[6, 0] = -np.inf
    feat[7] = 3e38             # its squares are not
    feat[8, 5] = 1.0
    feat[9] = np.repeat([2.0, -2.0], 20)
    feat[10] = 1e-45
    gamma = np.ones(40, np.float32)
    gamma[5] = 0.0
    op = api.RmsNorm(40, gamma, max_voxels=12, eps=1e-6)
    got = op(dev(feat), num(12))
    assert_norm(got, feat, None, gamma, 1e-6, 12)
    s = got[1].cpu().numpy()[:, 0]
    assert s[0] == np.float32(2.0 ** -100) and s[8] == np.float32(2.0 ** -100) and np.isnan(s[4:8]).all()
    assert (codes(got[0])[[0, 8]] & 0x7f == 0).all()
    # FP16 values whose sum is beyond FP16: the norm is that of the sum, the stored sum infinite
    f = np.full((1, 16), 60000, np.float16)
    got = api.RmsNorm(16, np.ones(16, np.float32), max_voxels=1)(dev(f), num(1), dev(f))
    assert torch.isinf(got[2]).all() and (codes(got[0]) == 0x7e).all()


def test_norm_with_eps_zero_gives_rows_of_zeros_no_value():
    feat = np.zeros((2, 8), np.float32)
    feat[1] = 2.0
    q, s = api.RmsNorm(8, np.ones(8, np.float32), max_voxels=2, eps=0.0)(dev(feat), num(2))
    assert torch.isnan(s[0]).all() and (codes(q)[0] & 0x7f == 0x7f).all() and (codes(q)[1] == 0x7e).all()


@pytest.mark.parametrize("onto", ["feat", "residual"])
@pytest.mark.parametrize("c", [64, 37])
def test_norm_sum_in_place(onto, c):
    rng = np.random.default_rng(3)
    feat, res, gamma = norm_inputs(rng, 90, c, HALF, True)
    op = api.RmsNorm(c, gamma, max_voxels=90)
    f, r = dev(feat), dev(res)
    apart = op(f, num(80), r)
    q, s = torch.empty_like(apart[0]), torch.empty_like(apart[1])
    target = f if onto == "feat" else r
    op.enqueue([f, num(80), r], [q, s, target])
    assert torch.equal(codes_t(q), codes_t(apart[0])) and torch.equal(s, apart[1]) and torch.equal(target, apart[2])


def codes_t(t):
    return t.view(torch.uint8)


def test_norm_leaves_rows_behind_the_last_as_they_were():
    op = api.RmsNorm(48, np.ones(48, np.float32), max_voxels=100)
    op.set_flags(D.SESSD_FLAG_SKIP_PAD_ROWS)
    f = torch.randn(100, 48, device=DEV).half()
    outs = [torch.full((100, 48), 0x55, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn), torch.full((100, 1), 7.0, device=DEV),
            torch.full((100, 48), 7.0, dtype=HALF, device=DEV)]
    ins = [f, num(61), f.clone()]
    op.configure(ins, outs)
    op.enqueue(ins, outs)
    assert (codes(outs[0])[61:] == 0x55).all() and (outs[1][61:] == 7).all() and (outs[2][61:] == 7).all()
    assert torch.equal(outs[2][:61], f[:61] * 2)


def linear_inputs(rng, rows, cin, cout):
    q = rng.integers(0, 256, (rows, cin)).astype(np.uint8)
    q[(q & 0x7f) == 0x7f] = 0x11
    s = (2.0 ** rng.uniform(-6, 3, (rows, 1))).astype(np.float32)
    w = (rng.standard_normal((cin, cout)) / np.sqrt(cin)).astype(np.float32)
    return q, s, w


def e4m3(q):
    return dev(q).view(torch.float8_e4m3fn)


def assert_linear(got, want, magnitude, cin):
    half = got.dtype == HALF
    tol = L.linear_tolerance(want, magnitude, cin, half)
    g = got.cpu().numpy().astype(np.float64)
    big = np.abs(want) + tol >= 65504 if half else np.zeros(want.shape, bool)   # (FP16 may round those to infinity)
    off = (np.abs(g - want) > tol) & ~big
    assert not off.any(), (int(off.sum()), float((np.abs(g - want) / tol)[off].max()))


@pytest.mark.parametrize("cin,cout", [(16, 1), (16, 16), (16, 7), (32, 64), (48, 65), (64, 192), (80, 24), (128, 384), (144, 100), (256, 1024),
                                      (512, 128), (1040, 33), (4096, 72), (64, 4096)])
@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("epilogue", ["none", "shift", "relu"])
def test_linear_widths(cin, cout, dtype, epilogue):
    rng = np.random.default_rng(cin * 5000 + cout)
    q, s, w = linear_inputs(rng, 150, cin, cout)
    scale = rng.uniform(0.5, 1.5, cout).astype(np.float32) if epilogue == "relu" else None
    shift = rng.uniform(-1, 1, cout).astype(np.float32) if epilogue != "none" else None
    op = api.Linear8(cin, cout, w, max_voxels=150)
    if epilogue != "none":
        op.set_epilogue(scale, shift, relu=epilogue == "relu")
    got = op(e4m3(q), dev(s), num(133), out_dtype=dtype)
    qz, sz = q.copy(), s.copy()
    qz[133:], sz[133:] = 0, 0
    want, magnitude = L.linear(qz, sz, w, scale, shift, epilogue == "relu")
    assert_linear(got, want, magnitude, cin)


@pytest.mark.parametrize("rows,n", [(1, 1), (1, 0), (15, 15), (17, 16), (63, 63), (64, 64), (65, 65), (129, 1), (1000, -3), (1000, 5000), (20000, 16825)])
@pytest.mark.parametrize("dtype", [HALF, FLOAT])
def test_linear_rows(rows, n, dtype):
    rng = np.random.default_rng(rows)
    q, s, w = linear_inputs(rng, rows, 64, 96)
    got = api.Linear8(64, 96, w, max_voxels=rows)(e4m3(q), dev(s), num(n), out_dtype=dtype)
    n = min(max(n, 0), rows)
    q[n:], s[n:] = 0, 0
    want, magnitude = L.linear(q, s, w)
    assert_linear(got, want, magnitude, 64)


def test_linear_knows_every_e4m3_value_of_rows_and_weights():
    """Row i has value i in one place, the weights are ones there: the products are the values.  And the other way round."""
    q = np.zeros((256, 16), np.uint8)
    q[:, 5] = np.arange(256)
    w = np.zeros((16, 8), np.float32)
    w[5] = 1.0
    got = api.Linear8(16, 8, w, max_voxels=256)(e4m3(q), torch.full((256, 1), 448.0, device=DEV), num(256), out_dtype=FLOAT)
    values = L.VALUES * 448.0 * 448.0 * np.float64(np.float32(1.0) / np.float32(448.0))
    got = got.cpu().numpy()
    assert np.isnan(got[[0x7f, 0xff]]).all()
    rest = ~np.isnan(values)
    assert np.allclose(got[rest], values[rest][:, None], rtol=4 * L.U, atol=0)
    # weights: a column each, scaled by 448 so that wscale is exactly 1; halves between two values go to the even one
    w = np.zeros((16, 512), np.float32)
    w[0, :256] = np.nan_to_num(L.VALUES)
    mid = np.unique(np.abs(np.nan_to_num(L.VALUES)))
    w[0, 256:256 + len(mid) - 1] = (mid[1:] + mid[:-1]) / 2
    w[1] = 448.0
    q = np.zeros((1, 16), np.uint8)
    q[0, 0] = 0x38  # 1.0
    got = api.Linear8(16, 512, w, max_voxels=1)(e4m3(q), torch.ones((1, 1), device=DEV), num(1), out_dtype=FLOAT).cpu().numpy()[0]
    assert np.array_equal(got, L.VALUES[L.to_e4m3(w[0])].astype(np.float32))


def test_linear_rows_that_are_not_finite_stay_in_their_rows():
    rng = np.random.default_rng(0)
    q, s, w = linear_inputs(rng, 64, 32, 48)
    clean = api.Linear8(32, 48, w, max_voxels=64)(e4m3(q), dev(s), num(64), out_dtype=FLOAT)
    q[7, 3], s[21] = 0x7f, np.nan
    s[30] = np.inf
    op = api.Linear8(32, 48, w, max_voxels=64)
    got = op(e4m3(q), dev(s), num(64), out_dtype=FLOAT)
    assert torch.isnan(got[[7, 21]]).all() and not torch.isfinite(got[30]).any()
    rest = [i for i in range(64) if i not in (7, 21, 30)]
    assert torch.equal(got[rest], clean[rest])
    op.set_epilogue(None, None, relu=True)
    assert torch.isnan(op(e4m3(q), dev(s), num(64), out_dtype=FLOAT)[[7, 21]]).all()


def test_linear_column_of_zeros_and_skipped_rows():
    rng = np.random.default_rng(0)
    q, s, w = linear_inputs(rng, 40, 16, 20)
    w[:, 4] = 0
    op = api.Linear8(16, 20, w, max_voxels=40)
    op.set_flags(D.SESSD_FLAG_SKIP_PAD_ROWS)
    out = torch.full((40, 20), 9.0, device=DEV)
    ins = [e4m3(q), dev(s), num(33)]
    op.configure(ins, [out])
    op.enqueue(ins, [out])
    assert (out[33:] == 9).all() and (out[:33, 4] == 0).all() and (out[:33, :4] != 9).all()


def test_rows_beyond_32_bit_offsets():
    """Tensors of more than 2^32 bytes and 2^31 elements: the last rows."""
    rows, c = 540000, 4096
    gamma = np.ones(c, np.float32)
    f = torch.zeros((rows, c), dtype=HALF, device=DEV)
    tail = np.random.default_rng(1).standard_normal((40, c)).astype(np.float16)
    f[-40:] = dev(tail)
    q, s = api.RmsNorm(c, gamma, max_voxels=rows)(f, num(rows))
    del f
    assert_norm((q[-40:], s[-40:]), tail, None, gamma, 1e-6, 40)
    assert not codes_t(q[: rows - 40]).any()
    w = (np.random.default_rng(2).standard_normal((c, 16)) / 64).astype(np.float32)
    got = api.Linear8(c, 16, w, max_voxels=rows)(q, s, num(rows), out_dtype=FLOAT)
    want, magnitude = L.linear(codes(q[-40:]), s[-40:].cpu().numpy(), w)
    assert_linear(got[-40:], want, magnitude, c)
    assert not got[:-40].any()
    del q
    rows, c = 540000, 16
    q = torch.zeros((rows, c), dtype=torch.uint8, device=DEV)
    q[-1] = 0x38
    w = np.ones((c, 4096), np.float32)
    got = api.Linear8(c, 4096, w, max_voxels=rows)(q.view(torch.float8_e4m3fn), torch.ones((rows, 1), device=DEV), num(rows))
    assert (got[-1] == 16).all() and not got[:-1].any()


def test_layers_under_a_graph_and_on_another_stream():
    rng = np.random.default_rng(5)
    feat, res, gamma = norm_inputs(rng, 500, 64, HALF, True)
    w = linear_inputs(rng, 1, 64, 192)[2]
    a, b = api.RmsNorm(64, gamma, max_voxels=500), api.Linear8(64, 192, w, max_voxels=500)
    f, r, n = dev(feat), dev(res), num(450)

    def step(q, s, total, out, stream):
        a.enqueue([f, n, r], [q, s, total], stream)
        b.enqueue([q, s, n], [out], stream)

    def buffers():
        return (torch.empty((500, 64), dtype=torch.float8_e4m3fn, device=DEV), torch.empty((500, 1), device=DEV),
                torch.empty((500, 64), dtype=HALF, device=DEV), torch.empty((500, 192), dtype=HALF, device=DEV))
    eager = buffers()
    a.configure([f, n, r], list(eager[:3]))
    b.configure([eager[0], eager[1], n], [eager[3]])
    step(*eager, None)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = buffers()
    with torch.cuda.stream(side):
        step(*other, side)
    torch.cuda.current_stream().wait_stream(side)
    replayed = buffers()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step(*replayed, torch.cuda.current_stream())
    for k in range(4):
        f.copy_(dev(feat) * (1 + k))
        graph.replay()
        step(*eager, None)
        torch.cuda.synchronize()
        for x, y in zip(eager, replayed):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
        if k == 0:
            for x, y in zip(eager, other):
                assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_wrong_tensors_are_refused():
    f = torch.randn(64, 100, device=DEV).half()
    norm = api.RmsNorm(100, np.ones(100, np.float32), max_voxels=64)
    with pytest.raises(api.SessdError, match="contiguous"):
        norm(torch.randn(100, 64, device=DEV).half().t(), num(64))
    with pytest.raises(api.SessdError, match="not in GPU memory"):
        norm(f, num(64).cpu())
    with pytest.raises(api.SessdError, match="feat must be"):
        norm(f[:, :96].contiguous(), num(64))
    with pytest.raises(api.SessdError, match="feat must be"):
        norm(f[:63], num(63))
    with pytest.raises(api.SessdError, match="type"):
        norm(f, num(64), f.float())
    with pytest.raises(api.SessdError, match="aligned"):
        norm(torch.randn(6401, device=DEV).half()[1:].reshape(64, 100), num(64))
    lin = api.Linear8(32, 16, np.ones((32, 16), np.float32), max_voxels=64)
    q, s = torch.zeros(64, 32, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn), torch.ones(64, 1, device=DEV)
    for bad in ((q[:, :16].contiguous(), s, num(1)), (q, s.expand(64, 2), num(1)), (q, s, num(1).float()), (f, s, num(1)), (q, s.half(), num(1))):
        with pytest.raises(api.SessdError):
            lin(*bad)
    with pytest.raises(api.SessdError, match="FP32 or FP16"):
        lin(q, s, num(1), out_dtype=torch.float8_e4m3fn)
    assert torch.equal(lin(q, s, num(64)), torch.zeros(64, 16, dtype=HALF, device=DEV))
