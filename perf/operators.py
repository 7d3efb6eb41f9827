"""The operators of a transformer layer over voxel features, and the sizes by which their speed is judged.

A network that puts attention behind the sparse convolutions runs, for each of its layers, a norm that takes the residual in
and leaves its rows in 8 bits, projections that read such rows, and attention among the voxels of a window.  Their tensors are
those of the sparse layers: features [max_voxels, C] of which voxel_num rows count, coordinates (b, z, y, x).

    norm      h = x + r,  y = gamma * h / sqrt(mean(h^2) + eps),  s = max|y| / 448,  q = e4m3(y / s);  q, s and h are returned
    linear    y = (q W_q) * s * s_w, then * scale + shift and ReLU where the layer has them; W in e4m3 with a scale s_w a column
    attn      softmax over the rows of a voxel's own window of  c * tanh(q.k * d^-0.5 / c) - m_head * |p_i - p_j|,  times v

Inference is the only direction the library has.
"""
import functools
import math
import os
import sys

import numpy as np
import torch

own = False
DEV = "cuda:0" if torch.cuda.is_available() else "cpu"
EPS = 1e-6
E4M3_MOST = 448.0
SMALLEST_SCALE = 2.0 ** -100  # of a row of zeros


def listed():
    return [
        # --- norm: the rows of a small crop (latency), of a camera-FOV frame at its capacity, of two merged full-circle scans
        dict(name="norm_2k_64_fp16", kind="norm", sites=2000, rows=2000, channels=64, dtype="fp16", residual=True),
        dict(name="norm_17k_128_fp16", kind="norm", sites=16825, rows=20000, channels=128, dtype="fp16", residual=True),
        dict(name="norm_160k_256_fp32", kind="norm", sites=157301, rows=160000, channels=256, dtype="fp32", residual=True),
        # --- linear: query, key and value of a small crop and of a frame, the two sides of a feed-forward part
        dict(name="linear_2k_64x192_fp16", kind="linear", sites=2000, rows=2000, cin=64, cout=192, dtype="fp16", epilogue="none"),
        dict(name="linear_17k_128x384_fp16", kind="linear", sites=16825, rows=20000, cin=128, cout=384, dtype="fp16", epilogue="shift"),
        dict(name="linear_60k_512x128_fp32", kind="linear", sites=59999, rows=60000, cin=512, cout=128, dtype="fp32", epilogue="shift"),
        dict(name="linear_150k_256x1024_fp16", kind="linear", sites=150000, rows=160000, cin=256, cout=1024, dtype="fp16",
             epilogue="relu"),
        # --- attn: a small crop; the third stage of a frame in both types; the second stage of a full one with shifted windows and
        # keys shared by four heads; every voxel of a coarse frame against every other
        dict(name="attn_2k_fp16", kind="attn", points=2000, stage=3, rows=2000, heads=4, kv_heads=4, dim=16, window=12, height=0,
             shift=0, dtype="fp16", slope=1.0, cap=0.0),
        dict(name="attn_20k_fp16", kind="attn", points=20000, stage=3, rows=20000, heads=8, kv_heads=8, dim=16, window=12, height=0,
             shift=0, dtype="fp16", slope=0.5, cap=30.0),
        dict(name="attn_20k_fp32", kind="attn", points=20000, stage=3, rows=20000, heads=8, kv_heads=8, dim=24, window=16, height=4,
             shift=8, dtype="fp32", slope=0.5, cap=0.0),
        dict(name="attn_60k_fp16", kind="attn", points=60000, stage=2, rows=60000, heads=8, kv_heads=2, dim=32, window=16, height=0,
             shift=8, dtype="fp16", slope=0.25, cap=0.0),
        dict(name="attn_whole_fp16", kind="attn", points=60000, stage=3, rows=30000, heads=8, kv_heads=4, dim=64, window=0, height=0,
             shift=0, dtype="fp16", slope=0.05, cap=50.0),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "linear", "attn", "attn"])
    dtype = rng.choice(["fp16", "fp32"])
    if kind == "norm":
        channels = rng.choice([16, 32, 64, 96, 128, 192, 256, rng.randint(5, 256)])
        sites = _spread(rng, 1, 150000)
        return dict(kind=kind, sites=sites, rows=sites + rng.choice([0, 1, sites // 4]), channels=channels, dtype=dtype,
                    residual=rng.random() < 0.7)
    if kind == "linear":
        sites = _spread(rng, 1, 100000)
        return dict(kind=kind, sites=sites, rows=sites + rng.choice([0, 1, sites // 4]), cin=16 * _spread(rng, 1, 32),
                    cout=rng.choice([64, 128, 192, 384, 512, rng.randint(9, 512)]), dtype=dtype,
                    epilogue=rng.choice(["none", "shift", "relu"]))
    kv_heads = rng.choice([1, 2, 4, 8])
    whole = rng.random() < 0.2
    points = _spread(rng, 20, 12000 if whole else 60000)
    return dict(kind=kind, points=points, stage=rng.choice([2, 3, 4]), rows=points + rng.choice([0, 1, 300]),
                heads=kv_heads * rng.choice([1, 2, 4] if kv_heads < 8 else [1]), kv_heads=kv_heads, dim=8 * rng.randint(1, 8),
                window=0 if whole else rng.randint(4, 20), height=0 if whole else rng.choice([0, 2, 5]), shift=0 if whole else rng.randint(0, 3),
                dtype=dtype, slope=rng.choice([0.0, 0.25, 1.0]), cap=rng.choice([0.0, 20.0, 50.0]))


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------

GRIDS = {2: (21, 800, 704), 3: (11, 400, 352), 4: (5, 200, 176)}  # z, y, x
EXTENT = (4.0, 80.0, 70.4)                                         # metres


def _cells(points, stage, seed):
    """Distinct cells (z, y, x) that a scan of so many points meets, in the order in which it meets them."""
    rng = np.random.default_rng([int(seed), 5])
    r = 2.0 + rng.exponential(15.0, points)
    az = rng.uniform(-0.25 * np.pi, 0.25 * np.pi, points)
    ground = rng.random(points) < 0.35
    z = np.where(ground, 1.3 + 0.05 * rng.standard_normal(points), rng.uniform(1.2, 3.9, points))
    p = np.stack([z, 40.0 + r * np.sin(az), r * np.cos(az)], 1)
    grid = np.array(GRIDS[stage])
    c = np.floor(p * grid / EXTENT).astype(np.int64)
    c = c[((c >= 0) & (c < grid)).all(1)]
    key = (c[:, 0] * grid[1] + c[:, 1]) * grid[2] + c[:, 2]
    return c[np.sort(np.unique(key, return_index=True)[1])]


def _window(case):
    """(z, y, x): cells of a window and how far the windows are shifted; 0 cells stand for the whole axis."""
    grid = GRIDS[case["stage"]]
    w = (case["height"] or grid[0], case["window"] or grid[1], case["window"] or grid[2])
    return w, tuple(min(case["shift"], v - 1) if case["window"] else 0 for v in (1, w[1], w[2]))


def _type(case):
    return torch.float16 if case["dtype"] == "fp16" else torch.float32


def _normal(shape, seed, stream, spread=1.0):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed) * 16 + stream)
    return torch.randn(shape, generator=gen, device=DEV) * spread


def _to_e4m3(y, dim):
    """y over its largest magnitude along `dim` in e4m3, and the scales."""
    s = (y.abs().amax(dim, keepdim=True) / E4M3_MOST).clamp_min(SMALLEST_SCALE)
    return (y / s).to(torch.float8_e4m3fn), s


@functools.lru_cache(4)
def _linear_weights(cin, cout, epilogue, seed):
    """W as a model file has it, its e4m3 form with a scale for each column, scale and shift of the epilogue."""
    rng = np.random.default_rng([int(seed), 9])
    w = (rng.standard_normal((cin, cout)) / math.sqrt(cin)).astype(np.float32)
    q, s = _to_e4m3(torch.from_numpy(w), 0)
    scale = rng.uniform(0.5, 1.5, cout).astype(np.float32) if epilogue == "relu" else None
    shift = rng.uniform(-0.3, 0.3, cout).astype(np.float32) if epilogue != "none" else None
    return w, q, s, scale, shift


def _inputs(case, seed):
    s = dict(case, seed=seed)
    if case["kind"] == "attn":
        cells = _cells(case["points"], case["stage"], seed)[:case["rows"]]
        n, grid = len(cells), GRIDS[case["stage"]]
        coors = np.zeros((case["rows"], 4), np.int32)
        coors[:n, 1:] = cells
        s["coors"] = torch.from_numpy(coors).to(DEV)
        s["feat"] = _normal((case["rows"], (case["heads"] + 2 * case["kv_heads"]) * case["dim"]), seed, 0).to(_type(case))
        s["cell"] = tuple(float(np.float32(EXTENT[a] / grid[a])) for a in range(3))  # z, y, x
        # heads look from near to far: each at three quarters of the slope of the one before
        s["slopes"] = (case["slope"] * 0.75 ** np.arange(case["heads"])).astype(np.float32)
    else:
        n = case["sites"]
        if case["kind"] == "norm":
            c = case["channels"]
            s["feat"] = _normal((case["rows"], c), seed, 0).to(_type(case))
            s["added"] = (_normal((case["rows"], c), seed, 1, 2.0) * (1.0 + 4.0 * (torch.arange(c, device=DEV) % 61 == 3))).to(_type(case))
            s["gamma"] = np.random.default_rng([int(seed), 9]).uniform(0.5, 1.5, c).astype(np.float32)
        else:
            s["q"], s["scale"] = _to_e4m3(_normal((case["rows"], case["cin"]), seed, 0), 1)
    s["n"] = n
    s["num"] = torch.tensor([n], dtype=torch.int32, device=DEV)
    return s


# ---------------------------------------------------------------------------------------------------------------
# preparing and running
# ---------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    s = _inputs(case, int(seed))
    if case["kind"] == "norm":
        s["gamma_dev"] = torch.from_numpy(s["gamma"]).to(DEV)
    elif case["kind"] == "linear":
        s["w"], wq, ws, s["bn_scale"], s["bn_shift"] = _linear_weights(case["cin"], case["cout"], case["epilogue"], int(seed))
        s["wq"], s["ws"] = wq.to(DEV), ws.to(DEV)
        s["scale_dev"], s["shift_dev"] = (None if v is None else torch.from_numpy(v).to(DEV) for v in (s["bn_scale"], s["bn_shift"]))
    else:
        s["slopes_dev"], s["cell_dev"] = torch.from_numpy(s["slopes"]).to(DEV), torch.tensor(s["cell"], device=DEV)
        s["window_dev"], s["shift_dev"] = (torch.tensor(v, device=DEV) for v in _window(case))
    if own:
        s["op"] = _plugin(case, s)
    return s


def _plugin(case, s):
    if os.path.join(os.getcwd(), "se-ssd-ai-trt_amd") not in sys.path:
        sys.path.insert(0, os.path.join(os.getcwd(), "se-ssd-ai-trt_amd"))
    from sessd3d import api
    if case["kind"] == "norm":
        return api.RmsNorm(case["channels"], s["gamma"], max_voxels=case["rows"], eps=EPS)
    if case["kind"] == "linear":
        op = api.Linear8(case["cin"], case["cout"], s["w"], max_voxels=case["rows"])
        if case["epilogue"] != "none":
            op.set_epilogue(s["bn_scale"], s["bn_shift"], relu=case["epilogue"] == "relu")
        return op
    window, shift = _window(case)
    return api.VoxelAttention(case["heads"], case["kv_heads"], case["dim"], GRIDS[case["stage"]][::-1], window[::-1],
                              shift_xyz=shift[::-1], slopes=s["slopes"] if case["slope"] else None, cell_size_xyz=s["cell"][::-1],
                              cap=case["cap"], max_voxels=case["rows"])


def run(s):
    if own:
        if s["kind"] == "norm":
            return s["op"](s["feat"], s["num"], s["added"] if s["residual"] else None)
        if s["kind"] == "linear":
            return s["op"](s["q"], s["scale"], s["num"], out_dtype=_type(s))
        return s["op"](s["feat"], s["coors"], s["num"])
    return {"norm": _norm, "linear": _linear, "attn": _attention}[s["kind"]](s)


def _norm(s):
    n = s["n"]
    h = s["feat"].float()
    if s["residual"]:
        h = h + s["added"].float()
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * s["gamma_dev"]
    scale = (y.abs().amax(1, keepdim=True) / E4M3_MOST).clamp_min(SMALLEST_SCALE)
    q = y / scale
    q[n:], scale[n:] = 0.0, 0.0
    if not s["residual"]:
        return q.to(torch.float8_e4m3fn), scale
    h[n:] = 0.0
    return q.to(torch.float8_e4m3fn), scale, h.to(s["feat"].dtype)


def _linear(s):
    y = (s["q"].float() @ s["wq"].float()) * s["scale"] * s["ws"]
    y[s["n"]:] = 0.0
    if s["scale_dev"] is not None:
        y = y * s["scale_dev"]
    if s["shift_dev"] is not None:
        y = y + s["shift_dev"]
    if s["epilogue"] == "relu":
        y = y.clamp_min(0.0)
    return y.to(_type(s))


def _attention(s):
    n, heads, kv, d = s["n"], s["heads"], s["kv_heads"], s["dim"]
    x, cells = s["feat"][:n].float(), s["coors"][:n, 1:].long()
    w = (cells + s["shift_dev"]) // s["window_dev"]
    order = torch.argsort((w[:, 0] * 4096 + w[:, 1]) * 4096 + w[:, 2], stable=True)
    w = w[order]
    new = torch.ones(n, dtype=torch.bool, device=x.device)
    new[1:] = (w[1:] != w[:-1]).any(1)
    group = new.long().cumsum(0) - 1                       # of each row in that order: its window, and its place there
    starts = new.nonzero()[:, 0]
    counts = torch.diff(starts, append=starts.new_full((1,), n))
    place = torch.arange(n, device=x.device) - starts[group]
    # blocks of up to 64 rows of one window, each beside all rows of that window, up to the longest window's length
    block = (place % 64 == 0).long().cumsum(0) - 1
    first = (place % 64 == 0).nonzero()[:, 0]
    longest = int(counts.max())
    tall = min(longest, 64)
    mine = order[(first[:, None] + torch.arange(tall, device=x.device)).clamp_max(n - 1)]
    keys = starts[group[first]][:, None] + torch.arange(longest, device=x.device)
    there = keys < (starts + counts)[group[first]][:, None]
    keys = order[keys.clamp_max(n - 1)]
    q, k, v = (t.reshape(n, -1, d) for t in x.split((heads * d, kv * d, kv * d), 1))
    q = q[mine].transpose(1, 2).reshape(len(first), kv, heads // kv * tall, d)  # block, head, row, d
    score = (q @ k[keys].permute(0, 2, 3, 1).contiguous()).mul_(d ** -0.5).reshape(len(first), heads, tall, longest)
    if s["cap"]:
        score = score.div_(s["cap"]).tanh_().mul_(s["cap"])
    if s["slope"]:
        at = cells.float()
        far = (((at[mine][:, :, None] - at[keys][:, None]) * s["cell_dev"]) ** 2).sum(3).sqrt()
        score.addcmul_(far[:, None], s["slopes_dev"][:, None, None], value=-1.0)
    score.masked_fill_(~there[:, None, None], -math.inf)
    p = score.sub_(score.amax(3, keepdim=True)).exp_()
    total = p.sum(3, keepdim=True)
    o = p.reshape(len(first), kv, heads // kv * tall, longest) @ v[keys].transpose(1, 2).contiguous()
    o = (o.reshape(len(first), heads, tall, d) / total).transpose(1, 2).reshape(len(first), tall, heads * d)
    out = torch.zeros((s["rows"], heads * d), dtype=_type(s), device=x.device)
    out[order] = o[block, torch.arange(n, device=x.device) - first[block]].to(out.dtype)
    return out


# ---------------------------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, int(seed))
    n = s["n"]
    if case["kind"] == "norm":
        h = s["feat"][:n].double()
        if case["residual"]:
            h += s["added"][:n].double()
        mean = torch.einsum("rc,rc->r", h, h)[:, None] / case["channels"]
        y = h / torch.sqrt(mean + EPS) * torch.from_numpy(s["gamma"]).to(DEV).double()
        scale = torch.maximum(y.max(1).values, -y.min(1).values)[:, None] / E4M3_MOST
        scale = torch.where(scale > SMALLEST_SCALE, scale, torch.full_like(scale, SMALLEST_SCALE))
        got = [(y / scale).to(torch.float8_e4m3fn).double(), scale] + ([h] if case["residual"] else [])
        return tuple(torch.cat([t, t.new_zeros((case["rows"] - n, t.shape[1]))]) for t in got)
    if case["kind"] == "linear":
        _, wq, ws, scale, shift = _linear_weights(case["cin"], case["cout"], case["epilogue"], int(seed))
        y = torch.zeros((case["rows"], case["cout"]), dtype=torch.float64, device=DEV)
        y[:n] = (s["q"][:n].double() * s["scale"][:n].double()) @ (wq.double() * ws.double()).to(DEV)
        if scale is not None:
            y *= torch.from_numpy(scale).to(DEV)
        if shift is not None:
            y += torch.from_numpy(shift).to(DEV)
        return torch.relu(y) if case["epilogue"] == "relu" else y
    heads, kv, d = case["heads"], case["kv_heads"], case["dim"]
    cells = s["coors"][:n, 1:].cpu().numpy().astype(np.int64)
    window, shift = _window(case)
    _, which = np.unique((cells + shift) // window, axis=0, return_inverse=True)
    which = which.reshape(-1)
    by = np.split(np.argsort(which, kind="stable"), np.cumsum(np.bincount(which))[:-1])
    if sum(float(len(b)) ** 2 for b in by) * heads * d > 1e12:
        return None
    feat = s["feat"][:n].double()
    place = torch.from_numpy(cells * np.array(s["cell"])).to(DEV)
    slopes = torch.from_numpy(s["slopes"].astype(np.float64)).to(DEV)
    out = torch.zeros((case["rows"], heads, d), dtype=torch.float64, device=DEV)
    for b in by:
        b = torch.from_numpy(b).to(DEV)
        x = feat[b]
        far = torch.linalg.vector_norm(place[b][:, None] - place[b][None], dim=2)
        for h in range(heads):
            g = h // (heads // kv)
            k = x[:, (heads + g) * d:(heads + g + 1) * d]
            v = x[:, (heads + kv + g) * d:(heads + kv + g + 1) * d]
            t = x[:, h * d:(h + 1) * d] @ k.T / math.sqrt(d)
            if case["cap"]:
                t = case["cap"] * torch.tanh(t / case["cap"])
            out[b, h] = torch.softmax(t - slopes[h] * far, 1) @ v
    return out.reshape(case["rows"], heads * d)


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------

@functools.lru_cache(None)
def _pairs(points, stage, rows, window, shift):
    """Of the scan with seed 0: its cells and the pairs of cells that share a window."""
    cells = _cells(points, stage, 0)[:rows]
    counts = np.unique((cells + shift) // window, axis=0, return_counts=True)[1].astype(np.float64)
    return len(cells), float((counts ** 2).sum())


def work(case):
    es = 2.0 if case["dtype"] == "fp16" else 4.0
    if case["kind"] == "norm":
        c, n, rows = case["channels"], case["sites"], case["rows"]
        wide = 1 if case["residual"] else 0
        return {"bytes": n * c * es * (1 + wide) + rows * (c * es * wide + c + 4.0) + 4.0 * c, "flops": 8.0 * n * c}
    if case["kind"] == "linear":
        n, rows, cin, cout = case["sites"], case["rows"], case["cin"], case["cout"]
        return {"bytes": n * (cin + 4.0) + cin * cout + rows * cout * es, "flops": 2.0 * n * cin * cout}
    n, pairs = _pairs(case["points"], case["stage"], case["rows"], *_window(case))
    heads, kv, d = case["heads"], case["kv_heads"], case["dim"]
    return {"bytes": n * ((heads + 2 * kv) * d * es + 16.0) + case["rows"] * heads * d * es, "flops": 4.0 * pairs * heads * d}
