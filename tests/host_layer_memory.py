"""What RmsNorm, Linear8 and VoxelAttention keep in device memory, on the stand-in runtime of fake_hip_memory.cpp, without torch and without a GPU: run
as a program of its own (tests/test_layer_memory_cpu.py), because one process holds one HIP runtime.

    python tests/host_layer_memory.py <path of the stand-in library> <check>
"""
import ctypes as C
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [os.path.join(ROOT, "se-ssd-ai-trt_amd"), os.path.join(ROOT, "tests")]
sys.modules["torch"] = None  # (sessd3d.api binds the library to torch's runtime where it finds torch)

import numpy as np  # noqa: E402
from sessd3d import api, ctypes_defs as D  # noqa: E402

FAKE = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
FAKE.fake_log.restype = C.c_char_p
FAKE.fake_largest_allocation.argtypes = [C.c_ulonglong]
FAKE.fake_fail_copy.argtypes = [C.c_long]
L = api.lib()
I32, F32, F16, FP8 = D.SESSD_INT32, D.SESSD_FLOAT, D.SESSD_HALF, D.SESSD_FP8


def log():
    lines = [l.split() for l in FAKE.fake_log().decode().splitlines()]
    FAKE.fake_clear_log()
    return lines


def of_kind(lines, kind):
    return [(int(a), int(b)) for k, a, b in lines if k == kind]


def descs(*shapes):
    return (D.TensorDesc * len(shapes))(*[D.TensorDesc.make(list(s), t) for s, t in shapes])


def pointers(*values):
    return (C.c_void_p * len(values))(*values)


class Linear:
    def __init__(self, cin, cout, w, rows=100):
        log()
        self.h = C.c_void_p()
        w = np.ascontiguousarray(w, np.float32)
        assert L.sessd_linear8_create(C.byref(D.Linear8Desc(cin, cout, rows)), w.ctypes.data, C.byref(self.h)) == 0
        self.memory = of_kind(log(), "malloc")
        self.ins = descs(((1, rows, cin), FP8), ((1, rows, 1), F32), ((1,), I32))
        self.cout, self.rows = cout, rows

    def call(self, dtype=F16):
        outs = descs(((1, self.rows, self.cout), dtype))
        assert L.sessd_linear8_configure(self.h, self.ins, 3, outs, 1) == 0
        return L.sessd_linear8_enqueue(self.h, self.ins, outs, pointers(4096, 8192, 64), pointers(16384), None, None)

    def set_epilogue(self, scale, shift, relu):
        p = lambda a: None if a is None else np.ascontiguousarray(a, np.float32).ctypes.data_as(C.c_void_p)  # noqa: E731
        return L.sessd_linear8_set_epilogue(self.h, p(scale), p(shift), relu)

    def blob(self):
        buf = C.create_string_buffer(L.sessd_linear8_serialization_size(self.h))
        assert L.sessd_linear8_serialize(self.h, buf) == 0
        return buf.raw

    def device_memory(self):
        return [C.string_at(p, n) for p, n in self.memory]


def check_epilogue():
    """A new epilogue waits for the calls that read the old one, and one that cannot be had changes nothing."""
    rng = np.random.default_rng(0)
    lin = Linear(32, 20, rng.standard_normal((32, 20)))
    sc, sh = rng.standard_normal((2, 20)).astype(np.float32)
    assert lin.set_epilogue(sc, sh, 1) == 0
    assert lin.call() == 0
    log()
    assert lin.set_epilogue(-sc, None, 0) == 0
    assert not of_kind(log(), "unordered")
    assert lin.call() == 0 and lin.set_epilogue(None, sh, 1) == 0 and not of_kind(log(), "unordered")
    # what fails leaves the plugin and the GPU as they were
    blob, memory = lin.blob(), lin.device_memory()
    FAKE.fake_fail_copy(0)
    assert lin.set_epilogue(sc, sh, 0) == D.SESSD_E_HIP
    FAKE.fake_fail_copy(-1)
    assert lin.blob() == blob and lin.device_memory() == memory
    FAKE.fake_largest_allocation(16)
    assert lin.set_epilogue(sc, sh, 0) == D.SESSD_E_HIP
    FAKE.fake_largest_allocation(1 << 62)
    assert lin.blob() == blob and lin.device_memory() == memory
    L.sessd_linear8_destroy(lin.h)


def check_device():
    """A layer that was made on one device refuses calls while another is current."""
    rows = 100
    feat = [((1, rows, 48), F16), ((1,), I32)]
    h = C.c_void_p()
    g = np.ones(48, np.float32)
    assert L.sessd_rmsnorm_create(C.byref(D.RmsNormDesc(48, rows, 1e-6)), g.ctypes.data, C.byref(h)) == 0
    i, o = descs(*feat), descs(((1, rows, 48), FP8), ((1, rows, 1), F32))
    assert L.sessd_rmsnorm_configure(h, i, 2, o, 2) == 0
    a = C.c_void_p()
    d = D.VoxelAttnDesc(2, 2, 8, rows, (C.c_int32 * 3)(20, 20, 4), (C.c_int32 * 3)(5, 5, 4), (C.c_int32 * 3)(), (C.c_float * 3)(1, 1, 1), 0, 0)
    assert L.sessd_voxelattn_create(C.byref(d), None, C.byref(a)) == 0
    ai, ao = descs(((1, rows, 48), F16), ((1, rows, 4), I32), ((1,), I32)), descs(((1, rows, 16), F16))
    assert L.sessd_voxelattn_configure(a, ai, 3, ao, 1) == 0
    FAKE.fake_set_device(2)
    lin = Linear(32, 20, np.ones((32, 20)))
    calls = [lambda: L.sessd_rmsnorm_enqueue(h, i, o, pointers(4096, 64), pointers(8192, 16384), None, None),
             lambda: L.sessd_voxelattn_enqueue(a, ai, ao, pointers(4096, 8192, 64), pointers(16384), 65536, None),
             lambda: L.sessd_voxelattn_enqueue_shared(a, ai, ao, pointers(4096, 8192, 64), pointers(16384), 65536, None)]
    own = [lin.call, lambda: lin.set_epilogue(None, np.ones(20), 1)]
    for device in (2, 0, 1, 0, 2):
        FAKE.fake_set_device(device)
        for call, made in [(c, 0) for c in calls] + [(c, 2) for c in own]:
            log()
            rc, text = call(), L.sessd_last_error().decode()
            if made == device:
                assert rc == 0
            else:
                assert rc == D.SESSD_E_INVALID and "device %d" % made in text and "one is %d" % device in text, text
                assert not log()
    FAKE.fake_set_device(0)


def check_weights():
    """The weights that the GPU has are the e4m3 nearest to W / wscale, widened to halves, each where the instructions want it: of 16 columns times 32
    channels, lane l has column l % 16 and the eight channels of its quarter; columns are dealt so that a lane's results are neighbours."""
    import layer_oracle as O
    rng = np.random.default_rng(0)
    for cin, cout in ((16, 5), (48, 70), (256, 64), (272, 33), (512, 40), (1040, 100)):
        w = (rng.standard_normal((cin, cout)) * 10.0 ** rng.uniform(-20, 20, cout)).astype(np.float32)
        w[:, 3] = 0
        w[0, 1:3] = 448 * np.abs(w[:, 1:3]).max()     # (a scale of which ties and the values below 2^-6 are reached)
        w[1:16, 1] = w[0, 1] / 448 * np.arange(1, 16) * 2.0 ** -10
        w[1:16, 2] = w[0, 2] / 448 * (16.5 + np.arange(15))
        wscale = np.maximum(np.abs(w).max(0) / np.float32(448), np.float32(2.0 ** -100)).astype(np.float32)
        codes = O.to_e4m3(w / wscale)
        lin = Linear(cin, cout, w)
        (p, size), (cp, csize) = lin.memory
        tiles = 2 if 256 < cin <= 512 else 4
        blocks, steps = -(-cout // (16 * tiles)), 2 * -(-cin // 64)
        halves = np.frombuffer(C.string_at(p, size), np.float16).reshape(2, blocks, steps, tiles, 64, 8)  # FP32 outputs, FP16 ones
        seen = np.zeros((2, cin, cout), int)
        for half in (0, 1):
            for b in range(blocks):
                for s in range(steps):
                    for t in range(tiles):
                        for lane in range(64):
                            r, g = lane % 16, lane // 16
                            # of instruction t, results 4 (r / 4) .. + 3 go to one lane: FP16 stores 8 of a pair of instructions, FP32 4 of one
                            col = b * 16 * tiles + ((t // 2) * 32 + (r // 4) * 8 + (t % 2) * 4 + r % 4 if half else t * 16 + r)
                            for e in range(8):
                                ch = (s // 2) * 64 + g * 16 + (s % 2) * 8 + e   # (a lane reads 16 neighbouring bytes of a row for two steps)
                                got = float(halves[half, b, s, t, lane, e])
                                if col < cout and ch < cin:
                                    assert got == O.VALUES[codes[ch, col]], (cin, cout, half, ch, col, got)
                                    seen[half, ch, col] += 1
                                else:
                                    assert got == 0
        assert (seen == 1).all()
        pad = blocks * 16 * tiles
        sc, sh = rng.standard_normal((2, cout)).astype(np.float32)
        for scale, shift, relu in ((None, None, None), (sc, sh, 1), (None, sh, 0), (sc, None, 1)):
            if relu is not None:
                assert lin.set_epilogue(scale, shift, relu) == 0
            columns = np.frombuffer(C.string_at(cp, csize), np.float32)
            assert np.array_equal(columns[:cout], wscale if scale is None else wscale * scale) and not columns[cout:pad].any()
            assert np.array_equal(columns[pad:pad + cout], np.zeros(cout) if shift is None else shift) and not columns[pad + cout:2 * pad].any()
            assert columns[2 * pad] == (relu or 0)
        L.sessd_linear8_destroy(lin.h)


def check_fields():
    """Fields that hold fewer values than the layer has are refused, those with a single one as well."""
    i = lambda *v: np.array(v, np.int32)  # noqa: E731
    f = lambda *v: np.array(v, np.float32)  # noqa: E731
    three = dict(spatial_shape=i(20, 20, 4), window_shape=i(5, 5, 4), window_shift=i(0, 0, 0), cell_size=f(1, 1, 1))
    plugins = {"RmsNormPlugin": dict(channel=i(48), max_voxels=i(100), eps=f(1e-6), gamma=f(*[1] * 48)),
               "Linear8Plugin": dict(in_channel=i(32), out_channel=i(20), max_voxels=i(100), weights=f(*[1] * 640)),
               "VoxelAttentionPlugin": dict(num_heads=i(4), num_kv_heads=i(2), head_dim=i(16), max_voxels=i(100), softmax_scale=f(0), score_cap=f(0),
                                            slopes=f(1, 2, 3, 4), **three)}
    for name, fields in plugins.items():
        assert api.create_plugin(name, fields).max_voxels == 100
        for key, v in fields.items():
            for bad in (v[:1], v[:-1], v[:0], np.concatenate([v, v])):
                if bad.size == v.size:
                    continue
                try:
                    api.create_plugin(name, dict(fields, **{key: bad}))
                    raise AssertionError((name, key))
                except api.SessdError as e:
                    assert key in str(e), e


CHECKS = {k[6:]: v for k, v in list(globals().items()) if k.startswith("check_")}

if __name__ == "__main__":
    CHECKS[sys.argv[2]]()
    print("ok")
