"""RmsNorm, Linear8 and VoxelAttention on the stand-in runtime of fake_hip.cpp, without torch and without a GPU: run as a program of its
own (tests/test_layers_cpu.py), because one process holds one HIP runtime.

    python tests/host_layers.py <path of the stand-in library> <check>
"""
import ctypes as C
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "se-ssd-ai-trt_amd"))
sys.modules["torch"] = None  # (sessd3d.api binds the library to torch's runtime where it finds torch)

import numpy as np  # noqa: E402
from sessd3d import api, ctypes_defs as D  # noqa: E402

FAKE = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
FAKE.fake_log.restype = C.c_char_p
FAKE.fake_largest_allocation.argtypes = [C.c_ulonglong]
FAKE.fake_fail_new.argtypes = [C.c_long]
L = api.lib()
GRID, WINDOW = (70, 80, 10), (8, 8, 10)
I32, F32, F16, FP8 = D.SESSD_INT32, D.SESSD_FLOAT, D.SESSD_HALF, D.SESSD_FP8


def launches():
    lines = [l.split() for l in FAKE.fake_log().decode().splitlines()]
    FAKE.fake_clear_log()
    return [l for l in lines if l[0] == "launch"]


def descs(*shapes):
    return (D.TensorDesc * len(shapes))(*[D.TensorDesc.make(list(s), t) for s, t in shapes])


def pointers(*values):
    return (C.c_void_p * len(values))(*values)


def refused(rc, code, *words):
    text = L.sessd_last_error().decode()
    assert rc == code and all(w in text for w in words), (rc, text)
    assert not launches()


def norm(channel=48, rows=100, eps=1e-6, gamma=None):
    h = C.c_void_p()
    g = np.ones(max(channel, 1), np.float32) if gamma is None else np.asarray(gamma, np.float32)
    return L.sessd_rmsnorm_create(C.byref(D.RmsNormDesc(channel, rows, eps)), g.ctypes.data, C.byref(h)), h


def linear(cin=32, cout=20, rows=100, w=None):
    h = C.c_void_p()
    w = np.ones((abs(cin) + 1) * (abs(cout) + 1), np.float32) if w is None else np.ascontiguousarray(w, np.float32)
    return L.sessd_linear8_create(C.byref(D.Linear8Desc(cin, cout, rows)), w.ctypes.data, C.byref(h)), h


def attention(heads=4, kv=2, dim=16, rows=100, grid=GRID, window=WINDOW, shift=(0, 0, 0), cell=(1, 1, 1), scale=0.0, cap=0.0, slopes=None):
    d = D.VoxelAttnDesc(heads, kv, dim, rows, (C.c_int32 * 3)(*grid), (C.c_int32 * 3)(*window), (C.c_int32 * 3)(*shift), (C.c_float * 3)(*cell),
                        scale, cap)
    h = C.c_void_p()
    s = None if slopes is None else np.asarray(slopes, np.float32)
    return L.sessd_voxelattn_create(C.byref(d), None if s is None else s.ctypes.data, C.byref(h)), h


def check_create():
    E, U = D.SESSD_E_INVALID, D.SESSD_E_UNSUPPORTED
    for kw, code in ((dict(channel=0), E), (dict(channel=-4), E), (dict(rows=0), E), (dict(channel=4097), U), (dict(rows=(1 << 24) + 1), U), (dict(eps=-1.0), E),
                     (dict(eps=float("nan")), E), (dict(eps=float("inf")), E), (dict(gamma=[1.0] * 47 + [float("nan")]), E)):
        refused(norm(**kw)[0], code, "rmsnorm")
    bad = np.ones((32, 20))
    bad[3, 4] = np.inf
    for kw, code in ((dict(cin=0), E), (dict(cin=-16), E), (dict(cout=0), E), (dict(rows=-1), E), (dict(cin=24), U), (dict(cin=4112), U),
                     (dict(cout=4097), U), (dict(rows=(1 << 24) + 1), U), (dict(w=bad), E)):
        refused(linear(**kw)[0], code, "linear8")
    for kw, code in ((dict(heads=0), E), (dict(kv=0), E), (dict(heads=4, kv=3), E), (dict(dim=0), E), (dict(dim=12), U), (dict(dim=136), U), (dict(rows=(1 << 24) + 1), U),
                     (dict(rows=0), E), (dict(heads=2048, kv=2048), U), (dict(window=(0, 8, 8)), E), (dict(shift=(8, 0, 0)), E),
                     (dict(shift=(0, -1, 0)), E), (dict(grid=(70, 0, 10)), E), (dict(grid=(1 << 25, 1, 1), window=(1 << 20, 1, 1)), U),
                     (dict(grid=(4096, 1024, 2), window=(1, 1, 1)), U), (dict(grid=(1 << 24, 1 << 24, 1 << 24), window=(1, 1, 1)), U),
                     (dict(cell=(1, float("nan"), 1)), E), (dict(cap=-1.0), E), (dict(cap=float("inf")), E), (dict(scale=float("nan")), E),
                     (dict(slopes=[0, 1, float("inf"), 2]), E), (dict(scale=1e-13), U), (dict(scale=-2e12), U), (dict(cap=1e-20), U), (dict(cap=1e20), U),
                     (dict(cell=(1, -3e6, 1)), U), (dict(slopes=[0, 1, 2, -2e6]), U)):
        refused(attention(**kw)[0], code, "voxelattn")
    assert attention(grid=(4096, 1024, 1), window=(1, 1, 1))[0] == 0       # 2^22 windows
    assert L.sessd_rmsnorm_create(None, None, None) == E and L.sessd_linear8_create(None, None, None) == E
    assert L.sessd_voxelattn_create(None, None, None) == E
    # device memory that runs out
    FAKE.fake_largest_allocation(16)
    for made in (norm(), linear(), attention(slopes=[1] * 4 + [0] * 4, heads=8)):
        assert made[0] == D.SESSD_E_HIP and not made[1].value
    FAKE.fake_largest_allocation(1 << 62)
    for make in (norm, linear, lambda: attention(slopes=[1, 2, 3, 4])):
        for k in range(6):
            FAKE.fake_fail_new(k)
            rc, h = make()
            FAKE.fake_fail_new(-1)
            assert rc in (0, D.SESSD_E_NOMEM) and bool(h.value) == (rc == 0), (k, rc)


NORM_IN = lambda c=48, n=100, t=F16: [((1, n, c), t), ((1,), I32), ((1, n, c), t)]  # noqa: E731
NORM_OUT = lambda c=48, n=100, t=F16: [((1, n, c), FP8), ((1, n, 1), F32), ((1, n, c), t)]  # noqa: E731


def change(tensors, i, shape=None, dtype=None):
    tensors = list(tensors)
    tensors[i] = (shape or tensors[i][0], tensors[i][1] if dtype is None else dtype)
    return tensors


def check_norm():
    E, U = D.SESSD_E_INVALID, D.SESSD_E_UNSUPPORTED
    h = norm()[1]
    conf = lambda i, o: L.sessd_rmsnorm_configure(h, descs(*i), len(i), descs(*o), len(o))  # noqa: E731
    assert conf(NORM_IN(), NORM_OUT()) == 0
    assert conf(NORM_IN()[:2], NORM_OUT()[:2]) == 0
    refused(conf(NORM_IN()[:2], NORM_OUT()), E, "3 and 3")
    refused(conf(NORM_IN(), NORM_OUT()[:2]), E, "3 and 3")
    refused(L.sessd_rmsnorm_configure(h, None, 2, None, 2), E)
    refused(L.sessd_rmsnorm_configure(None, None, 2, None, 2), E)
    for i, o, code in ((change(NORM_IN(), 0, (1, 100, 47)), NORM_OUT(), E), (change(NORM_IN(), 0, (1, 99, 48)), NORM_OUT(), E),
                       (change(NORM_IN(), 0, (2, 100, 48)), NORM_OUT(), E), (change(NORM_IN(), 0, (100, 48)), NORM_OUT(), E),
                       (change(NORM_IN(), 0, dtype=I32), NORM_OUT(), U), (change(NORM_IN(), 1, (2,)), NORM_OUT(), E),
                       (change(NORM_IN(), 1, dtype=F32), NORM_OUT(), E), (change(NORM_IN(), 2, dtype=F32), NORM_OUT(), U),
                       (change(NORM_IN(), 2, (1, 100, 40)), NORM_OUT(), E), (NORM_IN(), change(NORM_OUT(), 0, dtype=F16), U),
                       (NORM_IN(), change(NORM_OUT(), 1, dtype=F16), U), (NORM_IN(), change(NORM_OUT(), 1, (1, 100, 48)), E),
                       (NORM_IN(), change(NORM_OUT(), 2, dtype=F32), U)):
        refused(conf(i, o), code, "rmsnorm")
    assert conf(NORM_IN(), NORM_OUT()) == 0
    assert L.sessd_rmsnorm_workspace_size(h, descs(*NORM_IN()), 3, descs(*NORM_OUT()), 3) == 0
    i, o = descs(*NORM_IN()), descs(*NORM_OUT())
    go = lambda a, b, i=i, o=o: L.sessd_rmsnorm_enqueue(h, i, o, a, b, None, None)  # noqa: E731
    a, b = pointers(4096, 8196, 16384), pointers(32768, 65536, 131072)
    assert go(a, b) == 0 and len(launches()) == 1
    for k in range(3):
        for bad in (None, 4104):
            if not (k == 1 and bad):
                v = [4096, 8196, 16384]
                v[k] = bad
                refused(go(pointers(*v), b), E, "rmsnorm.enqueue")
            v = [32768, 65536, 131072]
            v[k] = bad
            refused(go(a, pointers(*v)), E, "rmsnorm.enqueue")
    refused(go(None, b), E)
    refused(go(a, b, descs(*NORM_IN(t=F32)), descs(*NORM_OUT(t=F32))), E, "configured")
    refused(go(a, b, descs(*NORM_IN(c=40)), o), E)
    refused(L.sessd_rmsnorm_enqueue(None, i, o, a, b, None, None), E)
    # without a residual the third tensors are not looked at
    assert conf(NORM_IN()[:2], NORM_OUT()[:2]) == 0
    assert L.sessd_rmsnorm_enqueue(h, descs(*NORM_IN()[:2]), descs(*NORM_OUT()[:2]), pointers(4096, 8192), pointers(32768, 65536), None, None) == 0
    assert len(launches()) == 1
    L.sessd_rmsnorm_destroy(h)
    L.sessd_rmsnorm_destroy(None)


LIN_IN = [((1, 100, 32), FP8), ((1, 100, 1), F32), ((1,), I32)]
LIN_OUT = [((1, 100, 20), F16)]


def check_linear():
    E, U = D.SESSD_E_INVALID, D.SESSD_E_UNSUPPORTED
    h = linear()[1]
    conf = lambda i, o: L.sessd_linear8_configure(h, descs(*i), len(i), descs(*o), len(o))  # noqa: E731
    assert conf(LIN_IN, change(LIN_OUT, 0, dtype=F32)) == 0 and conf(LIN_IN, LIN_OUT) == 0
    for i, o, code in ((LIN_IN[:2], LIN_OUT, E), (LIN_IN, LIN_OUT * 2, E), (change(LIN_IN, 0, dtype=F16), LIN_OUT, U), (change(LIN_IN, 1, dtype=F16), LIN_OUT, U),
                       (change(LIN_IN, 0, (1, 100, 16)), LIN_OUT, E), (change(LIN_IN, 1, (1, 100, 32)), LIN_OUT, E), (change(LIN_IN, 2, (0,)), LIN_OUT, E),
                       (LIN_IN, change(LIN_OUT, 0, (1, 100, 24)), E), (LIN_IN, change(LIN_OUT, 0, (1, 96, 20)), E), (LIN_IN, change(LIN_OUT, 0, dtype=FP8), U)):
        refused(conf(i, o), code, "linear8")
    i, o = descs(*LIN_IN), descs(*LIN_OUT)
    go = lambda a, b, o=o: L.sessd_linear8_enqueue(h, i, o, a, b, None, None)  # noqa: E731
    assert go(pointers(4096, 8192, 12292), pointers(16384)) == 0 and len(launches()) == 1
    for v, w in (((4097, 8192, 64), 16384), ((4096, 8200, 64), 16384), ((4096, 8192, 64), 16392), ((0, 8192, 64), 16384), ((4096, 0, 64), 16384),
                 ((4096, 8192, 0), 16384), ((4096, 8192, 64), 0)):
        refused(go(pointers(*v), pointers(w)), E, "linear8.enqueue")
    refused(go(pointers(4096, 8192, 64), pointers(16384), descs(*change(LIN_OUT, 0, dtype=F32))), E, "configured")
    L.sessd_linear8_destroy(h)


ATT_IN = [((1, 100, 128), F16), ((1, 100, 4), I32), ((1,), I32)]
ATT_OUT = [((1, 100, 64), F16)]


def check_attention():
    E, U = D.SESSD_E_INVALID, D.SESSD_E_UNSUPPORTED
    h = attention()[1]
    conf = lambda i, o: L.sessd_voxelattn_configure(h, descs(*i), len(i), descs(*o), len(o))  # noqa: E731
    both = lambda t: (change(ATT_IN, 0, dtype=t), change(ATT_OUT, 0, dtype=t))  # noqa: E731
    assert conf(*both(F32)) == 0 and conf(ATT_IN, ATT_OUT) == 0
    for i, o, code in ((ATT_IN[:2], ATT_OUT, E), (ATT_IN, ATT_OUT * 2, E), (*both(I32), U), (*both(FP8), U), (ATT_IN, change(ATT_OUT, 0, dtype=F32), U),
                       (change(ATT_IN, 0, (1, 100, 192)), ATT_OUT, E), (change(ATT_IN, 1, (1, 100, 3)), ATT_OUT, E), (change(ATT_IN, 1, dtype=F32), ATT_OUT, E),
                       (change(ATT_IN, 2, (3,)), ATT_OUT, E), (ATT_IN, change(ATT_OUT, 0, (1, 100, 128)), E), (ATT_IN, change(ATT_OUT, 0, (1, 101, 64)), E)):
        refused(conf(i, o), code, "voxelattn")
    i, o = descs(*ATT_IN), descs(*ATT_OUT)
    size = L.sessd_voxelattn_workspace_size(h, i, 3, o, 1)
    assert 0 < size < 1 << 20
    a, b = pointers(4096, 8192, 12292), pointers(16384)
    for call, n in ((L.sessd_voxelattn_enqueue, 2), (L.sessd_voxelattn_enqueue_shared, 1)):
        assert call(h, i, o, a, b, 65536, None) == 0
        assert len(launches()) == n
        for v, w, ws in (((4104, 8192, 64), 16384, 65536), ((4096, 8200, 64), 16384, 65536), ((4096, 8192, 64), 16386, 65536), ((0, 8192, 64), 16384, 65536),
                         ((4096, 0, 64), 16384, 65536), ((4096, 8192, 0), 16384, 65536), ((4096, 8192, 64), 0, 65536), ((4096, 8192, 64), 16384, 0),
                         ((4096, 8192, 64), 16384, 65544)):
            refused(call(h, i, o, pointers(*v), pointers(w), ws, None), E, "voxelattn.enqueue")
        refused(call(h, descs(*both(F32)[0]), descs(*both(F32)[1]), a, b, 65536, None), E, "configured")
        refused(call(None, i, o, a, b, 65536, None), E)
    L.sessd_voxelattn_destroy(h)
    # a list of the rows by windows where there are many, from counts or from tickets; layers that share it need none
    for grid, window, own in ((GRID, WINDOW, 4), ((1000, 1000, 1), (2, 2, 1), 6)):
        h = attention(rows=5000, grid=grid, window=window)[1]
        i, o = descs(((1, 5000, 128), F16), ((1, 5000, 4), I32), ((1,), I32)), descs(((1, 5000, 64), F16))
        assert L.sessd_voxelattn_configure(h, i, 3, o, 1) == 0
        for call, n in ((L.sessd_voxelattn_enqueue, own), (L.sessd_voxelattn_enqueue_shared, 1)):
            assert call(h, i, o, a, b, 65536, None) == 0
            assert len(launches()) == n
        L.sessd_voxelattn_destroy(h)


def blob_of(name, h):
    n = getattr(L, "sessd_%s_serialization_size" % name)(h)
    buf = C.create_string_buffer(n)
    assert getattr(L, "sessd_%s_serialize" % name)(h, buf) == 0
    return buf.raw


def check_life():
    """Serialised, read back, cloned, made by name: the same plugin; blobs that are too short are refused."""
    rng = np.random.default_rng(0)
    w, gamma, slopes = rng.standard_normal((32, 20)).astype(np.float32), rng.standard_normal(48).astype(np.float32), [3, 2, 1, 0.5]
    lin = linear(w=w)[1]
    sc, sh = rng.standard_normal(20).astype(np.float32), rng.standard_normal(20).astype(np.float32)
    assert L.sessd_linear8_set_epilogue(lin, sc.ctypes.data, sh.ctypes.data, 1) == 0
    for name, h in (("rmsnorm", norm(gamma=gamma)[1]), ("linear8", lin), ("linear8", linear(w=w)[1]), ("voxelattn", attention(slopes=slopes, cap=3.0)[1]),
                    ("voxelattn", attention()[1])):
        blob = blob_of(name, h)
        g = C.c_void_p()
        assert getattr(L, "sessd_%s_deserialize" % name)(blob, len(blob), C.byref(g)) == 0
        assert blob_of(name, g) == blob
        c = C.c_void_p()
        assert getattr(L, "sessd_%s_clone" % name)(h, C.byref(c)) == 0 and blob_of(name, c) == blob
        assert getattr(L, "sessd_%s_clone" % name)(None, C.byref(c)) == D.SESSD_E_INVALID
        shortest = {"rmsnorm": len(blob), "linear8": 12 + w.nbytes, "voxelattn": len(blob)}[name]
        for n in (0, 3, 11, shortest - 4, shortest - 1):
            bad = C.c_void_p()
            refused(getattr(L, "sessd_%s_deserialize" % name)(blob, n, C.byref(bad)), D.SESSD_E_INVALID, "too short")
            assert not bad.value
        if len(blob) > shortest:
            refused(L.sessd_linear8_deserialize(blob, len(blob) - 1, C.byref(C.c_void_p())), D.SESSD_E_INVALID, "truncated")
        for k in (h, g, c):
            getattr(L, "sessd_%s_destroy" % name)(k)
    assert L.sessd_rmsnorm_deserialize((2 ** 31 - 1).to_bytes(4, "little") + bytes(8), 12, C.byref(C.c_void_p())) == D.SESSD_E_INVALID
    i = lambda *v: np.array(v, np.int32)  # noqa: E731
    f = lambda *v: np.array(v, np.float32)  # noqa: E731
    fields = {"RmsNormPlugin": dict(channel=i(48), max_voxels=i(100), eps=f(1e-6), gamma=gamma),
              "Linear8Plugin": dict(in_channel=i(32), out_channel=i(20), max_voxels=i(100), weights=w.reshape(-1)),
              "VoxelAttentionPlugin": dict(num_heads=i(4), num_kv_heads=i(2), head_dim=i(16), max_voxels=i(100), spatial_shape=i(*GRID), window_shape=i(*WINDOW),
                                           window_shift=i(0, 0, 0), cell_size=f(1, 1, 1), softmax_scale=f(0), score_cap=f(3), slopes=f(*slopes))}
    same = {"RmsNormPlugin": norm(gamma=gamma)[1], "Linear8Plugin": linear(w=w)[1], "VoxelAttentionPlugin": attention(slopes=slopes, cap=3.0)[1]}
    for name, fs in fields.items():
        assert [k for k, _, _ in api.plugin_field_names(name)] == list(fs)
        p = api.create_plugin(name, fs)
        assert p.serialize() == blob_of(p.kind, same[name]) and p.max_voxels == 100
        assert p.clone().serialize() == p.serialize()
        for missing in fs:
            try:
                api.create_plugin(name, {k: v for k, v in fs.items() if k != missing})
                raise AssertionError(missing)
            except api.SessdError as e:
                assert missing in str(e)
        last = list(fs)[-1]
        try:
            api.create_plugin(name, dict(fs, **{last: fs[last][:-1]}))
            raise AssertionError(last)
        except api.SessdError as e:
            assert last in str(e)


def check_weights():
    """The weights that Linear8 gives the GPU are the e4m3 nearest to W / wscale, each in its place."""
    sys.path.insert(0, os.path.join(ROOT, "tests"))
    import layer_oracle as O
    vals = O.VALUES[:0x7f]
    x = np.concatenate([vals, (vals[1:] + vals[:-1]) / 2, np.nextafter(((vals[1:] + vals[:-1]) / 2).astype(np.float32), np.float32(1e9)),
                        np.nextafter(((vals[1:] + vals[:-1]) / 2).astype(np.float32), np.float32(0)), [460.0, 1e-30]])
    codes = O.to_e4m3(x)
    near = np.abs(vals[None] - np.minimum(x, 448)[:, None])
    assert (np.abs(O.VALUES[codes] - np.minimum(x, 448)) == near.min(1)).all()
    tie = (near == near.min(1, keepdims=True)).sum(1) > 1
    assert tie.sum() >= 100 and (codes[tie] % 2 == 0).all()


CHECKS = {"create": check_create, "norm": check_norm, "linear": check_linear, "attention": check_attention, "life": check_life, "weights": check_weights}

if __name__ == "__main__":
    CHECKS[sys.argv[2]]()
    print("ok")
