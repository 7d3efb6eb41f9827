"""The host side of RmsNorm, Linear8 and VoxelAttention: what they refuse, their blobs, clones and creators.  Nothing runs on a GPU: the
library is loaded onto a stand-in for the HIP runtime (fake_hip.cpp) in a process of its own (host_layers.py)."""
import os
import shutil
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def fake_hip(tmp_path_factory):
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    if not shutil.which("g++"):
        pytest.skip("no C++ compiler")
    out = str(tmp_path_factory.mktemp("fake_hip") / "libfake_hip.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(rocm, "include"),
                    os.path.join(HERE, "fake_hip.cpp"), "-o", out], check=True)
    return out


@pytest.mark.parametrize("check", ["create", "norm", "linear", "attention", "life", "weights"])
def test_host_side(fake_hip, check):
    r = subprocess.run([sys.executable, os.path.join(HERE, "host_layers.py"), fake_hip, check], stdout=subprocess.PIPE, stderr=subprocess.STDOUT,
                       text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.rstrip().endswith("ok"), r.stdout[-4000:]


def test_struct_layouts_match_the_header(tmp_path):
    import ctypes as C
    from sessd3d import ctypes_defs as D
    if not shutil.which("gcc"):
        pytest.skip("no C compiler")
    pairs = [("sessd_rmsnorm_desc", D.RmsNormDesc), ("sessd_linear8_desc", D.Linear8Desc), ("sessd_voxelattn_desc", D.VoxelAttnDesc)]
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "sessd3d.h"', 'int main(void) {', '    printf("FP8 %d\\n", (int)SESSD_FP8);']
    for cname, mirror in pairs:
        lines.append('    printf("%s %%zu\\n", sizeof(%s));' % (cname, cname))
        lines += ['    printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (cname, f, cname, f) for f, _ in mirror._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["    return 0;", "}"]) + "\n")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Wextra", "-pedantic", "-Werror", "-I", os.path.join(HERE, "..", "include"), str(src), "-o", str(exe)], check=True)
    out = dict(l.split() for l in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    assert int(out["FP8"]) == D.SESSD_FP8
    for cname, mirror in pairs:
        assert int(out[cname]) == C.sizeof(mirror)
        for f, _ in mirror._fields_:
            assert int(out["%s.%s" % (cname, f)]) == getattr(mirror, f).offset


def test_tensors_in_host_memory_are_refused():
    import torch
    from sessd3d import api
    with pytest.raises(api.SessdError, match="not in GPU memory"):
        api._dense(torch.zeros(4, 4))
    with pytest.raises(api.SessdError, match="contiguous"):
        api._dense(torch.zeros(4, 6).t())
