"""What RmsNorm, Linear8 and VoxelAttention keep in device memory and when they change it.  Nothing runs on a GPU: the library is loaded onto a
stand-in for the HIP runtime (fake_hip_memory.cpp) in a process of its own (host_layer_memory.py)."""
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
    out = str(tmp_path_factory.mktemp("fake_hip_memory") / "libfake_hip_memory.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(rocm, "include"), "-I", HERE,
                    os.path.join(HERE, "fake_hip_memory.cpp"), "-o", out], check=True)
    return out


@pytest.mark.parametrize("check", ["epilogue", "device", "weights", "fields"])
def test_device_memory(fake_hip, check):
    r = subprocess.run([sys.executable, os.path.join(HERE, "host_layer_memory.py"), fake_hip, check], stdout=subprocess.PIPE, stderr=subprocess.STDOUT,
                       text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.rstrip().endswith("ok"), r.stdout[-4000:]
