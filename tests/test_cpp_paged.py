"""The paged key-value cache from C++ (examples/paged_decode.cpp on
include/mxmoe.hpp): it compiles against the C ABI, refuses bad configurations
with exceptions, and on a GPU agrees with dense attention on the host."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIBDIR = os.path.join(ROOT, "burn-extended_b200", "mxmoe")
SRC = os.path.join(ROOT, "burn-extended_b200", "examples", "paged_decode.cpp")
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("cpp") / "paged_decode")
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "include"), "-I", os.path.join(CUDA, "include"), SRC,
                    "-o", out, "-L", LIBDIR, "-lmxmoe", f"-Wl,-rpath,{LIBDIR}", "-L", os.path.join(CUDA, "lib64"), "-lcudart",
                    f"-Wl,-rpath,{os.path.join(CUDA, 'lib64')}"], check=True)
    return out


def test_refusals_are_exceptions(exe):
    r = subprocess.run([exe, "--check-errors"], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "errors caught: 3" in r.stdout


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 17, 300, 5000])
def test_agrees_with_dense_attention(exe, n):
    r = subprocess.run([exe, str(n)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
