"""The C++ mirror of the paged entry points (include/cbx_layer_helpers.hpp):
compiles and links on the CPU box, and its test program
(tests/cpp/test_paged_helpers.cpp) passes on a GPU."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA = "/usr/local/cuda"


def _build(tmp_path):
    from chatterbox_amdvulkan_b200 import _lib, build
    if not os.path.exists(_lib.LIB_PATH):
        build.build()
    exe, pkg = os.path.join(str(tmp_path), "test_paged_helpers"), os.path.dirname(_lib.LIB_PATH)
    cmd = [shutil.which("g++") or "/usr/bin/g++", "-std=c++17", "-O1", "-Wall", "-I", os.path.join(ROOT, "include"),
           "-I", os.path.join(CUDA, "include"), os.path.join(ROOT, "tests", "cpp", "test_paged_helpers.cpp"),
           "-o", exe, "-L", pkg, "-lcbx_ops", "-L", os.path.join(CUDA, "lib64"), "-lcudart",
           f"-Wl,-rpath,{pkg}:{os.path.join(CUDA, 'lib64')}"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    return exe


def test_paged_helpers_compile_and_link(tmp_path):
    assert os.path.exists(_build(tmp_path))


@pytest.mark.gpu
def test_paged_helpers_on_gpu(tmp_path):
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    r = subprocess.run([_build(tmp_path)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "PASSED" in r.stdout
