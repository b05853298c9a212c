"""The C++ paged helpers refuse tensors that are not dense (tests/cpp/test_paged_refusals.cpp); no GPU needed."""
import os
import shutil
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA = "/usr/local/cuda"


def test_paged_helpers_refuse_tensors_with_gaps(tmp_path):
    from chatterbox_amdvulkan_b200 import _lib, build
    if not os.path.exists(_lib.LIB_PATH):
        build.build()
    exe, pkg = os.path.join(str(tmp_path), "test_paged_refusals"), os.path.dirname(_lib.LIB_PATH)
    cmd = [shutil.which("g++") or "/usr/bin/g++", "-std=c++17", "-O1", "-Wall", "-I", os.path.join(ROOT, "include"),
           "-I", os.path.join(CUDA, "include"), os.path.join(ROOT, "tests", "cpp", "test_paged_refusals.cpp"),
           "-o", exe, "-L", pkg, "-lcbx_ops", f"-Wl,-rpath,{pkg}"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "PASSED" in r.stdout, r.stdout + r.stderr
