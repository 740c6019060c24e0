"""What a failed runtime call leaves behind, and calls from several host threads,
checked on the host against a stand-in for the CUDA runtime (no GPU needed)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "ornith-flight_b200", "csrc")
NATIVE = os.path.join(ROOT, "tests", "native")
NVCC = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"


def run_check(tmp_path, name):
    if not os.path.exists(NVCC):
        pytest.skip("no nvcc")
    exe = tmp_path / name
    subprocess.run([NVCC, "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-cudart", "none", "-Xcompiler", "-pthread",
                    "-I", CSRC, "-I", os.path.join(ROOT, "include"), os.path.join(NATIVE, name + ".cu"),
                    os.path.join(NATIVE, "fake_runtime.cc"), os.path.join(CSRC, "status.cu"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert (r.returncode, r.stdout.strip()) == (0, "0"), r


def test_a_reported_failure_is_not_reported_again(tmp_path):
    run_check(tmp_path, "last_error_check")


def test_threads_never_lower_a_shared_memory_limit(tmp_path):
    run_check(tmp_path, "smem_limit_check")
