"""The kernels' bounded waits on the GPU (tests/cpp/wait_check.cu): limits of milliseconds that
run out on flags that nothing sets, and the status that is read then."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def build(path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    exe = path / "wait_check"
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O2", "--expt-relaxed-constexpr",
                    "-o", str(exe), os.path.join(ROOT, "tests", "cpp", "wait_check.cu")], check=True)
    return exe


def test_wait_check_compiles(tmp_path):
    build(tmp_path)


@pytest.mark.gpu
def test_waits_give_up_and_settle(tmp_path):
    out = subprocess.run([str(build(tmp_path))], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr
