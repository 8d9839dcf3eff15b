"""CPU test of the 4-bit cache's division of a group's span by 15."""
import shutil
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent


def test_a_fifteenth_is_the_rounded_quotient(tmp_path):
    """tests/csrc/test_kv4_fifteenth.cu runs the kernel's function as host code."""
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(nvcc).exists():
        pytest.skip("nvcc not available")
    exe = tmp_path / "test_kv4_fifteenth"
    subprocess.run([nvcc, "-std=c++17", "-O1", "-gencode", "arch=compute_100a,code=sm_100a", "-o",
                    str(exe), str(HERE / "csrc" / "test_kv4_fifteenth.cu")], check=True,
                   capture_output=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout + out.stderr
    assert out.stdout.startswith("ok")
