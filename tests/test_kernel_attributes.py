"""Kernel attributes are set once a device: before any launch that needs them, whichever thread is first, and again after a failure."""
import os
import subprocess

from tensorlib_b200.build import NVCC

HERE = os.path.dirname(os.path.abspath(__file__))


def test_attributes_are_set_before_they_count_as_set(tmp_path):
    exe = str(tmp_path / "attributes_test")
    r = subprocess.run([NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "--expt-relaxed-constexpr", "-ccbin", "g++",
                        os.path.join(HERE, "cpp", "attributes_test.cu"), "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "OK attributes" in r.stdout, r.stdout + r.stderr
