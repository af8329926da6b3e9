"""The page of a token, as attention's kernels divide, on the host (CPU only)."""

import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")


@pytest.mark.skipif(not shutil.which("g++"), reason="g++ is not installed")
def test_page_of_a_token(tmp_path):
    """tests/native/paged_division_test.cpp: set_division's multiplier and shift, for every
    block size up to 4,096 and others up to the largest."""
    exe = str(tmp_path / "paged_division_test")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-D__HIP_PLATFORM_AMD__",
                    f"-I{ROCM}/include", f"-I{ROOT}/include", f"-I{ROOT}/pegaflow_amd/csrc",
                    os.path.join(ROOT, "tests", "native", "paged_division_test.cpp"), "-o", exe],
                   check=True)
    r = subprocess.run([exe], timeout=120, stdout=subprocess.PIPE, text=True)
    assert r.returncode == 0 and r.stdout.endswith("ok\n"), r.stdout
