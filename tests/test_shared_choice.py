"""Which way a batch of shared tokens and many rows runs, on the host (CPU only)."""

import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(not shutil.which("g++"), reason="g++ is not installed")
def test_the_faster_way_is_taken(tmp_path):
    """tests/native/paged_shared_choice_test.cpp: where the ways' measured times are far apart."""
    exe = str(tmp_path / "paged_shared_choice_test")
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-D__HIP_PLATFORM_AMD__",
                    f"-I{rocm}/include", f"-I{ROOT}/include", f"-I{ROOT}/pegaflow_amd/csrc",
                    os.path.join(ROOT, "tests", "native", "paged_shared_choice_test.cpp"), "-o",
                    exe], check=True)
    r = subprocess.run([exe], timeout=120, stdout=subprocess.PIPE, text=True)
    assert r.returncode == 0 and r.stdout.endswith("ok\n"), r.stdout
