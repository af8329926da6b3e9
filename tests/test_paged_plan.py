"""The launch rules of attention over the paged cache, on the host (CPU only)."""

import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")


@pytest.mark.skipif(not shutil.which("g++"), reason="g++ is not installed")
def test_attention_launch_rules(tmp_path):
    """tests/native/paged_plan_test.cpp: tiles, shares and their places in the workspace."""
    exe = str(tmp_path / "paged_plan_test")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-D__HIP_PLATFORM_AMD__",
                    f"-I{ROCM}/include", f"-I{ROOT}/include", f"-I{ROOT}/pegaflow_amd/csrc",
                    os.path.join(ROOT, "tests", "native", "paged_plan_test.cpp"), "-o", exe],
                   check=True)
    r = subprocess.run([exe], timeout=120, stdout=subprocess.PIPE, text=True)
    assert r.returncode == 0 and r.stdout.endswith("ok\n"), r.stdout
