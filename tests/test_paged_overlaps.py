"""Memory that a call on all layers of a cache may not be given twice, on the host (CPU only)."""

import os
import shutil
import subprocess

import pytest

from pegaflow_amd import _lib, build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")


@pytest.mark.skipif(not shutil.which("g++"), reason="g++ is not installed")
def test_memory_given_twice_is_refused(tmp_path):
    """tests/native/paged_overlap_test.cpp: layers that overlap,
    anywhere, lengths written where others are read, and nothing else."""
    _lib.load()  # built, if it was not
    exe = str(tmp_path / "paged_overlap_test")
    lib = os.path.dirname(build.LIB)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-D__HIP_PLATFORM_AMD__",
                    f"-I{ROCM}/include", f"-I{ROOT}/include",
                    os.path.join(ROOT, "tests", "native", "paged_overlap_test.cpp"), "-o", exe,
                    "-rdynamic", f"-L{lib}", f"-Wl,-rpath,{lib}", "-lpegaflow_hip",
                    f"-Wl,-rpath-link,{ROCM}/lib"], check=True)
    r = subprocess.run([exe], timeout=120, stdout=subprocess.PIPE, text=True)
    assert r.returncode == 0 and r.stdout.endswith("ok\n"), r.stdout
