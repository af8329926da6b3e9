"""Vector registers that the attention kernels spill, as the built library's own notes say (CPU
only): a change that makes a kernel spill more than it is known to shows here."""

import os
import re
import shutil
import struct
import subprocess

import pytest

from pegaflow_amd import _lib, build

ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
READELF = os.path.join(ROCM, "llvm", "bin", "llvm-readelf")
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"

# Of attend_many_kernel<rows, pages, head size, rows of a tile> and attend_shared_kernel<rows,
# pages, head size>; all others spill none.  Pages: 1 bf16, 2 fp16, 3 e4m3, 4 int8.
KNOWN = {
    ("attend_many_kernel", "BF16", 1, 128, 128): 11, ("attend_many_kernel", "FP16", 2, 128, 128): 11,
    ("attend_many_kernel", "BF16", 1, 256, 128): 31, ("attend_many_kernel", "FP16", 2, 256, 128): 31,
    ("attend_many_kernel", "FP16", 3, 128, 128): 2, ("attend_many_kernel", "BF16", 3, 256, 128): 6,
    ("attend_shared_kernel", "BF16", 1, 256): 6, ("attend_shared_kernel", "FP16", 2, 256): 6,
    ("attend_shared_kernel", "BF16", 3, 256): 6,
}


def code_objects():
    """The GPU's code objects in the library."""
    with open(build.LIB, "rb") as f:
        data = f.read()
    at = data.find(MAGIC)
    while at >= 0:
        entries, = struct.unpack_from("<Q", data, at + len(MAGIC))
        p = at + len(MAGIC) + 8
        for _ in range(entries):
            offset, size, length = struct.unpack_from("<QQQ", data, p)
            if data[p + 24:p + 24 + length].endswith(build.ARCH.encode()) and size:
                yield data[at + offset:at + offset + size]
            p += 24 + length
        at = data.find(MAGIC, at + 1)


@pytest.mark.skipif(not (os.path.exists(READELF) and shutil.which("c++filt")),
                    reason="llvm-readelf or c++filt is not installed")
def test_spilled_registers(tmp_path):
    _lib.load()  # built, if it was not
    spills = {}
    for i, code in enumerate(code_objects()):
        path = tmp_path / f"{i}.elf"
        path.write_bytes(code)
        notes = subprocess.run([READELF, "--notes", str(path)], check=True, capture_output=True,
                               text=True).stdout
        for part in notes.split("  - .agpr_count")[1:]:
            name = re.search(r"\.name:\s+(\S+)", part)[1]
            spills[name] = int(re.search(r"\.vgpr_spill_count:\s+(\d+)", part)[1])
    names = subprocess.run(["c++filt", *spills], check=True, capture_output=True,
                           text=True).stdout.split("\n")
    seen = set()
    for name, count in zip(names, spills.values()):
        kernel = re.search(r"(attend_\w+)<(?:pf::)?(BF16|FP16), ([^>]*)>", name)
        if not kernel:
            continue
        of = (kernel[1], kernel[2], *(int(x.rstrip("u")) for x in kernel[3].split(", ")
                                      if x.rstrip("u").isdigit()))
        seen.add(of)
        assert count <= KNOWN.get(of, 0), (of, count)
    assert KNOWN.keys() <= seen and len(seen) > 100
