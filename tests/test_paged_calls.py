"""Calls of the paged-cache operators at the edges of their arguments.  No GPU."""

import pytest

from pegaflow_amd.paged_cache import PagedKVCache, segment_bytes
from pegaflow_amd.transfer import KVCacheRegistration

BASE = 0x10000000  # never dereferenced


def cache():
    seg = segment_bytes(16, 2, 64, "bf16")
    reg = KVCacheRegistration.create(BASE, 20 * seg, 10, seg, 10 * seg, 2)
    return PagedKVCache(reg, 16, 2, 64, "bf16")


def test_empty_torch_tensors_do_nothing():
    """Those have no memory: their addresses are all 0."""
    torch = pytest.importorskip("torch")
    k, v = (torch.empty(0, 2, 64, dtype=torch.bfloat16) for _ in range(2))
    slots = torch.empty(0, dtype=torch.int64)
    assert k.data_ptr() == v.data_ptr() == 0
    c = cache()
    c.write(k, v, slots)
    c.read(slots, k, v)
