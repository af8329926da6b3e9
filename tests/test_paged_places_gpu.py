"""Where the paged-cache operators' arrays may lie: pinned host memory beside the device's."""

import numpy as np
import pytest

from oracle import paged as oracle
from pegaflow_amd.runtime import DeviceArray, PinnedBuffer, synchronize
from test_paged_cache_gpu import (FORMS, LLAMA, Batch, device_array, device_rows, values,
                                  workspace)  # noqa: F401

pytestmark = pytest.mark.gpu


class Pinned:
    """Arrays in one pinned allocation."""

    def __init__(self, nbytes):
        self.buffer, self.used = PinnedBuffer(nbytes), 0

    def array(self, x, dtype):
        x = np.ascontiguousarray(x)
        at, self.used = self.used, self.used + -(-x.nbytes // 256) * 256
        self.buffer.array[at:at + x.nbytes] = x.view(np.uint8).reshape(-1)
        return DeviceArray(x.shape, dtype, self.buffer, at)

    def view(self, a, dtype=np.uint16):
        return self.buffer.array[a._offset:a._offset + a.nbytes].view(dtype).reshape(a.shape)


@pytest.mark.parametrize("form,group", [(LLAMA, 4), (FORMS[4], 5)], ids=str)
def test_rows_and_indexes_in_pinned_memory(gpu, workspace, form, group):
    kind, rows, heads, dim, bs, _ = form
    b = Batch([1, 40, 1], [300, 90, 2000], form, group, seed=60, strides="contiguous")
    rng = np.random.default_rng(61)
    host = Pinned(4 << 20)
    # Two tokens written and read back.
    k, v = values(rng, (2, heads, dim), rows), values(rng, (2, heads, dim), rows)
    slots = b.table[0, 3].astype(np.int64) * bs + np.arange(2)
    b.dev.cache.write(host.array(k, rows), host.array(v, rows), host.array(slots, "int64"))
    ko, vo = host.array(np.zeros_like(k), rows), host.array(np.zeros_like(v), rows)
    b.dev.cache.read(host.array(slots, "int64"), ko, vo)
    back = [device_rows(np.zeros_like(k), rows=rows)[0] for _ in range(2)]
    b.dev.cache.read(device_array(slots, "int64"), *back)
    out = host.array(np.zeros_like(b.q), rows)
    lse = host.array(np.zeros(b.q.shape[:2], np.float32), "fp32")
    b.dev.cache.attend(host.array(b.q, rows), out, host.array(b.table, "int32"),
                       host.array(b.lens, "int32"), host.array(b.starts, "int32"), lse=lse,
                       workspace=workspace)
    synchronize()
    for x, y in zip((ko, vo), back):
        assert np.array_equal(host.view(x), y.download().view(np.uint16).reshape(x.shape))
    b.pages.set(slots, k, v)
    assert np.array_equal(b.dev.bytes(), b.pages.bytes)
    got = host.view(out).copy()
    b.check(got, host.view(lse, np.float32))
    assert oracle.from_bits(got, rows).any()


def test_the_same_bits_every_time(gpu, workspace):
    """Shares are joined in order whoever finishes first: many rows, few, and both."""
    for new, cached in (((300,), (9000,)), ((1,), (9000,)), ((70, 1, 5), (3000, 4000, 10))):
        b = Batch(new, cached, LLAMA, 4, seed=62)
        first = b.run(workspace=workspace)
        for _ in range(5):
            again = b.run(workspace=workspace)
            assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])
