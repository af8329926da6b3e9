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


class Tensor:
    """A tensor's face without memory."""

    def __init__(self, shape, dtype):
        self.shape, self.dtype = shape, dtype

    def stride(self):
        out = [1]
        for n in reversed(self.shape[1:]):
            out.insert(0, out[0] * n)
        return tuple(out)

    def data_ptr(self):
        return BASE


@pytest.mark.parametrize("value", [0, 7, (1 << 32) - 1, 1 << 32, (1 << 32) + 5, (1 << 63) - 1])
def test_bounds_past_32_bits_bound_nothing(monkeypatch, value):
    """A window, a length or a number of rows that 32 bits do not hold is not cut to some other."""
    from pegaflow_amd import paged_cache

    class Library:
        def pf_kv_attend(self, pages, args, workspace, stream):
            seen.append(args._obj)
            return 0

    seen = []
    c = cache()
    monkeypatch.setattr(paged_cache, "lib", Library)
    c.attend(Tensor((5, 4, 64), "bf16"), Tensor((5, 4, 64), "bf16"), Tensor((2, 4), "int32"),
             Tensor((2,), "int32"), Tensor((3,), "int32"), window=value, max_seq_len=value,
             max_query_len=value)
    a, = seen
    want = min(value, (1 << 32) - 1)
    assert (a.window, a.max_seq_len, a.max_query_len) == (want, want, want)


@pytest.mark.parametrize("at", [0, 1, 2])
def test_sizes_past_32_bits_are_refused(at):
    for value in ((1 << 32) + 16, -16):
        sizes = [16, 2, 64]
        sizes[at] = value
        with pytest.raises(ValueError):
            segment_bytes(*sizes, "bf16")
        seg = segment_bytes(16, 2, 64, "bf16")
        reg = KVCacheRegistration.create(BASE, 20 * seg, 10, seg, 10 * seg, 2)
        with pytest.raises(ValueError):
            PagedKVCache(reg, *sizes, "bf16")


def test_torch_tensors_run_on_torchs_current_stream(monkeypatch):
    """Without a stream of the caller's, calls follow what torch has queued on their tensors."""
    torch = pytest.importorskip("torch")
    from pegaflow_amd import paged_cache
    from pegaflow_amd.runtime import Stream

    class OnDevice1(torch.Tensor):
        is_cuda = True

        def get_device(self):
            return 1

    def tensor(*shape, dtype=torch.bfloat16):
        return torch.zeros(shape, dtype=dtype).as_subclass(OnDevice1)

    class Library:
        def __getattr__(self, name):
            return lambda *args: seen.append(args[-1]) or 0

    seen = []
    c = cache()
    monkeypatch.setattr(paged_cache, "lib", Library)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 0x1230 + device,
                        raising=False)
    k, q = tensor(5, 2, 64), tensor(5, 4, 64)
    slots = tensor(5, dtype=torch.int64)
    batch = [tensor(*s, dtype=torch.int32) for s in ((2, 4), (2,), (3,))]
    for stream, want in ((None, 0x1231), (Stream(0x77, owned=False), 0x77)):
        c.write(k, k, slots, stream=stream)
        c.read(slots, k, k, stream=stream)
        c.attend(q, q, *batch, stream=stream)
        assert seen == [want] * 3
        seen.clear()
    face = Tensor((5, 2, 64), "bf16")
    c.write(face, face, Tensor((5,), "int64"))
    assert seen == [None]
