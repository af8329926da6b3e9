"""Paged-cache operators on registered layers: what a model does with the blocks
that the transfer path saves and restores.

``PagedKVCache`` describes a layer's blocks as pages; ``write`` puts new tokens' K
and V into them (at 16 bits, or as 8-bit codes with a scale for each token and
head), ``read`` gives them back, ``attend`` attends new tokens over them.  An 8-bit
layer keeps its scales inside its blocks, so it is saved and restored like any
other layer, at half the bytes.

Tensors are torch's, or anything with their ``data_ptr()``, ``shape``,
``stride()`` and ``dtype`` (``runtime.DeviceArray``).  Calls are asynchronous on
``stream`` (None: torch's current stream for torch's tensors, the current device's
null stream for others) and may be captured into a graph.  The reference has no counterpart: its blocks are filled and
read by the inference engine.
"""

from __future__ import annotations

import ctypes
import math
import sys

from . import _lib
from ._lib import AttendArgs, KVPages, KVRows, check
from .runtime import Stream
from .transfer import KVCacheRegistration

KV_TYPES = {"bf16": _lib.KV_BF16, "fp16": _lib.KV_FP16, "e4m3": _lib.KV_E4M3,
            "int8": _lib.KV_INT8}
_ROW_NAMES = {"bf16": _lib.KV_BF16, "bfloat16": _lib.KV_BF16, "fp16": _lib.KV_FP16,
              "float16": _lib.KV_FP16}
_row_types: dict = {}  # a tensor's dtype -> PF_KV_*
_MOST = 2 ** 32 - 1  # of a 32-bit field, which ctypes fills with a number's low bits


def lib():
    return _lib.load()


def _name(dtype) -> str:
    return str(dtype).rsplit(".", 1)[-1]


def _row_type(dtype) -> int:
    t = _row_types.get(dtype)
    if t is None:
        t = _ROW_NAMES.get(_name(dtype))
        if t is None:
            raise ValueError(f"rows are bf16 or fp16, not {dtype}")
        _row_types[dtype] = t
    return t


def _rows(x, heads: int | None, dim: int, what: str):
    """(KVRows, tokens, heads) of a [tokens, heads, head_dim] tensor."""
    shape = x.shape
    if len(shape) != 3 or shape[2] != dim or (heads is not None and shape[1] != heads):
        raise ValueError(f"{what} is [tokens, {heads or 'heads'}, {dim}], got {tuple(shape)}")
    by_token, by_head, by_value = x.stride()
    if by_value != 1:
        raise ValueError(f"{what}: the values of a row are not neighbours (stride {by_value})")
    t = _row_types.get(x.dtype) or _row_type(x.dtype)
    return KVRows(x.data_ptr(), by_token, by_head, t), shape[0], shape[1]


_index_types: dict = {}  # a tensor's dtype -> its name


def _index(x, dims: int, dtype: str, what: str):
    shape = x.shape
    name = _index_types.get(x.dtype)
    if name is None:
        name = _index_types[x.dtype] = _name(x.dtype)
    if len(shape) != dims or name != dtype:
        raise ValueError(f"{what} is a {dims}-dimensional {dtype} tensor, got "
                         f"{tuple(shape)} of {x.dtype}")
    if shape[-1] > 1 and x.stride()[-1] != 1:
        raise ValueError(f"{what}: its last dimension is not contiguous")
    return x.data_ptr()


_current_streams: dict = {}  # a tensor's type -> its device's current stream, or None


def _current_stream(kind: type):
    """What gives the handle of a device's current stream, for tensors of torch's."""
    torch = sys.modules.get("torch")
    if torch is None or not issubclass(kind, torch.Tensor):
        return None
    # current_stream() takes 1 to 2 us for its object, the other 0.1.
    return getattr(torch._C, "_cuda_getCurrentRawStream",
                   lambda device: torch.cuda.current_stream(device).cuda_stream)


def _stream(stream: Stream | None, x):
    """The handle of ``stream``, or else of the stream on which torch queues what it does
    with its tensor ``x``."""
    if stream is not None:
        return stream.handle
    kind = type(x)
    if kind not in _current_streams:
        _current_streams[kind] = _current_stream(kind)
    current = _current_streams[kind]
    if current is None:
        return None
    device = x.get_device()
    return current(device) if device >= 0 else None


def segment_bytes(block_size: int, num_kv_heads: int, head_dim: int, kv_type: str) -> int:
    """Bytes of K (or V) of one block: the values, the scales of 8-bit types, padded
    to 16 (pf_kv_segment_bytes).  A KV-first layer of such blocks is a
    [2, num_blocks, segment_bytes] uint8 tensor."""
    for n in (block_size, num_kv_heads, head_dim):
        if not 0 <= n <= _MOST:
            raise ValueError(f"pages of {block_size} tokens, {num_kv_heads} heads of {head_dim}")
    out = ctypes.c_uint64()
    check(lib().pf_kv_segment_bytes(block_size, num_kv_heads, head_dim, _kv_type(kv_type),
                                    ctypes.byref(out)), "segment_bytes")
    return out.value


def _kv_type(name: str) -> int:
    if name not in KV_TYPES:
        raise ValueError(f"unknown KV type {name!r} (one of {', '.join(KV_TYPES)})")
    return KV_TYPES[name]


class AttentionWorkspace:
    """Device memory in which ``attend`` joins the shares of split sequences
    (pf_attend_workspace).  Calls that share one must be ordered: one workspace a
    stream."""

    def __init__(self, nbytes: int = _lib.ATTEND_WORKSPACE_DEFAULT, device: int = 0):
        self.handle = None
        h = ctypes.c_void_p()
        check(lib().pf_attend_workspace_create(device, nbytes, ctypes.byref(h)),
              "pf_attend_workspace_create")
        self.handle = h.value

    def close(self) -> None:
        if self.handle:
            lib().pf_attend_workspace_destroy(self.handle)
        self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class PagedKVCache:
    """A registered layer's blocks as pages of ``block_size`` tokens (pf_kv_pages).

    ``kv_type``: what the pages hold, "bf16", "fp16", "e4m3" or "int8".
    ``head_major``: a block's values are [heads, block_size, head_dim] instead of
    [block_size, heads, head_dim].  The registration's memory is borrowed."""

    def __init__(self, registration: KVCacheRegistration, block_size: int, num_kv_heads: int,
                 head_dim: int, kv_type: str, head_major: bool = False):
        need = segment_bytes(block_size, num_kv_heads, head_dim, kv_type)
        have = registration.bytes_per_block // (1 if registration.segments == 2 else 2)
        if have < need:
            raise ValueError(f"a segment of {have} bytes cannot hold K or V of a block "
                             f"({need} bytes)")
        self.registration = registration
        self.block_size = block_size
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.kv_type = kv_type
        self.head_major = head_major
        self._pages = KVPages(registration.to_c(), block_size, num_kv_heads, head_dim,
                              _kv_type(kv_type),
                              _lib.KV_HEAD_MAJOR if head_major else _lib.KV_TOKEN_MAJOR, 0)
        self._ref = ctypes.byref(self._pages)

    def _move(self, fn, what, k, v, slots, stream):
        kr, n, _ = _rows(k, self.num_kv_heads, self.head_dim, "k")
        vr, m, _ = _rows(v, self.num_kv_heads, self.head_dim, "v")
        at = _index(slots, 1, "int64", "slots")
        if n != m or slots.shape[0] != n:
            raise ValueError(f"{n} rows of k, {m} of v and {slots.shape[0]} slots")
        check(fn(self._ref, ctypes.byref(kr), ctypes.byref(vr), at, n, _stream(stream, k)), what)

    def write(self, k, v, slots, stream: Stream | None = None) -> None:
        """Rows of ``k`` and ``v`` [tokens, kv_heads, head_dim] into ``slots`` (int64,
        block * block_size + position; distinct).  A negative slot, or one past the
        last block, is padding and written nowhere (pf_kv_write)."""
        self._move(lib().pf_kv_write, "paged write", k, v, slots, stream)

    def read(self, slots, k, v, stream: Stream | None = None) -> None:
        """The values at ``slots`` into rows of ``k`` and ``v``; rows of padding slots
        are left as they were (pf_kv_read)."""
        self._move(lib().pf_kv_read, "paged read", k, v, slots, stream)

    def attend(self, q, out, block_table, seq_lens, query_starts, *, scale: float | None = None,
               causal: bool = True, window: int = 0, lse=None, max_seq_len: int = 0,
               max_query_len: int = 0, workspace: AttentionWorkspace | None = None,
               stream: Stream | None = None) -> None:
        """Attention of new tokens ``q`` [rows, heads, head_dim] over the pages into
        ``out``, the same shape and type (pf_kv_attend).

        Sequence b has rows ``query_starts[b]`` to ``query_starts[b + 1]`` (int32),
        ``seq_lens[b]`` tokens in all (int32), the new ones last and written already,
        in the blocks ``block_table[b]`` (int32).  ``window``: a row sees only so many
        tokens, itself included.  ``scale`` defaults to head_dim ** -0.5.  ``lse``, if
        given, is an fp32 [rows, heads] tensor.  ``max_seq_len``, the longest sequence, is
        a hint that shapes the launch; ``max_query_len`` says that no sequence has more
        rows, and those that one has beyond it may stay as they were.  Without a
        ``workspace`` no sequence is split, which is slow where few rows attend
        long sequences."""
        qr, n, heads = _rows(q, None, self.head_dim, "q")
        outr, m, out_heads = _rows(out, heads, self.head_dim, "out")
        if n != m:
            raise ValueError(f"{n} rows of q and {m} of out")
        table = _index(block_table, 2, "int32", "block_table")
        lens = _index(seq_lens, 1, "int32", "seq_lens")
        starts = _index(query_starts, 1, "int32", "query_starts")
        seqs, width = block_table.shape
        if seq_lens.shape[0] != seqs or query_starts.shape[0] != seqs + 1:
            raise ValueError(f"{seqs} block tables, {seq_lens.shape[0]} lengths and "
                             f"{query_starts.shape[0]} query starts (one more than sequences)")
        if window < 0 or max_seq_len < 0 or max_query_len < 0:
            raise ValueError("window, max_seq_len and max_query_len are not negative")
        lse_at = 0
        if lse is not None:
            if tuple(lse.shape) != (n, heads) or _name(lse.dtype) not in ("float32", "fp32"):
                raise ValueError(f"lse is an fp32 [{n}, {heads}] tensor")
            stride = lse.stride()
            if n and heads and (stride[1] != 1 and heads > 1 or stride[0] != heads and n > 1):
                raise ValueError("lse is not contiguous")
            lse_at = lse.data_ptr()
        args = AttendArgs(qr, outr, n, table, block_table.stride()[0], lens, starts, lse_at, heads,
                          seqs, width, min(window, _MOST), causal,
                          1 / math.sqrt(self.head_dim) if scale is None else scale,
                          min(max_seq_len, _MOST), min(max_query_len, _MOST))
        check(lib().pf_kv_attend(self._ref, ctypes.byref(args),
                                 workspace.handle if workspace is not None else None,
                                 _stream(stream, q)), "attend")


__all__ = ["KV_TYPES", "AttentionWorkspace", "PagedKVCache", "segment_bytes"]
