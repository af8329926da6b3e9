"""Paged-cache operators on registered layers: what a model does with the blocks
that the transfer path saves and restores.

``PagedKVCache`` describes a layer's blocks as pages; ``write`` puts new tokens' K
and V into them (at 16 bits, or as 8-bit codes with a scale for each token and
head), ``write_rotated`` does so as it turns queries and keys to their positions
(``RotaryPositions``), ``read`` gives them back, ``attend`` attends new tokens over
them.  An 8-bit layer keeps its scales inside its blocks, so it is saved and restored
like any other layer, at half the bytes.  ``PagedLayers`` moves blocks and tokens
within all layers at once: forks of sequences, copies of blocks, kept tokens moved
together.

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
from ._lib import AttendArgs, CompactArgs, ForkArgs, KVPages, KVRows, SharedArgs, check
from .runtime import Stream
from .transfer import KVCacheRegistration

KV_TYPES = {"bf16": _lib.KV_BF16, "fp16": _lib.KV_FP16, "e4m3": _lib.KV_E4M3,
            "int8": _lib.KV_INT8}
_ROW_NAMES = {"bf16": _lib.KV_BF16, "bfloat16": _lib.KV_BF16, "fp16": _lib.KV_FP16,
              "float16": _lib.KV_FP16}
_row_types: dict = {}  # a tensor's dtype -> PF_KV_*
SHARE_ANYWAY = _lib.SHARED_LEN_ANYWAY
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


def _most(what: str, n: int) -> int:
    """A hint or bound that a 32-bit field holds."""
    if n < 0:
        raise ValueError(f"{what} is not negative")
    return min(n, _MOST)


def _wavelengths(rotary_dim: int, base: float, scaling: dict | None):
    """(radians a position of each pair, factor of turned values) of a named scaling."""
    if not base > 0:
        raise ValueError(f"base {base}")
    pairs = range(rotary_dim // 2)
    s = dict(scaling or {"type": "none"})
    kind = s.pop("type", None)
    takes = {"none": (), "linear": ("factor",), "ntk": ("factor",),
             "llama3": ("factor", "original_max_position", "low_freq_factor", "high_freq_factor"),
             "yarn": ("factor", "original_max_position", "beta_fast", "beta_slow",
                      "attention_factor")}
    if kind not in takes:
        raise ValueError(f"unknown scaling {kind!r} (one of {', '.join(takes)})")
    needed = set(takes[kind][:2])
    if set(s) - set(takes[kind]) or needed - set(s):
        raise ValueError(f"scaling {kind!r} takes {', '.join(takes[kind])}, got {', '.join(s)}")
    by = float(s.get("factor", 1.0))
    if not by > 0 or not float(s.get("original_max_position", 1)) > 0:
        raise ValueError("scaling: factor and original_max_position are above 0")
    if kind == "ntk" and rotary_dim > 2:
        base = base * by ** (rotary_dim / (rotary_dim - 2))
    f = [base ** (-2 * i / rotary_dim) for i in pairs]
    if kind == "linear":
        return [x / by for x in f], 1.0
    if kind == "llama3":
        # By the turns that a pair makes over the original context: many, and it stays; few,
        # and it is stretched; in between a mean of both.
        low, high = float(s.get("low_freq_factor", 1.0)), float(s.get("high_freq_factor", 4.0))
        if not high > low:
            raise ValueError("scaling: high_freq_factor is above low_freq_factor")
        out = []
        for x in f:
            turns = s["original_max_position"] * x / (2 * math.pi)
            keep = min(max((turns - low) / (high - low), 0.0), 1.0)
            out.append(keep * x + (1 - keep) * x / by)
        return out, 1.0
    if kind == "yarn":
        # As above, along the index of the pair, between those that make beta_fast and
        # beta_slow turns.
        fast, slow = float(s.get("beta_fast", 32.0)), float(s.get("beta_slow", 1.0))
        if not fast > slow > 0 or not base > 1:
            raise ValueError("scaling: beta_fast is above beta_slow, beta_slow above 0, base above 1")

        def index(turns):
            return (rotary_dim * math.log(s["original_max_position"] / (turns * 2 * math.pi))
                    / (2 * math.log(base)))

        low = max(math.floor(index(fast)), 0)
        high = min(math.ceil(index(slow)), rotary_dim - 1)
        width = high - low if high != low else 0.001
        out = []
        for i, x in enumerate(f):
            stretch = min(max((i - low) / width, 0.0), 1.0)
            out.append(stretch * x / by + (1 - stretch) * x)
        factor = s.get("attention_factor")
        if factor is None:
            factor = 0.1 * math.log(by) + 1.0 if by > 1 else 1.0
        return out, float(factor)
    return f, 1.0


class RotaryPositions:
    """The angles by which a model turns queries and keys to their positions (pf_rotary).

    The first ``rotary_dim`` values of a head are turned, in pairs: ``layout`` "half" pairs
    values i and i + rotary_dim / 2, "interleaved" 2 i and 2 i + 1.  Pair i turns by
    ``base`` ** (-2 i / rotary_dim) radians a position, for contexts beyond the trained
    ones by less, as ``scaling`` says:

    * {"type": "linear", "factor": s}: all s times slower;
    * {"type": "ntk", "factor": s}: base * s ** (rotary_dim / (rotary_dim - 2));
    * {"type": "llama3", "factor": s, "original_max_position": n}: s times slower where a
      pair turns once or less over n positions, as before where four times or more
      ("low_freq_factor" 1, "high_freq_factor" 4);
    * {"type": "yarn", "factor": s, "original_max_position": n}: the same along the index,
      between 32 turns and one ("beta_fast", "beta_slow"), turned values 0.1 ln s + 1
      times as large ("attention_factor").

    Or ``frequencies`` are the radians a position of each pair, and ``factor`` that of turned
    values.  No angle loses precision at far positions.  It lives on ``device``, one for all
    layers; close it after the last call, or graph, that uses it."""

    def __init__(self, rotary_dim: int, *, base: float = 10000.0, layout: str = "half",
                 scaling: dict | None = None, frequencies=None, factor: float | None = None,
                 device: int = 0):
        self.handle = None
        if rotary_dim < 2 or rotary_dim % 2:
            raise ValueError(f"rotary_dim {rotary_dim} is not an even number from 2 on")
        if layout not in ("half", "interleaved"):
            raise ValueError(f"unknown layout {layout!r} (half or interleaved)")
        if frequencies is None:
            if factor is not None:
                raise ValueError("a factor goes with frequencies")
            frequencies, factor = _wavelengths(rotary_dim, base, scaling)
        elif scaling is not None:
            raise ValueError("either frequencies or a scaling")
        self.frequencies = [float(x) for x in frequencies]
        self.factor = 1.0 if factor is None else float(factor)
        if len(self.frequencies) != rotary_dim // 2:
            raise ValueError(f"{len(self.frequencies)} frequencies of {rotary_dim // 2} pairs")
        self.rotary_dim = rotary_dim
        self.layout = layout
        h = ctypes.c_void_p()
        check(lib().pf_rotary_create(
            device, (ctypes.c_double * len(self.frequencies))(*self.frequencies),
            len(self.frequencies),
            _lib.ROTARY_HALF if layout == "half" else _lib.ROTARY_INTERLEAVED, self.factor,
            ctypes.byref(h)), "pf_rotary_create")
        self.handle = h.value

    def rotate(self, x, out, positions, stream: Stream | None = None) -> None:
        """Rows of ``x`` [tokens, heads, head_dim], turned to ``positions`` (int64), into
        ``out``, the same shape and type, which may be ``x`` itself (pf_rotary_rotate)."""
        dim = x.shape[-1]
        xr, n, heads = _rows(x, None, dim, "x")
        outr, m, _ = _rows(out, heads, dim, "out")
        at = _index(positions, 1, "int64", "positions")
        if n != m or positions.shape[0] != n:
            raise ValueError(f"{n} rows of x, {m} of out and {positions.shape[0]} positions")
        if n >= 2 ** 31 or heads > _MOST or dim > _MOST:
            raise ValueError(f"rows [{n}, {heads}, {dim}] are too many")
        check(lib().pf_rotary_rotate(self.handle, ctypes.byref(xr), ctypes.byref(outr), at, n,
                                     heads, dim, _stream(stream, x)), "rotate")

    def close(self) -> None:
        if self.handle:
            lib().pf_rotary_destroy(self.handle)
        self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


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

    def write_rotated(self, q, q_out, k, v, positions, slots, rotary: RotaryPositions,
                      stream: Stream | None = None) -> None:
        """Queries ``q`` [tokens, heads, head_dim], turned to their ``positions`` (int64),
        into ``q_out`` (which may be ``q`` itself), and rows of ``k``, turned, and of ``v`` into
        ``slots``, as ``write`` does (pf_kv_write_rotated).  A turned key is rounded once, to
        what the pages hold.  Without queries ``q`` and ``q_out`` are None."""
        kr, n, _ = _rows(k, self.num_kv_heads, self.head_dim, "k")
        vr, m, _ = _rows(v, self.num_kv_heads, self.head_dim, "v")
        at = _index(slots, 1, "int64", "slots")
        places = _index(positions, 1, "int64", "positions")
        if n != m or slots.shape[0] != n or positions.shape[0] != n:
            raise ValueError(f"{n} rows of k, {m} of v, {positions.shape[0]} positions and "
                             f"{slots.shape[0]} slots")
        if (q is None) != (q_out is None):
            raise ValueError("q and q_out go together")
        q_ref = out_ref = None
        heads = 0
        if q is not None:
            qr, m, heads = _rows(q, None, self.head_dim, "q")
            outr, m_out, _ = _rows(q_out, heads, self.head_dim, "q_out")
            if m != n or m_out != n:
                raise ValueError(f"{n} rows of k, {m} of q and {m_out} of q_out")
            if heads > _MOST:
                raise ValueError(f"{heads} heads are too many")
            q_ref, out_ref = ctypes.byref(qr), ctypes.byref(outr)
        check(lib().pf_kv_write_rotated(self._ref, rotary.handle, q_ref, out_ref, heads,
                                        ctypes.byref(kr), ctypes.byref(vr), places, at, n,
                                        _stream(stream, k)), "write_rotated")

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
        args = self._attend_args(q, out, block_table, seq_lens, query_starts, scale, causal,
                                 window, lse, max_seq_len, max_query_len)
        check(lib().pf_kv_attend(self._ref, ctypes.byref(args),
                                 workspace.handle if workspace is not None else None,
                                 _stream(stream, q)), "attend")

    def attend_shared(self, q, out, block_table, seq_lens, query_starts, group_starts, shared_lens,
                      *, scale: float | None = None, causal: bool = True, window: int = 0,
                      lse=None, max_shared_len: int = 0, max_own_len: int = 0,
                      max_query_len: int = 0, max_seq_len: int = 0,
                      workspace: AttentionWorkspace | None = None,
                      stream: Stream | None = None) -> None:
        """``attend`` of a batch in which groups of sequences share their first tokens, which
        are passed over once for all of a group (pf_kv_attend_shared).

        The sequences of group g are ``group_starts[g]`` to ``group_starts[g + 1]`` (int32);
        the first entries of their rows of ``block_table`` are the same blocks, in which their
        first ``shared_lens[g]`` tokens lie (int32; none of them new).  Others share nothing.
        ``max_shared_len`` and ``max_own_len``, the most tokens that a group shares and that a
        sequence has behind these, are hints that shape the launch.  Sharing takes a
        ``workspace``, a ``max_query_len`` (at most 64 rows a KV head), no ``window``, and
        enough tokens to be worth it, or a ``max_shared_len`` of ``SHARE_ANYWAY`` or more; else
        the call runs as ``attend``, shaped by the shorter of these two hints' sum and
        ``max_seq_len``, if given."""
        starts = _index(group_starts, 1, "int32", "group_starts")
        lens = _index(shared_lens, 1, "int32", "shared_lens")
        groups = shared_lens.shape[0]
        if group_starts.shape[0] != groups + 1:
            raise ValueError(f"{groups} shared lengths and {group_starts.shape[0]} group starts "
                             "(one more than groups)")
        args = self._attend_args(q, out, block_table, seq_lens, query_starts, scale, causal,
                                 window, lse, max_seq_len, max_query_len)
        shared = SharedArgs(starts, lens, min(groups, _MOST),
                            _most("max_shared_len", max_shared_len),
                            _most("max_own_len", max_own_len), 0)
        check(lib().pf_kv_attend_shared(self._ref, ctypes.byref(args), ctypes.byref(shared),
                                        workspace.handle if workspace is not None else None,
                                        _stream(stream, q)), "attend_shared")

    def _attend_args(self, q, out, block_table, seq_lens, query_starts, scale, causal, window, lse,
                     max_seq_len, max_query_len) -> AttendArgs:
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
        return AttendArgs(qr, outr, n, table, block_table.stride()[0], lens, starts, lse_at, heads,
                          seqs, width, min(window, _MOST), causal,
                          1 / math.sqrt(self.head_dim) if scale is None else scale,
                          min(max_seq_len, _MOST), min(max_query_len, _MOST))



class PagedLayers:
    """All layers of a cache, ``PagedKVCache`` of one shape, for what moves blocks and tokens
    within them, each layer alike (pf_kv_layers).  The layers' memory, on ``device``, is borrowed;
    close it after the last call, or graph, that uses it."""

    def __init__(self, caches, device: int = 0):
        self.handle = None
        self.caches = list(caches)
        if not self.caches:
            raise ValueError("no layers")
        h = ctypes.c_void_p()
        pages = (KVPages * len(self.caches))(*[c._pages for c in self.caches])
        check(lib().pf_kv_layers_create(device, pages, len(self.caches), ctypes.byref(h)),
              "pf_kv_layers_create")
        self.handle = h.value

    def copy_blocks(self, from_blocks, to_blocks, stream: Stream | None = None) -> None:
        """Block ``from_blocks[i]`` over block ``to_blocks[i]`` (int32), K and V, in every layer
        (pf_kv_copy_blocks).  A block that does not exist makes its pair padding."""
        src = _index(from_blocks, 1, "int32", "from_blocks")
        dst = _index(to_blocks, 1, "int32", "to_blocks")
        n = from_blocks.shape[0]
        if to_blocks.shape[0] != n:
            raise ValueError(f"{n} blocks to copy and {to_blocks.shape[0]} to copy to")
        check(lib().pf_kv_copy_blocks(self.handle, src, dst, n, _stream(stream, from_blocks)),
              "copy_blocks")

    def fork(self, block_table, seq_lens, parents, new_blocks, out_table,
             stream: Stream | None = None) -> None:
        """Child i of sequence ``parents[i]`` (int32) gets row i of ``out_table``: its parent's
        row of ``block_table``, with ``new_blocks[i]`` (int32) for its next token, into which
        the parent's part-filled block, if any, is copied in every layer (pf_kv_fork).  A
        negative new block leaves the row as the parent's; a parent that does not exist leaves
        the child's row as it was."""
        table = _index(block_table, 2, "int32", "block_table")
        lens = _index(seq_lens, 1, "int32", "seq_lens")
        who = _index(parents, 1, "int32", "parents")
        new = _index(new_blocks, 1, "int32", "new_blocks")
        out = _index(out_table, 2, "int32", "out_table")
        seqs, width = block_table.shape
        n = parents.shape[0]
        if seq_lens.shape[0] != seqs or new_blocks.shape[0] != n or \
                tuple(out_table.shape) != (n, width):
            raise ValueError(f"{seqs} block tables of {width}, {seq_lens.shape[0]} lengths, {n} "
                             f"parents, {new_blocks.shape[0]} new blocks and an out_table of "
                             f"{tuple(out_table.shape)}")
        if max(seqs, width, n) > _MOST:
            raise ValueError("too many sequences")
        args = ForkArgs(table, block_table.stride()[0], lens, who, new, out,
                        out_table.stride()[0], seqs, width, n, 0)
        check(lib().pf_kv_fork(self.handle, ctypes.byref(args), _stream(stream, block_table)),
              "fork")

    def compact(self, block_table, kept, kept_starts, *, first=None, out_table=None,
                out_lens=None, max_kept: int = 0, stream: Stream | None = None) -> None:
        """Moves the kept tokens of sequences together, in every layer (pf_kv_compact).

        Sequence b keeps the tokens at positions ``kept[kept_starts[b]]`` to
        ``kept[kept_starts[b + 1] - 1]`` (int32, ascending); they go to positions ``first[b]``
        (int32; None: 0) and on of its row of ``out_table``, by default in place of what
        ``block_table`` holds there.  In place no token may move up; other blocks that tokens
        go to may not be among those that are read.  ``out_lens`` (int32), if given, receives
        first + kept tokens; ``max_kept``, the most of a sequence, is a hint that shapes the
        launch."""
        table = _index(block_table, 2, "int32", "block_table")
        at = _index(kept, 1, "int32", "kept")
        starts = _index(kept_starts, 1, "int32", "kept_starts")
        seqs, width = block_table.shape
        if out_table is None:
            out_table = block_table
        out = _index(out_table, 2, "int32", "out_table")
        if tuple(out_table.shape) != (seqs, width) or kept_starts.shape[0] != seqs + 1:
            raise ValueError(f"block tables [{seqs}, {width}], an out_table of "
                             f"{tuple(out_table.shape)} and {kept_starts.shape[0]} starts of kept "
                             "tokens (one more than sequences)")
        optional = []
        for x, what in ((first, "first"), (out_lens, "out_lens")):
            optional.append(0 if x is None else _index(x, 1, "int32", what))
            if x is not None and x.shape[0] != seqs:
                raise ValueError(f"{seqs} sequences and {x.shape[0]} of {what}")
        if max(seqs, width) > _MOST:
            raise ValueError("too many sequences")
        args = CompactArgs(table, block_table.stride()[0], out, out_table.stride()[0], at,
                           kept.shape[0], starts, optional[0], optional[1], seqs, width,
                           _most("max_kept", max_kept), 0)
        check(lib().pf_kv_compact(self.handle, ctypes.byref(args), _stream(stream, block_table)),
              "compact")

    def close(self) -> None:
        if self.handle:
            lib().pf_kv_layers_destroy(self.handle)
        self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


__all__ = ["KV_TYPES", "SHARE_ANYWAY", "AttentionWorkspace", "PagedKVCache", "PagedLayers",
           "RotaryPositions", "segment_bytes"]
