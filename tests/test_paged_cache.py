"""The paged-cache operators' argument checks and the oracle's own conversions.  No GPU."""

import ctypes

import numpy as np
import pytest
from hypothesis import given, settings, strategies as st

from oracle import paged as oracle
from pegaflow_amd import _lib
from pegaflow_amd._lib import AttendArgs, KVLayout, KVPages, KVRows, PegaFlowError
from pegaflow_amd.paged_cache import AttentionWorkspace, PagedKVCache, segment_bytes
from pegaflow_amd.transfer import KVCacheRegistration

BASE = 0x10000000  # never dereferenced: refused before any launch


def test_struct_sizes_match_the_header():
    assert ctypes.sizeof(KVPages) == 56 + 24
    assert ctypes.sizeof(KVRows) == 32
    assert ctypes.sizeof(AttendArgs) == 64 + 48 + 32


@pytest.mark.parametrize("bs,heads,dim,kind,want", [
    (16, 8, 128, "bf16", 32768), (16, 12, 64, "fp16", 24576), (16, 8, 128, "e4m3", 16896),
    (16, 8, 128, "int8", 16896), (1, 1, 16, "e4m3", 32), (3, 5, 80, "int8", 1264)])
def test_segment_bytes(bs, heads, dim, kind, want):
    assert segment_bytes(bs, heads, dim, kind) == want
    assert want == oracle.Pages(1, bs, heads, dim, kind).segment


@pytest.mark.parametrize("args", [(0, 8, 128), (16, 0, 128), (16, 8, 0), (16, 8, 24), (16, 8, 272),
                                  (1 << 20, 1 << 20, 128)])
def test_segment_bytes_refusals(args):
    with pytest.raises(PegaFlowError) as e:
        segment_bytes(*args, "e4m3")
    assert e.value.code == _lib.PF_ERR_INVALID_ARGUMENT


def test_unknown_type():
    with pytest.raises(ValueError):
        segment_bytes(16, 8, 128, "int4")
    out = ctypes.c_uint64()
    assert _lib.load().pf_kv_segment_bytes(16, 8, 128, 9, ctypes.byref(out)) == 1
    assert _lib.load().pf_kv_segment_bytes(16, 8, 128, 1, None) == 1


def pages(kind=_lib.KV_BF16, nb=10, bs=16, heads=2, dim=64, order=0, **layout):
    size = 2 if kind in (1, 2) else 1
    bpb = layout.pop("bpb", (bs * heads * dim * size + (4 * bs * heads if size == 1 else 0)))
    kv = layout.pop("kv", nb * bpb)
    segs = layout.pop("segments", 2)
    total = layout.pop("size", nb * bpb + (kv if segs == 2 else 0))
    base = layout.pop("base", BASE)
    assert not layout
    return KVPages(KVLayout(base, total, nb, bpb, bpb * segs, kv, segs), bs, heads, dim, kind, order)


def rows(t=1, ts=128, hs=64, data=BASE):
    return KVRows(data, ts, hs, t, 0)


def refused(rc, text):
    assert rc == _lib.PF_ERR_INVALID_ARGUMENT
    assert text in _lib.last_error(), _lib.last_error()


ROWS_REFUSALS = [
    (dict(pages=None), "null pages"),
    (dict(k=None), "null rows"),
    (dict(pages=pages(kind=7)), "unknown KV type 7"),
    (dict(pages=pages(order=2)), "unknown order"),
    (dict(pages=pages(dim=72)), "head_dim 72"),
    (dict(pages=pages(bpb=2048)), "cannot hold K or V"),
    (dict(pages=pages(segments=1, kv=0)), "cannot hold K or V"),
    (dict(pages=pages(segments=3)), "one or two segments"),
    (dict(pages=pages(nb=0)), "between 1 and 2^31 - 1 blocks"),
    (dict(pages=pages(base=BASE + 8)), "not 16-byte aligned"),
    (dict(pages=pages(bpb=4104)), "not 16-byte aligned"),
    (dict(pages=pages(kv=4096)), "K and V segments of the pages overlap"),
    (dict(pages=pages(size=81919)), "exceed the registered memory"),
    (dict(pages=pages(kind=_lib.KV_FP16)), "16-bit pages hold the rows' own type"),
    (dict(k=rows(t=2)), "differ in type"),
    (dict(k=rows(t=3), v=rows(t=3, data=BASE + 4096), pages=pages(kind=3)), "rows are bf16 or fp16"),
    (dict(k=rows(data=BASE + 1)), "unaligned address"),
    (dict(k=rows(ts=1 << 62)), "strides overflow"),
    (dict(slots=BASE + 4), "unaligned address"),
    (dict(n=1 << 31), "too many rows"),
    (dict(), "not inside one device or pinned allocation"),
]


@pytest.mark.parametrize("change,text", ROWS_REFUSALS, ids=[t for _, t in ROWS_REFUSALS])
@pytest.mark.parametrize("op", ["pf_kv_write", "pf_kv_read"])
def test_write_and_read_refusals(op, change, text):
    a = dict(pages=pages(), k=rows(), v=rows(data=BASE + (1 << 20)), slots=BASE, n=5)
    a.update(change)
    ref = [ctypes.byref(x) if x is not None else None for x in (a["pages"], a["k"], a["v"])]
    refused(getattr(_lib.load(), op)(*ref, a["slots"], a["n"], None), text)


@pytest.mark.parametrize("r", [rows(ts=64, hs=64), rows(ts=128, hs=32), rows(ts=0, hs=0),
                               rows(ts=64, hs=4 * 64)])
def test_overlapping_outputs_are_refused(r):
    p = pages()
    args = (ctypes.byref(p), ctypes.byref(r), ctypes.byref(rows(data=BASE + (1 << 20))))
    refused(_lib.load().pf_kv_read(*args, BASE, 5, None), "rows overlap")
    # The same strides are fine to read from.
    refused(_lib.load().pf_kv_write(*args, BASE, 5, None), "not inside one device")


def test_same_output_for_k_and_v_is_refused():
    p, r = pages(), rows()
    refused(_lib.load().pf_kv_read(ctypes.byref(p), ctypes.byref(r), ctypes.byref(r), BASE, 5, None),
            "K and V rows overlap")


def attend_args(**change):
    a = dict(q=rows(ts=256), out=rows(ts=256), num_rows=5, block_table=BASE, table_stride=4,
             seq_lens=BASE, query_starts=BASE, lse=0, num_q_heads=4, num_seqs=2, table_width=4,
             window=0, causal=1, scale=0.125, max_seq_len=0, max_query_len=0)
    a.update(change)
    return AttendArgs(*a.values())


ATTEND_REFUSALS = [
    (dict(q=rows(t=3)), "bf16 or fp16"),
    (dict(q=rows(t=2)), "of one type"),
    (dict(q=rows(t=2), out=rows(t=2)), "16-bit pages hold the rows' own type"),
    (dict(num_q_heads=3), "no multiple of 2 KV heads"),
    (dict(num_q_heads=0), "no multiple of 2 KV heads"),
    (dict(window=5, causal=0), "a window needs causal"),
    (dict(scale=float("nan")), "not finite"),
    (dict(scale=float("inf")), "not finite"),
    (dict(scale=-3e38), "not finite"),
    (dict(table_width=0), "no entries"),
    (dict(table_width=(1 << 27) - 4095), "2^31 - 65536 tokens"),
    (dict(table_stride=3), "rows of the block table overlap"),
    (dict(num_rows=1 << 30), "too many rows"),
    (dict(out=rows(ts=128)), "out: rows overlap"),
    (dict(block_table=BASE + 2), "block table: unaligned"),
    (dict(seq_lens=BASE + 2), "seq_lens: unaligned"),
    (dict(query_starts=BASE + 1), "query_starts: unaligned"),
    (dict(lse=BASE + 2), "lse: unaligned"),
    (dict(table_stride=1 << 60, num_seqs=1 << 20), "strides overflow"),
    (dict(), "not inside one device or pinned allocation"),
]


@pytest.mark.parametrize("change,text", ATTEND_REFUSALS, ids=[t for _, t in ATTEND_REFUSALS])
def test_attend_refusals(change, text):
    p, a = pages(), attend_args(**change)
    refused(_lib.load().pf_kv_attend(ctypes.byref(p), ctypes.byref(a), None, None), text)
    refused(_lib.load().pf_kv_attend(ctypes.byref(p), None, None, None), "null arguments")


def test_empty_calls_do_nothing():
    lib, p = _lib.load(), pages()
    r = rows(data=0)
    for op in (lib.pf_kv_write, lib.pf_kv_read):
        v = rows(data=BASE)
        assert op(ctypes.byref(p), ctypes.byref(r), ctypes.byref(v), 0, 0, None) == _lib.PF_OK
    for change in (dict(num_rows=0), dict(num_seqs=0)):
        a = attend_args(**change)
        assert lib.pf_kv_attend(ctypes.byref(p), ctypes.byref(a), None, None) == _lib.PF_OK


def test_workspace_refusals():
    out = ctypes.c_void_p()
    assert _lib.load().pf_attend_workspace_create(0, 0, ctypes.byref(out)) == _lib.PF_ERR_ZERO_SIZE
    assert _lib.load().pf_attend_workspace_create(0, 64, None) == _lib.PF_ERR_INVALID_ARGUMENT
    with pytest.raises(PegaFlowError):
        AttentionWorkspace(device=-1)
    assert _lib.load().pf_attend_workspace_destroy(None) == _lib.PF_OK


class Tensor:
    """A tensor's face without memory."""

    def __init__(self, shape, dtype="torch.bfloat16", stride=None):
        self.shape, self.dtype = shape, dtype
        if stride is None:
            stride = tuple(int(np.prod(shape[i + 1:])) for i in range(len(shape)))
        self._stride = stride

    def stride(self):
        return self._stride

    def data_ptr(self):
        return BASE


def cache(**kw):
    seg = segment_bytes(16, 2, 64, "bf16")
    reg = KVCacheRegistration.create(BASE, 20 * seg, 10, seg, 10 * seg, 2)
    return PagedKVCache(reg, 16, 2, 64, "bf16", **kw)


def test_python_checks():
    c = cache()
    k, slots = Tensor((5, 2, 64)), Tensor((5,), "torch.int64")
    for bad in (Tensor((5, 3, 64)), Tensor((5, 2, 128)), Tensor((5, 128)),
                Tensor((5, 2, 64), "torch.float32"), Tensor((5, 2, 64), stride=(256, 128, 2)),
                Tensor((4, 2, 64))):
        with pytest.raises(ValueError):
            c.write(bad, k, slots)
        with pytest.raises(ValueError):
            c.read(slots, k, bad)
    for bad in (Tensor((5,), "torch.int32"), Tensor((6,), "torch.int64"),
                Tensor((5, 1), "torch.int64"), Tensor((5,), "torch.int64", (2,))):
        with pytest.raises(ValueError):
            c.write(k, k, bad)
    good = dict(q=Tensor((5, 4, 64)), out=Tensor((5, 4, 64)),
                block_table=Tensor((2, 4), "torch.int32"), seq_lens=Tensor((2,), "torch.int32"),
                query_starts=Tensor((3,), "torch.int32"))
    for change in (dict(q=Tensor((5, 4, 32))), dict(out=Tensor((5, 2, 64))),
                   dict(out=Tensor((6, 4, 64))), dict(block_table=Tensor((2, 4), "torch.int64")),
                   dict(seq_lens=Tensor((3,), "torch.int32")), dict(window=-1),
                   dict(query_starts=Tensor((2,), "torch.int32")), dict(max_seq_len=-1),
                   dict(lse=Tensor((5, 4))), dict(lse=Tensor((5, 2), "torch.float32")),
                   dict(lse=Tensor((5, 4), "torch.float32", (8, 1)))):
        with pytest.raises(ValueError):
            c.attend(**{**good, **change})
    with pytest.raises(PegaFlowError):  # everything in order but the memory
        c.attend(**good)
    seg = segment_bytes(16, 2, 64, "e4m3")
    reg = KVCacheRegistration.create(BASE, 20 * seg, 10, seg, 10 * seg, 2)
    with pytest.raises(ValueError):
        PagedKVCache(reg, 16, 2, 64, "bf16")


# -- the oracle's conversions ---------------------------------------------------------
@settings(max_examples=200, deadline=None)
@given(st.floats(-500, 500, width=32))
def test_oracle_e4m3_rounds_to_nearest_even(x):
    code = int(oracle.to_e4m3(np.float32(x)))
    got = oracle.E4M3[code]
    finite = oracle.E4M3[np.isfinite(oracle.E4M3)]
    assert abs(got - x) == np.abs(finite - np.float64(np.float32(x))).min()
    if (np.abs(finite - x) == abs(got - x)).sum() > 1 and got != 0:
        assert code % 2 == 0


def test_oracle_bf16_bits_match_torch():
    torch = pytest.importorskip("torch")
    x = np.random.default_rng(0).standard_normal(1000).astype(np.float32)
    x[:4] = [np.inf, -np.inf, 3.4e38, 1e-40]
    want = torch.from_numpy(x).to(torch.bfloat16).view(torch.int16).numpy().view(np.uint16)
    assert np.array_equal(oracle.to_bits(x, "bf16"), want)
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(codes, oracle.E4M3.astype(np.float32), equal_nan=True)
    y = x[4:] * 100
    y = y[np.abs(y) < 448]
    want = torch.from_numpy(y).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(oracle.to_e4m3(y), want)


@pytest.mark.parametrize("d", [1, 2, 3, 5, 7, 8, 12, 16, 17, 48, 64, 100, 1000, 65537])
def test_division_by_multiplication(d):
    """The kernels' token / block_size, from its multiplier and shift, at the edges of every
    quotient near powers of two and 2^31 - 1."""
    s = 0
    while 1 << s < d:
        s += 1
    mul = ((1 << (31 + s)) + d - 1) // d
    assert mul < 1 << 32
    tops = [1 << i for i in range(31)] + [(1 << 31) - 1]
    for top in tops:
        for x in (top - 1, top, top // d * d, max(0, top // d * d - 1)):
            assert x * mul >> (31 + s) == x // d
