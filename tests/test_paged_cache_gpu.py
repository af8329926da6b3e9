"""The paged-cache operators on the GPU against their definitions (oracle/paged.py): writes
and reads bit by bit, attention within the bound that its roundings allow."""

import ctypes
import math

import numpy as np
import pytest

from oracle import paged as oracle
from pegaflow_amd.engine import PegaEngine
from pegaflow_amd.load_state import PyLoadState
from pegaflow_amd.paged_cache import AttentionWorkspace, PagedKVCache, segment_bytes
from pegaflow_amd.runtime import DeviceArray, DeviceBuffer, Stream, synchronize
from pegaflow_amd.transfer import KVCacheRegistration

pytestmark = pytest.mark.gpu

NAN16 = {"bf16": 0x7fc1, "fp16": 0x7e01}
INF16 = {"bf16": 0x7f80, "fp16": 0x7c00}


class DevicePages:
    """oracle.Pages and the same bytes on the device."""

    def __init__(self, pages):
        self.host = pages
        self.buf = DeviceBuffer(pages.bytes.nbytes)
        self.upload()
        seg, nb = pages.segment, pages.num_blocks
        if pages.blocks_first:
            reg = KVCacheRegistration.create(self.buf.ptr, self.buf.nbytes, nb, 2 * seg, 0, 1)
        else:
            reg = KVCacheRegistration.create(self.buf.ptr, self.buf.nbytes, nb, seg, nb * seg, 2)
        self.cache = PagedKVCache(reg, pages.block_size, pages.heads, pages.dim, pages.kind,
                                  head_major=pages.head_major)

    def upload(self):
        self.buf.upload(self.host.bytes)

    def bytes(self):
        return self.buf.download().reshape(self.host.bytes.shape)


def device_rows(bits, strides="contiguous", rows="bf16", offset=0):
    """A DeviceArray of uint16 bits [n, heads, dim] in a buffer of other values, and that
    buffer's host copy."""
    n, heads, dim = bits.shape
    if strides == "contiguous":
        st = (heads * dim, dim, 1)
    elif strides == "fused":  # a slice of a wider projection
        st = (3 * heads * dim + 8, dim, 1)
    elif strides == "heads_first":
        st = (dim, max(n, 1) * dim, 1)
    else:  # odd: rows that no 16-byte load can take
        st = (heads * (dim + 1) + 2, dim + 1, 1)
    size = offset + ((n - 1) * st[0] + (heads - 1) * st[1] + dim if n else 1)
    flat = np.full(size, 0x4242, np.uint16)
    view = np.lib.stride_tricks.as_strided(flat[offset:], (n, heads, dim), [2 * s for s in st])
    view[:] = bits
    buf = DeviceBuffer(2 * size)
    buf.upload(flat)
    return DeviceArray((n, heads, dim), rows, buf, 2 * offset, st), flat, view


def device_array(x, dtype):
    a = DeviceArray(x.shape, dtype)
    a.upload(np.ascontiguousarray(x))
    return a


def values(rng, shape, rows):
    x = rng.standard_normal(shape) * np.exp(rng.standard_normal(shape[-1]) * 0.5)
    return oracle.to_bits(x.astype(np.float32), rows)


# kind, rows, heads, dim, block size, head major
FORMS = [("bf16", "bf16", 8, 128, 16, False), ("fp16", "fp16", 12, 64, 16, False),
         ("e4m3", "bf16", 8, 128, 16, False), ("int8", "bf16", 8, 128, 16, True),
         ("e4m3", "fp16", 3, 80, 8, True), ("int8", "fp16", 5, 96, 7, False),
         ("e4m3", "bf16", 1, 256, 64, False), ("int8", "bf16", 2, 192, 1, True),
         ("bf16", "bf16", 1, 16, 3, True), ("e4m3", "fp16", 1, 16, 1, False)]


@pytest.mark.parametrize("n", [0, 1, 2, 17, 130])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_write_then_read(gpu, form, n):
    """Every byte of the pages after a write, and every row read back, padding included."""
    kind, rows, heads, dim, bs, head_major = form
    rng = np.random.default_rng(n + dim)
    nb = n // bs * 2 + 5
    pages = oracle.Pages(nb, bs, heads, dim, kind, head_major, rows, pad=16 * (n % 2),
                         blocks_first=n % 2 == 1 and bs % 2 == 0)
    pages.bytes[:] = rng.integers(0, 256, pages.bytes.shape, np.uint8)
    dev = DevicePages(pages)
    strides = ["contiguous", "fused", "heads_first", "odd"][(n + heads) % 4]
    k, v = values(rng, (n, heads, dim), rows), values(rng, (n, heads, dim), rows)
    if n > 4:  # zeros, infinities, NaN, subnormal rows, one value, the largest
        k[0] = 0
        k[1, 0, 3] = INF16[rows]
        v[1, :, dim - 1] = NAN16[rows] | 0x8000
        k[2] = rng.integers(0, 3, (heads, dim))
        v[3] = 0
        v[3, :, 5] = 1
        k[4] = INF16[rows] - 1
        k[3] = 0x8000  # -0
    slots = rng.permutation(nb * bs)[:n].astype(np.int64)
    if n > 10:
        slots[5], slots[6], slots[7], slots[8] = -1, nb * bs, -(1 << 40), 1 << 40
    at = device_array(slots, "int64")
    kd, _, _ = device_rows(k, strides, rows, offset=8 if strides != "odd" else 1)
    vd, _, _ = device_rows(v, strides, rows)
    dev.cache.write(kd, vd, at)
    synchronize()
    pages.set(slots, k, v)
    got = dev.bytes()
    if kind in oracle.LARGEST:  # a NaN scale: any NaN
        mine = oracle.Pages(nb, bs, heads, dim, kind, head_major, rows, pages.segment - oracle.Pages(
            nb, bs, heads, dim, kind).segment, pages.blocks_first)
        mine.bytes = got
        a, b = mine.scales(), pages.scales()
        assert np.array_equal(a, b, equal_nan=True)
        assert np.array_equal(mine.values(), pages.values())
        written = slots[(slots >= 0) & (slots < nb * bs)]
        pages.scales()[:, written // bs, written % bs] = a[:, written // bs, written % bs]
    assert np.array_equal(got, pages.bytes)
    # Back, into rows that hold something else.
    for order in (np.arange(n), rng.permutation(n)):
        ko, flat_k, view_k = device_rows(np.zeros_like(k), strides, rows)
        vo, flat_v, view_v = device_rows(np.zeros_like(v), strides, rows, offset=3)
        dev.cache.read(device_array(slots[order], "int64"), ko, vo)
        synchronize()
        keep = (slots[order] >= 0) & (slots[order] < nb * bs)
        want = pages.get(np.where(keep, slots[order], 0))[1]
        for flat, view, x, o in ((flat_k, view_k, want[0], ko), (flat_v, view_v, want[1], vo)):
            bits = oracle.to_bits(x, rows) if kind in oracle.LARGEST else x
            if kind not in oracle.LARGEST:
                raw = pages.values()[0 if o is ko else 1]
                s = np.where(keep, slots[order], 0)
                bits = raw[s // bs, s % bs]
            nan = np.isnan(x)
            view[keep] = bits[keep]
            back = o.buffer.download().view(np.uint16)
            got_view = np.lib.stride_tricks.as_strided(
                back[o._offset // 2:], view.shape, view.strides)
            if kind in oracle.LARGEST:
                got_x = oracle.from_bits(got_view, rows)
                assert np.isnan(got_x[keep][nan[keep]]).all()
                view[keep[:, None, None] & nan] = got_view[keep[:, None, None] & nan]
            assert np.array_equal(back, flat)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("rows", ["bf16", "fp16"])
def test_codes_at_the_ties(gpu, kind, rows):
    """Rows whose quotients lie on and next to the borders between codes: a largest value that
    fixes the scale, and every 16-bit value below it in turn."""
    bits = np.arange(INF16[rows], dtype=np.uint16)
    x = oracle.from_bits(bits, rows)
    n = 600
    rng = np.random.default_rng(7)
    k = np.zeros((n, 1, 256), np.uint16)
    for i in range(n):
        top = int(rng.integers(1, INF16[rows])) if i > 3 else (1, 2, 0x80, INF16[rows] - 1)[i]
        low = max(0, top - 0x600) if i % 2 else 0
        k[i, 0] = rng.integers(low, top + 1, 256)
        k[i, 0, i % 256] = top
    k[:, :, ::3] |= 0x8000
    assert len(x)
    pages = oracle.Pages(n, 1, 1, 256, kind, rows=rows)
    dev = DevicePages(pages)
    slots = np.arange(n, dtype=np.int64)
    kd = device_rows(k, rows=rows)[0]
    vd = device_rows(k[::-1].copy(), rows=rows)[0]
    dev.cache.write(kd, vd, device_array(slots, "int64"))
    synchronize()
    pages.set(slots, k, k[::-1])
    assert np.array_equal(dev.bytes(), pages.bytes)


class Batch:
    """A ragged batch over pages whose other blocks, and tokens past each end, hold NaN."""

    def __init__(self, new, cached, form, group, seed=0, holes=False, strides="fused",
                 sharp=1.0, table_pad=1):
        self.kind, self.rows, heads, dim, bs, head_major = form
        rng = np.random.default_rng(seed)
        self.new, self.cached = list(new), list(cached)
        lens = np.array([max(a + b, 0) for a, b in zip(new, cached)])
        used = [-(-int(n) // bs) for n in lens]
        nb = sum(used) + 4
        pages = oracle.Pages(nb, bs, heads, dim, self.kind, head_major, self.rows)
        if self.kind in oracle.LARGEST:
            pages.values()[:] = 0x7f if self.kind == "e4m3" else 0x55
            pages.scales()[:] = np.nan
        else:
            pages.values()[:] = NAN16[self.rows]
        order = rng.permutation(nb).astype(np.int32)
        self.table = np.full((len(lens), max(used + [0]) + table_pad), -1, np.int32)
        at = 0
        for i, (n, u) in enumerate(zip(lens, used)):
            self.table[i, :u] = order[at:at + u]
            at += u
            t = np.arange(n)
            slots = self.table[i][t // bs].astype(np.int64) * bs + t % bs
            pages.set(slots, values(rng, (n, heads, dim), self.rows),
                      values(rng, (n, heads, dim), self.rows))
        # Past a sequence's blocks the table names some block (another's, or none).
        for i, u in enumerate(used):
            self.table[i, u:] = (order[0], -7, nb, 2 ** 31 - 1)[i % 4]
        if holes:
            for i, u in enumerate(used):
                if u > 2:
                    self.table[i, rng.integers(0, u, max(1, u // 3))] = (-1, nb, -2 ** 31)[i % 3]
        self.pages, self.dev = pages, DevicePages(pages)
        self.lens = lens.astype(np.int32)
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        total = int(self.starts[-1])
        q = rng.standard_normal((total, heads * group, dim)) * sharp
        self.q = oracle.to_bits(q.astype(np.float32), self.rows)
        self.strides, self.group = strides, group
        self.scale = dim ** -0.5

    def run(self, tail=0, front=0, workspace=None, lse=True, stream=None, hints=True, **kw):
        """(out bits, lse) of one call, after checking that rows outside the sequences and
        the values between the rows stay."""
        n, heads, dim = self.q.shape
        bits = np.concatenate([np.full((front, heads, dim), 0x1111, np.uint16), self.q,
                               np.full((tail, heads, dim), 0x1111, np.uint16)])
        q = device_rows(bits, self.strides, self.rows, offset=8)[0]
        out, flat, view = device_rows(np.full_like(bits, 0x5a5a), self.strides, self.rows)
        l = device_array(np.full(bits.shape[:2], 77, np.float32), "fp32") if lse else None
        if hints:
            kw.setdefault("max_seq_len", int(self.lens.max()) if len(self.lens) else 0)
            kw.setdefault("max_query_len", max(self.new) if self.new else 0)
        self.dev.cache.attend(q, out, device_array(self.table, "int32"),
                              device_array(self.lens, "int32"),
                              device_array(self.starts + front, "int32"), lse=l,
                              workspace=workspace, stream=stream, **kw)
        synchronize()
        back = out.buffer.download().view(np.uint16)
        got = np.lib.stride_tricks.as_strided(back, view.shape, view.strides).copy()
        view[front:front + n] = got[front:front + n]
        assert np.array_equal(back, flat)
        if not lse:
            return got[front:front + n], None
        got_lse = l.download().view(np.float32).reshape(bits.shape[:2])
        assert (got_lse[:front] == 77).all() and (got_lse[front + n:] == 77).all()
        return got[front:front + n], got_lse[front:front + n]

    def check(self, got, lse, causal=True, window=0, scale=None, every=1, **kw):
        out, want_lse, bound, lse_bound = (x[::every] for x in oracle.attend(
            self.pages, self.q, self.rows, self.table, self.lens, self.starts,
            scale or self.scale, causal, window, every=every,
            fine=np.flatnonzero(np.diff(self.starts) * self.group <= 16)))
        x = oracle.from_bits(got, self.rows).astype(np.float64)[::every]
        lse = None if lse is None else lse[::every]
        assert np.array_equal(np.isnan(x), np.isnan(out))
        fine = np.isfinite(out)
        off = np.abs(x - out)[fine] / np.maximum(bound[fine], 1e-300)
        assert off.size == 0 or off.max() <= 1, off.max()
        if lse is not None:
            gone = np.isneginf(want_lse)
            assert np.array_equal(np.isneginf(lse), gone)
            assert (x[gone] == 0).all()
            keep = np.isfinite(want_lse)
            assert (np.abs(lse - want_lse)[keep] <= lse_bound[keep]).all()
        return off.max() if off.size else 0.0


@pytest.fixture(scope="module")
def workspace(gpu):
    w = AttentionWorkspace()
    yield w
    w.close()


LLAMA = ("bf16", "bf16", 8, 128, 16, False)
# form, group
ATTEND_FORMS = [(f, g) for f, g in zip(FORMS, (4, 1, 4, 4, 5, 1, 7, 3, 2, 16))]
ATTEND_FORMS += [(("bf16", "bf16", 1, 128, 16, False), 8), (("fp16", "fp16", 2, 80, 32, False), 3),
                 (("bf16", "bf16", 2, 192, 16, True), 2), (("fp16", "fp16", 1, 256, 5, False), 2),
                 (("bf16", "bf16", 1, 96, 16, False), 33), (("e4m3", "bf16", 2, 64, 16, False), 1),
                 (("int8", "fp16", 1, 256, 16, False), 8)]


@pytest.mark.parametrize("form,group", ATTEND_FORMS, ids=str)
def test_single_tokens(gpu, workspace, form, group):
    """One new token each, behind nothing, one token, and lengths about a page and a tile."""
    cached = [0, 1, 15, 16, 31, 63, 64, 65, 130, 300]
    b = Batch([1] * len(cached), cached, form, group, seed=1)
    for w in (None, workspace):
        b.check(*b.run(workspace=w, tail=2))


@pytest.mark.parametrize("form,group", ATTEND_FORMS, ids=str)
def test_chunks(gpu, workspace, form, group):
    """Chunks of odd lengths and single tokens in one batch, in any order."""
    b = Batch([7, 1, 70, 33, 1, 2], [90, 5, 0, 131, 64, 0], form, group, seed=2)
    for w in (None, workspace):
        b.check(*b.run(workspace=w, front=1, tail=3))
    b.check(*b.run(workspace=workspace, hints=False))


@pytest.mark.parametrize("form,group", [(LLAMA, 4), (FORMS[2], 4), (FORMS[1], 1), (FORMS[3], 4)],
                         ids=str)
@pytest.mark.parametrize("new,cached", [((1,), (5000,)), ((1, 1, 1), (2049, 0, 4095)),
                                        ((3,), (2600,)), ((40,), (2100,)),
                                        ((1, 9, 1), (1500, 1200, 3))], ids=str)
def test_long_sequences_are_split_and_joined(gpu, workspace, form, group, new, cached):
    """Few rows over thousands of tokens, with a workspace of any size and without one."""
    b = Batch(new, cached, form, group, seed=3)
    b.check(*b.run(workspace=workspace))
    first = b.run(workspace=workspace)
    for _ in range(3):  # the same bits every time
        again = b.run(workspace=workspace)
        assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])
    small = AttentionWorkspace(70_000)
    b.check(*b.run(workspace=small))
    small.close()
    b.check(*b.run(workspace=None))
    # Bounds far too high, and a length hint that says too little, change the launch alone.
    b.check(*b.run(workspace=workspace, max_seq_len=1 << 20, max_query_len=1 << 20))
    b.check(*b.run(workspace=workspace, max_seq_len=1))


@pytest.mark.parametrize("form,group,new,cached", [
    (("bf16", "bf16", 64, 16, 16, False), 1, (1030,), (2300,)),
    (("int8", "fp16", 32, 208, 16, True), 2, (70, 500, 1), (2900, 2500, 2600))], ids=str)
def test_tiles_left_over_are_split(gpu, workspace, form, group, new, cached):
    """A few tiles of rows more than the chip holds at once: the last ones in shares, and
    whole without a workspace."""
    b = Batch(new, cached, form, group, seed=17)
    for w in (workspace, None):
        b.check(*b.run(workspace=w, tail=1), every=37)


@pytest.mark.parametrize("form,group,new,cached", [
    (("bf16", "bf16", 64, 16, 16, False), 1, (1030,), (2300,)),
    (("int8", "fp16", 32, 208, 16, True), 2, (70, 500, 1), (2900, 2500, 2600))], ids=str)
def test_tiles_left_over_are_split(gpu, workspace, form, group, new, cached):
    """A few tiles of rows more than the chip holds at once: the last ones in shares, and
    whole without a workspace."""
    b = Batch(new, cached, form, group, seed=17)
    for w in (workspace, None):
        b.check(*b.run(workspace=w, tail=1), every=37)


@pytest.mark.parametrize("options", [{}, {"window": 3990}, {"causal": False}], ids=str)
@pytest.mark.parametrize("form,group", [
    (LLAMA, 4), (FORMS[2], 4), (FORMS[4], 5), (FORMS[5], 1), (FORMS[1], 1), (FORMS[8], 2),
    (("e4m3", "bf16", 2, 64, 16, False), 1), (("int8", "fp16", 2, 48, 16, False), 3)], ids=str)
def test_wide_tiles(gpu, workspace, form, group, options):
    """Many rows of a long sequence, in tiles of 256: full ones and one of a few rows."""
    b = Batch([530 // group + 1], [4000], form, group, seed=18, holes=True)
    for w in (workspace, None):
        b.check(*b.run(workspace=w, tail=2, **options), every=23, **options)


def test_wide_tiles_of_several_sequences(gpu, workspace):
    """Wide tiles beside a single token and a short chunk, the last ones in shares."""
    form = ("fp16", "fp16", 64, 16, 16, False)
    b = Batch([1500, 1, 700, 9], [4200, 3000, 2900, 2800], form, 1, seed=19)
    for w in (workspace, None):
        b.check(*b.run(workspace=w, front=1), every=41)
    b = Batch([1500, 620], [4200, 2900], form, 1, seed=20)
    bs = b.pages.block_size
    for t, kv, bad in ((4300, 1, NAN16), (5000, 1, INF16), (5600, 0, NAN16)):
        b.pages.values()[kv, b.table[0][t // bs], t % bs, :, 3] = bad["fp16"]
    b.dev.upload()
    b.check(*b.run(workspace=workspace), every=41)


@pytest.mark.parametrize("window", [1, 2, 16, 17, 100, 1 << 31])
@pytest.mark.parametrize("form,group", [(LLAMA, 4), (FORMS[4], 5)], ids=str)
def test_window(gpu, workspace, form, group, window):
    b = Batch([50, 1, 1, 9], [40, 200, 3, 700], form, group, seed=4)
    w = min(window, 1 << 30)
    b.check(*b.run(workspace=workspace, window=w), window=w)


@pytest.mark.parametrize("form,group", [(LLAMA, 4), (FORMS[3], 4)], ids=str)
def test_not_causal(gpu, workspace, form, group):
    b = Batch([50, 1, 130], [40, 200, 0], form, group, seed=5)
    b.check(*b.run(workspace=workspace, causal=False), causal=False)


@pytest.mark.parametrize("form,group", [(LLAMA, 4), (FORMS[2], 4), (FORMS[5], 1)], ids=str)
def test_rows_that_attend_nothing(gpu, workspace, form, group):
    """Sequences shorter than their new rows, of no tokens, of no rows, and missing blocks."""
    b = Batch([5, 3, 0, 1, 4], [-3, -3, 40, -1, 0], form, group, seed=6)
    b.lens[3] = -5
    b.check(*b.run(workspace=workspace))
    b = Batch([3, 1, 40], [100, 90, 60], form, group, seed=7, holes=True)
    b.check(*b.run(workspace=workspace))
    b.table[:] = -1
    got, lse = b.run(workspace=workspace)
    assert not got.any() and np.isneginf(lse).all()
    b = Batch([], [], form, group, seed=8)
    b.run(tail=4, workspace=workspace)


@pytest.mark.parametrize("form,group", [(LLAMA, 4), (FORMS[2], 4), (FORMS[1], 1), (FORMS[5], 1)],
                         ids=str)
@pytest.mark.parametrize("new,cached", [((1, 1), (100, 20)), ((100, 30), (0, 50)),
                                        ((1,), (3000,))], ids=str)
def test_values_that_are_not_finite(gpu, workspace, form, group, new, cached):
    """A NaN or infinity in K or V reaches the rows that attend its token, and no other."""
    b = Batch(new, cached, form, group, seed=9)
    bs = b.pages.block_size
    length = int(b.lens[0])
    for i, (kv, bad) in enumerate(((1, NAN16), (0, NAN16), (1, INF16))):
        t = length - 1 - i if new[0] == 1 else (60, 71, 90)[i]
        block, off = b.table[0][t // bs], t % bs
        if b.kind in oracle.LARGEST:
            b.pages.scales()[kv, block, off, 0] = np.nan if bad is NAN16 else np.inf
        else:
            b.pages.values()[kv, block, off, 0, 3] = bad[b.rows]
    b.dev.upload()
    b.check(*b.run(workspace=workspace))


@pytest.mark.parametrize("sizes", ["growing", "falling", "mixed", "late"])
@pytest.mark.parametrize("form,group", [(FORMS[4], 5), (FORMS[5], 1), (FORMS[2], 4),
                                        (("int8", "fp16", 2, 128, 16, False), 4)], ids=str)
@pytest.mark.parametrize("new,cached", [((1, 1), (2000, 40)), ((150, 30, 1), (40, 300, 7))],
                         ids=str)
def test_scales_of_all_sizes(gpu, workspace, form, group, sizes, new, cached):
    """V's scales over 27 powers of two: rows that attend only small ones keep their precision
    beside rows that attend large ones."""
    b = Batch(new, cached, form, group, seed=14)
    bs, rng = b.pages.block_size, np.random.default_rng(15)
    for i, n in enumerate(b.lens):
        t = np.arange(n)
        size = {"growing": -20 + 27 * t / n, "falling": 7 - 27 * t / n,
                "mixed": rng.uniform(-20, 7, n), "late": np.where(t < n - 9, -12, 7)}[sizes]
        scale = np.exp2(size)[:, None] * rng.uniform(0.5, 1, (n, b.pages.heads))
        scale[(t % 50 < 3) & (t % 100 < 50)] = 0
        b.pages.scales()[1, b.table[i][t // bs], t % bs] = scale
    b.dev.upload()
    for w in (None, workspace):
        b.check(*b.run(workspace=w))


@pytest.mark.parametrize("form,group", [(LLAMA, 4), (FORMS[2], 4), (FORMS[1], 1)], ids=str)
def test_sharp_scores(gpu, workspace, form, group):
    """Scores of hundreds, whose largest comes late: the running maximum moves far."""
    b = Batch([1, 90, 1], [1200, 200, 77], form, group, seed=10, sharp=20.0)
    b.check(*b.run(workspace=workspace))
    b.check(*b.run(workspace=workspace, scale=-3.0 * b.scale), scale=-3.0 * b.scale)
    b.scale = 0.0
    got, lse = b.run(workspace=workspace, scale=0.0)
    out, want, bound, lse_bound = oracle.attend(
        b.pages, b.q, b.rows, b.table, b.lens, b.starts, 0.0, weights="bf16")
    assert (np.abs(oracle.from_bits(got, b.rows) - out) <= bound).all()
    assert (np.abs(lse - want) <= lse_bound).all()


@pytest.mark.parametrize("strides", ["contiguous", "heads_first", "odd"])
@pytest.mark.parametrize("new,cached", [((1, 1), (300, 20)), ((90, 3), (41, 8))], ids=str)
def test_strides(gpu, workspace, strides, new, cached):
    for form, group in ((LLAMA, 4), (FORMS[5], 1)):
        b = Batch(new, cached, form, group, seed=11, strides=strides)
        b.check(*b.run(workspace=workspace, tail=1))


def test_lengths_beyond_the_table_are_cut(gpu, workspace):
    b = Batch([1, 20], [63, 44], LLAMA, 4, seed=12, table_pad=0)
    want = b.run(workspace=workspace)
    b.lens += 1 << 20
    b.check(*b.run(workspace=workspace, max_seq_len=64))
    b.lens[:] = 2 ** 31 - 1
    got = b.run(workspace=workspace)
    assert np.array_equal(got[0], want[0])


def test_query_starts_are_bounded(gpu, workspace):
    """Starts outside the rows, or out of order, read and write no row outside the call's."""
    b = Batch([5, 6, 7], [20, 30, 40], LLAMA, 4, seed=13)
    n = len(b.q)
    for starts in ([-9, 5, 11, 4000], [2 ** 31 - 1, -2 ** 31, 0, 18], [18, 11, 5, 0]):
        # The values between the rows of a wider buffer, and 40 rows behind them.
        q = device_rows(b.q, "fused")[0]
        out, flat, view = device_rows(np.full((n + 40,) + b.q.shape[1:], 0x5a5a, np.uint16), "fused")
        rows = DeviceArray(b.q.shape, "bf16", out.buffer, out._offset, out.stride())
        b.dev.cache.attend(q, rows, device_array(b.table, "int32"), device_array(b.lens, "int32"),
                           device_array(np.array(starts, np.int32), "int32"), workspace=workspace)
        synchronize()
        back = out.buffer.download().view(np.uint16)
        got = np.lib.stride_tricks.as_strided(back, view.shape, view.strides)
        view[:n] = got[:n]
        assert np.array_equal(back, flat)


def test_rows_beyond_the_longest_query(gpu, workspace):
    """max_query_len bounds a sequence's rows: those beyond stay, or are attended."""
    b = Batch([9, 1, 3], [700, 20, 30], LLAMA, 4, seed=23)
    got, _ = b.run(workspace=workspace, max_query_len=1)
    want, _ = b.run(workspace=workspace)
    kept = (got == 0x5a5a).all((1, 2))
    assert kept.sum() and not kept[[0, 9, 10]].any()
    b.check(np.where(kept[:, None, None], want, got), None)


@pytest.mark.parametrize("first_block", [0, 1])
def test_offsets_past_32_bits(gpu, workspace, first_block):
    """Pages beyond 4 GiB: write, read and attend in the last blocks of a 9 GiB layer."""
    bs, heads, dim, seg = 16, 8, 128, 32768
    nb = (9 << 30) // (2 * seg)
    buf = DeviceBuffer(2 * nb * seg)
    reg = KVCacheRegistration.create(buf.ptr, 2 * nb * seg, nb, seg, nb * seg, 2)
    cache = PagedKVCache(reg, bs, heads, dim, "bf16")
    n = 100
    blocks = (nb - 1 - np.arange(7) * 3 - first_block).astype(np.int32)
    small = Batch([3], [97], LLAMA, 4, seed=14, table_pad=0)
    t = np.arange(n)
    slots = blocks[t // bs].astype(np.int64) * bs + t % bs
    host = small.pages.values()
    at = small.table[0][t // bs], t % bs
    k, v = host[0][at], host[1][at]
    sd = device_array(slots, "int64")
    kd, vd = device_rows(k)[0], device_rows(v)[0]
    cache.write(kd, vd, sd)
    ko, vo = device_rows(np.zeros_like(k))[0], device_rows(np.zeros_like(v))[0]
    cache.read(sd, ko, vo)
    q, out = device_rows(small.q)[0], device_rows(np.zeros_like(small.q))[0]
    cache.attend(q, out, device_array(blocks[None], "int32"), device_array(small.lens, "int32"),
                 device_array(small.starts, "int32"), workspace=workspace)
    synchronize()
    assert np.array_equal(ko.download().view(np.uint16), k.reshape(-1))
    assert np.array_equal(vo.download().view(np.uint16), v.reshape(-1))
    small.check(out.download().view(np.uint16).reshape(small.q.shape), None)


def _hip():
    h = ctypes.CDLL("libamdhip64.so.7")
    for name, args in (("hipStreamBeginCapture", [ctypes.c_void_p, ctypes.c_int]),
                       ("hipStreamEndCapture", [ctypes.c_void_p, ctypes.POINTER(ctypes.c_void_p)]),
                       ("hipGraphInstantiate", [ctypes.POINTER(ctypes.c_void_p), ctypes.c_void_p,
                                                ctypes.c_void_p, ctypes.c_char_p, ctypes.c_size_t]),
                       ("hipGraphLaunch", [ctypes.c_void_p, ctypes.c_void_p]),
                       ("hipGraphExecDestroy", [ctypes.c_void_p]),
                       ("hipGraphDestroy", [ctypes.c_void_p])):
        getattr(h, name).argtypes = args
    return h


@pytest.mark.parametrize("form,group", [(LLAMA, 4), (FORMS[2], 4)], ids=str)
def test_captured_step(gpu, workspace, form, group):
    """Write, attend and read captured into one graph and replayed as the lengths, tokens and
    blocks change, with eager calls between the replays."""
    kind, rows, heads, dim, bs, _ = form
    rng = np.random.default_rng(15)
    hip, stream, eager = _hip(), Stream(), AttentionWorkspace()
    b = Batch([1, 1], [1500, 40], form, group, seed=16, table_pad=3, strides="contiguous")
    # Blocks for the tokens to come.
    grown = oracle.Pages(b.pages.num_blocks + 4, bs, heads, dim, kind, rows=rows)
    grown.seg()[:, :b.pages.num_blocks] = b.pages.seg()
    b.table[0, -3:] = b.pages.num_blocks
    b.table[1, (41 + bs - 1) // bs:] = b.pages.num_blocks + 1
    b.pages, b.dev = grown, DevicePages(grown)
    k, v = (device_rows(values(rng, (2, heads, dim), rows), rows=rows)[0] for _ in range(2))
    ko, vo = (device_rows(np.zeros((2, heads, dim), np.uint16), rows=rows)[0] for _ in range(2))
    q, out = device_rows(b.q, rows=rows)[0], device_rows(np.zeros_like(b.q), rows=rows)[0]
    slots, table = DeviceArray((2,), "int64"), device_array(b.table, "int32")
    lens, starts = DeviceArray((2,), "int32"), device_array(b.starts, "int32")
    graph, run = ctypes.c_void_p(), ctypes.c_void_p()

    def step(stream, ws):
        b.dev.cache.write(k, v, slots, stream)
        b.dev.cache.attend(q, out, table, lens, starts, max_query_len=1, workspace=ws,
                           stream=stream)
        b.dev.cache.read(slots, ko, vo, stream)

    assert hip.hipStreamBeginCapture(stream.handle, 2) == 0
    step(stream, workspace)
    assert hip.hipStreamEndCapture(stream.handle, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, 0) == 0
    for i in range(4):
        at = b.lens - 1 + i
        where = b.table[np.arange(2), at // bs].astype(np.int64) * bs + at % bs
        new_k, new_v = values(rng, (2, heads, dim), rows), values(rng, (2, heads, dim), rows)
        slots.upload(where)
        lens.upload((at + 1).astype(np.int32))
        k.upload(new_k)
        v.upload(new_v)
        b.q = values(rng, b.q.shape, rows)
        q.upload(b.q)
        synchronize()
        assert hip.hipGraphLaunch(run, stream.handle) == 0
        stream.synchronize()
        replayed = out.download(), ko.download(), vo.download()
        b.pages.set(where, new_k, new_v)
        saved, b.lens = b.lens, (at + 1).astype(np.int32)
        b.check(replayed[0].view(np.uint16).reshape(b.q.shape), None)
        b.lens = saved
        step(None, eager)
        synchronize()
        for x, y in zip(replayed, (out.download(), ko.download(), vo.download())):
            assert np.array_equal(x, y)
    hip.hipGraphExecDestroy(run)
    hip.hipGraphDestroy(graph)
    eager.close()


def test_streams_side_by_side(gpu):
    """Two streams with a workspace each, calls in flight on both."""
    runs = []
    for seed in (20, 21):
        b = Batch([1, 1], [2500, 900], LLAMA, 4, seed=seed, strides="contiguous")
        q, out = device_rows(b.q)[0], device_rows(np.zeros_like(b.q))[0]
        runs.append((b, Stream(), AttentionWorkspace(), q, out, device_array(b.table, "int32"),
                     device_array(b.lens, "int32"), device_array(b.starts, "int32")))
    synchronize()
    for _ in range(20):
        for b, s, w, q, out, t, l, st in runs:
            b.dev.cache.attend(q, out, t, l, st, max_query_len=1, workspace=w, stream=s)
    synchronize()
    for b, _, w, _, out, *_ in runs:
        b.check(out.download().view(np.uint16).reshape(b.q.shape), None)
        w.close()


def test_scale_defaults_to_the_head_size(gpu, workspace):
    b = Batch([3, 1], [50, 60], LLAMA, 4, seed=22)
    got = b.run(workspace=workspace)
    same = b.run(workspace=workspace, scale=1 / math.sqrt(128))
    assert np.array_equal(got[0], same[0])


@pytest.mark.parametrize("kind,rows,head_major", [("e4m3", "bf16", False), ("int8", "fp16", True),
                                                  ("bf16", "bf16", False)])
def test_saved_blocks_answer_as_before(gpu, workspace, kind, rows, head_major):
    """A serving step's life: a prompt's K and V written and attended, its full blocks saved by
    hash, the pages given to others, the blocks loaded elsewhere, and the next tokens written
    and attended behind them, with the bits that the pages would have given in place."""
    heads, dim, bs, nb, group, layers = 2, 64, 16, 40, 4, 2
    prompt, steps = 150, 12
    full = prompt // bs
    rng = np.random.default_rng(30)
    seg = segment_bytes(bs, heads, dim, kind)
    engine = PegaEngine(pool_size=64 << 20)
    bufs, caches, names = [], [], [f"layer.{i}" for i in range(layers)]
    for name in names:
        buf = DeviceBuffer(2 * nb * seg)
        buf.fill_random(len(bufs) + 1)
        engine.register_context_layer("inst", "ns", 0, name, buf.ptr, buf.nbytes, nb, seg,
                                      nb * seg, 2, 0, 1, layers)
        reg = KVCacheRegistration.create(buf.ptr, buf.nbytes, nb, seg, nb * seg, 2)
        bufs.append(buf)
        caches.append(PagedKVCache(reg, bs, heads, dim, kind, head_major=head_major))
    hashes = [bytes([i]) * 32 for i in range(full)]

    def run(cache, table, first, k, v, q):
        """Writes tokens `first` on and attends them; the outputs' bits."""
        n = len(k)
        t = np.arange(first, first + n)
        slots = device_array((table[t // bs].astype(np.int64) * bs + t % bs), "int64")
        cache.write(device_rows(k, rows=rows)[0], device_rows(v, rows=rows)[0], slots)
        out = device_rows(np.zeros_like(q), rows=rows)[0]
        cache.attend(device_rows(q, rows=rows)[0], out, device_array(table[None], "int32"),
                     device_array(np.array([first + n], np.int32), "int32"),
                     device_array(np.array([0, n], np.int32), "int32"), workspace=workspace,
                     max_seq_len=first + n, max_query_len=n)
        synchronize()
        return out.download().view(np.uint16).reshape(q.shape)

    old = rng.permutation(nb)[:20].astype(np.int32)
    data = [[values(rng, (prompt + steps, h, dim), rows) for h in (heads, heads, heads * group)]
            for _ in names]
    for cache, (k, v, q) in zip(caches, data):
        host = oracle.Pages(nb, bs, heads, dim, kind, head_major, rows)
        t = np.arange(prompt)
        host.set(old[t // bs].astype(np.int64) * bs + t % bs, k[:prompt], v[:prompt])
        got = run(cache, old, 0, k[:prompt], v[:prompt], q[:prompt])
        want, _, bound, _ = oracle.attend(host, q[:prompt], rows, old[None], [prompt], [0, prompt],
                                          dim ** -0.5, every=11)
        x = oracle.from_bits(got, rows).astype(np.float64)
        assert (np.abs(x - want) <= bound)[::11].all()
    engine.batch_save_kv_blocks("inst", 0, 0, [(n, [int(b) for b in old[:full]], hashes)
                                               for n in names])
    assert engine.count_prefix_hit_blocks("inst", hashes) == full
    # What the next tokens answer with the blocks in place.
    kept = [[run(cache, old, prompt + i, k[prompt + i:][:1], v[prompt + i:][:1],
                 q[prompt + i:][:1]) for i in range(steps)]
            for cache, (k, v, q) in zip(caches, data)]
    for buf in bufs:  # other requests' tokens, of any bits
        buf.fill_random(99)
    new = rng.permutation(nb)[:20].astype(np.int32)
    state = PyLoadState(num_layers=layers)
    engine.batch_load_kv_blocks("inst", 0, 0, state.shm_name(), names,
                                [int(b) for b in new[:full]], hashes)
    for i in range(layers):
        assert state.wait_for_layer(i, 60.0)
    for cache, (k, v, q), want in zip(caches, data, kept):
        # The block that was not full is computed again.
        run(cache, new, full * bs, k[full * bs:prompt], v[full * bs:prompt], q[full * bs:prompt])
        for i in range(steps):
            got = run(cache, new, prompt + i, k[prompt + i:][:1], v[prompt + i:][:1],
                      q[prompt + i:][:1])
            assert np.array_equal(got, want[i])
    engine.close()
    for buf in bufs:
        buf.close()
