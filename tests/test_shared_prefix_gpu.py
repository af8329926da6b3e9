"""Attention of batches whose sequences share their first tokens, on the GPU against the
definition of attention over each sequence's whole block table (oracle/paged.py)."""

import numpy as np
import pytest

from oracle import paged as oracle
from pegaflow_amd._lib import PegaFlowError
from pegaflow_amd.paged_cache import AttentionWorkspace
from pegaflow_amd.runtime import Stream, synchronize
from test_paged_cache_gpu import (ATTEND_FORMS, FORMS, INF16, LLAMA, NAN16, Batch, DevicePages,
                                  device_array, device_rows, values, workspace)  # noqa: F401

pytestmark = pytest.mark.gpu


class SharedBatch(Batch):
    """Groups of sequences, ``sizes`` of them behind ``shared`` whole blocks each, and others
    behind them; blocks that no sequence has, and tokens past each end, hold NaN.  ``own`` cached
    tokens below 0 are missing of the shared ones."""

    def __init__(self, sizes, shared, own, new, form, group, seed=0, sharp=1.0, strides="fused"):
        self.kind, self.rows, heads, dim, bs, head_major = form
        rng = np.random.default_rng(seed)
        self.new = list(new)
        count = len(new)
        of = [g for g, n in enumerate(sizes) for _ in range(n)]
        of += [None] * (count - len(of))
        blocks = [0 if g is None else shared[g] for g in of]
        lens = np.array([b * bs + a + n for b, a, n in zip(blocks, own, new)])
        self.cached = [int(n) - m for n, m in zip(lens, new)]
        own_blocks = [max(-(-int(n) // bs) - b, 0) for n, b in zip(lens, blocks)]
        nb = sum(shared) + sum(own_blocks) + 4
        pages = oracle.Pages(nb, bs, heads, dim, self.kind, head_major, self.rows)
        if self.kind in oracle.LARGEST:
            pages.values()[:] = 0x7f if self.kind == "e4m3" else 0x55
            pages.scales()[:] = np.nan
        else:
            pages.values()[:] = NAN16[self.rows]
        order = rng.permutation(nb).astype(np.int32)
        self.table = np.full((count, int(-(-lens.max() // bs)) + 1), -1, np.int32)

        def fill(block_list, n):
            t = np.arange(n)
            slots = np.asarray(block_list)[t // bs].astype(np.int64) * bs + t % bs
            pages.set(slots, values(rng, (n, heads, dim), self.rows),
                      values(rng, (n, heads, dim), self.rows))

        at = 0
        first = []
        for n in shared:
            first.append(order[at:at + n])
            if n:
                fill(first[-1], n * bs)
            at += n
        for i, g in enumerate(of):
            b, u = blocks[i], own_blocks[i]
            if b:
                self.table[i, :b] = first[g]
            if lens[i] < b * bs:
                b = -(-int(lens[i]) // bs)
            self.table[i, b:b + u] = order[at:at + u]
            if u:
                fill(order[at:at + u], int(lens[i]) - b * bs)
            at += u
            self.table[i, b + u:] = (order[0], -7, nb, 2 ** 31 - 1)[i % 4]
        self.pages, self.dev = pages, DevicePages(pages)
        self.lens = lens.astype(np.int32)
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        total = int(self.starts[-1])
        q = rng.standard_normal((total, heads * group, dim)) * sharp
        self.q = oracle.to_bits(q.astype(np.float32), self.rows)
        self.strides, self.group = strides, group
        self.scale = dim ** -0.5
        self.group_starts = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
        self.shared_lens = (np.array(shared) * bs).astype(np.int32)

    def attend(self, q, out, lse, starts, workspace, stream, **kw):
        self.dev.cache.attend_shared(
            q, out, device_array(self.table, "int32"), device_array(self.lens, "int32"), starts,
            device_array(self.group_starts, "int32"), device_array(self.shared_lens, "int32"),
            lse=lse, workspace=workspace, stream=stream, **kw)

    def run(self, tail=0, front=0, workspace=None, lse=True, stream=None, hints=True, **kw):
        n, heads, dim = self.q.shape
        bits = np.concatenate([np.full((front, heads, dim), 0x1111, np.uint16), self.q,
                               np.full((tail, heads, dim), 0x1111, np.uint16)])
        q = device_rows(bits, self.strides, self.rows, offset=8)[0]
        out, flat, view = device_rows(np.full_like(bits, 0x5a5a), self.strides, self.rows)
        held = device_array(np.full(bits.shape[:2], 77, np.float32), "fp32") if lse else None
        if hints:
            # More than there is: a batch as small as these would not be worth sharing.
            kw.setdefault("max_shared_len", 1 << 30)
            kw.setdefault("max_own_len", int(self.lens.max()) if len(self.lens) else 0)
            kw.setdefault("max_query_len", max(self.new) if self.new else 0)
        self.attend(q, out, held, device_array(self.starts + front, "int32"), workspace, stream,
                    **kw)
        synchronize()
        back = out.buffer.download().view(np.uint16)
        got = np.lib.stride_tricks.as_strided(back, view.shape, view.strides).copy()
        view[front:front + n] = got[front:front + n]
        assert np.array_equal(back, flat)
        if not lse:
            return got[front:front + n], None
        got_lse = held.download().view(np.float32).reshape(bits.shape[:2])
        assert (got_lse[:front] == 77).all() and (got_lse[front + n:] == 77).all()
        return got[front:front + n], got_lse[front:front + n]

    def check(self, got, lse, causal=True, scale=None, every=1):
        """Weights of shared tokens are rounded once."""
        out, want_lse, bound, lse_bound = (x[::every] for x in oracle.attend(
            self.pages, self.q, self.rows, self.table, self.lens, self.starts,
            scale or self.scale, causal, 0, every=every))
        x = oracle.from_bits(got, self.rows).astype(np.float64)[::every]
        assert np.array_equal(np.isnan(x), np.isnan(out))
        assert np.array_equal(x[np.isinf(out)], out[np.isinf(out)])
        fine = np.isfinite(out)
        off = np.abs(x - out)[fine] / np.maximum(bound[fine], 1e-300)
        assert off.size == 0 or off.max() <= 1, off.max()
        if lse is not None:
            lse = lse[::every]
            gone = np.isneginf(want_lse)
            assert np.array_equal(np.isneginf(lse), gone)
            assert (x[gone] == 0).all()
            keep = np.isfinite(want_lse)
            assert (np.abs(lse - want_lse)[keep] <= lse_bound[keep]).all()


@pytest.mark.parametrize("strides", ["fused", "odd"])
@pytest.mark.parametrize("form,group", ATTEND_FORMS, ids=str)
def test_single_tokens(gpu, workspace, form, group, strides):
    """Two groups and two sequences alone, own tokens from none to several tiles."""
    bs = form[4]
    b = SharedBatch([5, 3], [-(-130 // bs), -(-64 // bs)], [0, 1, 31, 64, 150, 7, 0, 33, 90, 0],
                    [1] * 10, form, group, seed=1, strides=strides)
    for w in (None, workspace):
        b.check(*b.run(workspace=w, front=1, tail=2))


@pytest.mark.parametrize("form,group", ATTEND_FORMS, ids=str)
def test_drafts(gpu, workspace, form, group):
    """One to eight new tokens, up to 64 rows of a KV head and (where the call runs as
    ``attend``) beyond."""
    bs = form[4]
    most = max(1, min(8, 64 // group))
    new = [1 + (3 * i) % most for i in range(9)]
    new[4] = most
    for most_new in (most, 0):
        b = SharedBatch([2, 4], [-(-300 // bs), -(-77 // bs)], [0, 40, 3, 129, 0, 64, 20, 0, 65],
                        new, form, group, seed=2)
        b.check(*b.run(workspace=workspace, tail=1, max_query_len=most_new))


@pytest.mark.parametrize("form,group", [(LLAMA, 4), (FORMS[2], 4), (FORMS[1], 1), (FORMS[3], 4)],
                         ids=str)
@pytest.mark.parametrize("sizes,shared,own,new", [
    ((3,), (3000,), (10, 700, 0), (1, 1, 1)),
    ((2, 2), (2048, 1500), (1, 2000, 1100, 30), (1, 3, 2, 1)),
    ((40,), (1200,), tuple(range(40)), (1,) * 40)], ids=str)
def test_long_prefixes_are_split_and_joined(gpu, workspace, form, group, sizes, shared, own, new):
    """The same bits every time, in workspaces of any size, whatever the hints say."""
    b = SharedBatch(sizes, [n // form[4] for n in shared], own, new, form, group, seed=3)
    every = 7 if len(new) > 10 else 1
    first = b.run(workspace=workspace)
    b.check(*first, every=every)
    for _ in range(3):
        again = b.run(workspace=workspace)
        assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])
    rows = len(b.q) * b.q.shape[1] * (form[3] * 4 + 8)  # of one share
    for room in (1.5, 2.01, 3.01, 5.7):
        small = AttentionWorkspace(int(room * rows / (1 - 1 / 16)) + 4096)
        b.check(*b.run(workspace=small), every=every)
        small.close()
    for hints in (dict(max_shared_len=1, max_own_len=1), dict(max_shared_len=1 << 40),
                  dict(max_own_len=1), dict(max_shared_len=max(shared), max_own_len=max(own) + 1),
                  dict(max_own_len=1 << 31), dict(max_shared_len=0, max_own_len=0)):
        b.check(*b.run(workspace=workspace, **hints), every=every)


def test_shared_lengths_of_any_size(gpu, workspace):
    """Lengths that end inside a block, none and negative ones."""
    for shared in ([0, 5], [13, 47], [1, 64], [150, 64], [160, 63], [-3, -2 ** 31]):
        b = SharedBatch([3, 4], [10, 4], [0, 12, 40, 9, 0, 1, 70], [2, 1, 3, 1, 5, 1, 2], FORMS[0],
                        4, seed=4)
        b.shared_lens = np.array(shared, np.int32)
        b.check(*b.run(workspace=workspace))


@pytest.mark.parametrize("form,group", [(LLAMA, 4), (FORMS[4], 5)], ids=str)
def test_sequences_that_have_cached_less(gpu, workspace, form, group):
    """A sequence shares what it has cached, whatever the others have: its new tokens, and its
    end, may lie among the shared ones."""
    bs = form[4]
    n = [-(-k // bs) for k in (1000, 100)]
    b = SharedBatch([5, 3], n, [-900, 12, -1, -n[0] * bs, -400, -70, -n[1] * bs + 3, -3],
                    [2, 1, 3, 1, 2, 1, 2, 1], form, group, seed=15)
    b.check(*b.run(workspace=workspace))
    # Sequences that share all they have cached.
    b = SharedBatch([4], [60], [-50 * bs + 7, -1, -60 * bs + 5, -20 * bs], [2, 3, 1, 1], form, group, seed=16)
    b.shared_lens[:] = 2 ** 31 - 1
    b.check(*b.run(workspace=workspace))


@pytest.mark.parametrize("form", [FORMS[0], FORMS[4]], ids=str)
def test_padded_batches(gpu, workspace, form):
    """Sequences without rows, and without tokens, anywhere in a group; groups of none and of
    one."""
    bs = form[4]
    n = [-(-k // bs) for k in (200, 40, 90)]
    b = SharedBatch([4, 0, 1, 5], [n[0], 0, n[1], n[2]], [0, 9, 30, 2, 17, 0, 1, 2, 3, 4, 5],
                    [0, 1, 0, 2, 1, 0, 0, 1, 3, 1, 1], form, 4, seed=5)
    b.table[0] = -5  # a sequence without rows has a row of the table that says nothing
    b.check(*b.run(workspace=workspace, tail=1))
    # One that has rows but no tokens: its rows attend nothing.
    b.lens[8] = 0
    b.check(*b.run(workspace=workspace))
    b.lens[:] = 0
    got, lse = b.run(workspace=workspace)
    assert (oracle.from_bits(got, b.rows) == 0).all() and np.isneginf(lse).all()


def test_many_groups_and_sequences(gpu, workspace):
    """More than the 64 that a wave looks at together."""
    rng = np.random.default_rng(6)
    sizes = [int(n) for n in rng.integers(0, 4, 90)]
    new = [1] * (sum(sizes) + 3)
    b = SharedBatch(sizes, [int(n) for n in rng.integers(0, 6, 90)],
                    [int(n) for n in rng.integers(0, 60, len(new))], new, FORMS[1], 1, seed=6)
    b.check(*b.run(workspace=workspace))
    b = SharedBatch([130, 70], [20, 5], [i % 41 for i in range(203)], [1 + i % 2 for i in range(203)],
                    (*FORMS[2][:2], 2, *FORMS[2][3:]), 4, seed=7)
    b.check(*b.run(workspace=workspace))


def test_blocks_that_do_not_exist(gpu, workspace):
    """Missing blocks among the shared and the own ones hide their tokens."""
    for form in (FORMS[0], FORMS[5], FORMS[2]):
        bs = form[4]
        b = SharedBatch([4], [-(-300 // bs)], [100, 50, 0, 64], [1, 2, 1, 3], form, 3, seed=8)
        b.table[:4, 1] = -1
        b.table[:4, 3] = 2 ** 31 - 1
        b.table[0, -(-300 // bs)] = b.pages.num_blocks
        b.check(*b.run(workspace=workspace))
    b = SharedBatch([3], [8], [0, 0, 0], [1, 1, 1], FORMS[0], 4, seed=9)
    b.table[:] = -1
    got, lse = b.run(workspace=workspace)
    assert (got == 0).all() and np.isneginf(lse).all()


@pytest.mark.parametrize("kind,rows", [("bf16", "bf16"), ("fp16", "fp16"), ("e4m3", "bf16")])
def test_infinities_and_nan(gpu, workspace, kind, rows):
    """In V they spoil the values that they stand at, in K the rows; before, in and behind the
    last tile of the shared tokens and of the own."""
    form = (kind, rows, 2, 64, 16, False)
    b = SharedBatch([3], [17], [40, 5, 0], [1, 2, 1], form, 3, seed=10)
    v = b.pages.values()
    for where, t, value in ((0, 3, 5), (1, 270, 9), (0, 275, 30), (2, 271, 60)):
        block = b.table[where, t // 16]
        if kind == "e4m3":
            v[1, block, t % 16, 1, value] = 0x7f
        else:
            v[1, block, t % 16, 1, value] = (INF16, NAN16)[value % 2][rows]
    b.dev.upload()
    b.check(*b.run(workspace=workspace))
    if kind != "e4m3":
        v[0, b.table[1, 17], 1, 0, 7] = NAN16[rows]  # sequence 1's own token
        b.dev.upload()
        b.check(*b.run(workspace=workspace, lse=False))


@pytest.mark.parametrize("form,group", [(LLAMA, 4), (FORMS[4], 5)], ids=str)
def test_without_the_causal_mask(gpu, workspace, form, group):
    """Every row attends all its sequence's tokens, new ones too."""
    bs = form[4]
    b = SharedBatch([3, 2], [-(-200 // bs), -(-31 // bs)], [0, 70, 3, 129, 0, 64], [2, 1, 3, 1, 2, 1],
                    form, group, seed=11)
    b.check(*b.run(workspace=workspace, causal=False), causal=False)


@pytest.mark.parametrize("scale", [0.3, -0.2, 0.0])
def test_scales(gpu, workspace, scale):
    b = SharedBatch([4], [30], [0, 70, 3, 12], [1, 2, 1, 3], FORMS[0], 4, seed=12, sharp=2.0)
    got = b.run(workspace=workspace, scale=scale)
    b.check(*got, scale=scale or 1e-30)


def test_rows_beyond_the_bound_stay(gpu, workspace):
    """Rows that a sequence has beyond max_query_len are left or right, and all others right."""
    b = SharedBatch([3], [20], [0, 70, 3], [1, 30, 2], FORMS[0], 4, seed=13)
    out, _, bound, _ = oracle.attend(b.pages, b.q, b.rows, b.table, b.lens, b.starts, b.scale)
    got, lse = b.run(workspace=workspace, max_query_len=2)
    x = oracle.from_bits(got, b.rows).astype(np.float64)
    right = (np.abs(x - out) <= bound).all(-1)
    left = (got == 0x5a5a).all(-1) & (lse == 77)
    assert (right | left).all()
    keep = np.ones(len(got), bool)
    keep[3:31] = False  # sequence 1's rows from its third on
    assert right[keep].all()


def test_on_a_stream_and_refusals(gpu, workspace):
    b = SharedBatch([4], [30], [0, 70, 3, 12], [1, 2, 1, 3], FORMS[0], 4, seed=14)
    stream = Stream()
    b.check(*b.run(workspace=workspace, stream=stream))
    cache = b.dev.cache
    q, _, _ = device_rows(b.q)
    out, _, _ = device_rows(b.q)
    batch = [device_array(x, "int32") for x in (b.table, b.lens, b.starts)]
    starts, lens = device_array(b.group_starts, "int32"), device_array(b.shared_lens, "int32")
    with pytest.raises(ValueError, match="group starts"):
        cache.attend_shared(q, out, *batch, lens, lens)
    with pytest.raises(ValueError, match="int32"):
        cache.attend_shared(q, out, *batch, starts, device_array(np.zeros(1, np.int64), "int64"))
    for hint in ("max_shared_len", "max_own_len", "max_query_len"):
        with pytest.raises(ValueError, match="not negative"):
            cache.attend_shared(q, out, *batch, starts, lens, **{hint: -1})
    lens._offset = 1 << 20
    with pytest.raises(PegaFlowError, match="shared_lens"):
        cache.attend_shared(q, out, *batch, starts, lens, workspace=workspace)
    # No groups: attend's own bits.
    none = [device_array(np.zeros(1, np.int32), "int32"), device_array(np.zeros(0, np.int32), "int32")]
    cache.attend_shared(q, out, *batch, *none, max_query_len=3, workspace=workspace)
    synchronize()
    got = out.download()
    cache.attend(q, out, *batch, max_query_len=3, workspace=workspace)
    synchronize()
    assert np.array_equal(got, out.download())


def test_hints_as_they_are(gpu, workspace):
    """Batches that are worth sharing by their true lengths: many bytes saved, and drafts."""
    own = [(37 * i) % 200 for i in range(20)]
    b = SharedBatch([20], [95], own, [1] * 20, LLAMA, 4, seed=20)
    b.check(*b.run(workspace=workspace, max_shared_len=95 * 16, max_own_len=max(own) + 1), every=3)
    b = SharedBatch([3, 2], [20, 7], own[:6], [5, 1, 4, 2, 5, 3], FORMS[3], 4, seed=21)
    b.check(*b.run(workspace=workspace, max_shared_len=320, max_own_len=max(own[:6]) + 5))


@pytest.mark.parametrize("kw", [dict(window=7), dict(window=300), dict(workspace=None),
                                dict(max_query_len=0)], ids=str)
def test_calls_that_run_as_attend(gpu, workspace, kw):
    """With a window, without a workspace or with more rows than share: attend's own bits."""
    b = SharedBatch([4], [30], [0, 70, 3, 12], [30, 2, 1, 3], FORMS[0], 4, seed=22)
    kw = {"workspace": workspace, **kw}
    got = b.run(**kw)
    n, heads, dim = b.q.shape
    q, _, _ = device_rows(b.q, b.strides, b.rows, offset=8)
    out, _, _ = device_rows(b.q, "contiguous", b.rows)
    kw.setdefault("max_query_len", 30)
    b.dev.cache.attend(q, out, device_array(b.table, "int32"), device_array(b.lens, "int32"),
                       device_array(b.starts, "int32"),
                       max_seq_len=min(1 << 30, 2 ** 32 - 1) + int(b.lens.max()), **kw)
    synchronize()
    assert np.array_equal(got[0], out.download().view(np.uint16).reshape(n, heads, dim))


def test_two_calls_at_once(gpu):
    """On two streams, each with a workspace of its own."""
    batches = [SharedBatch([9], [40], [(13 * i) % 90 for i in range(10)], [1 + i % 3 for i in range(10)],
                           form, 4, seed=23) for form in (LLAMA, FORMS[2])]
    alone = []
    calls = []
    for b in batches:
        w = AttentionWorkspace()
        alone.append(b.run(workspace=w)[0])
        q, _, _ = device_rows(b.q, b.strides, b.rows)
        out, _, _ = device_rows(b.q, "contiguous", b.rows)
        arrays = [device_array(x, "int32") for x in (b.table, b.lens, b.starts, b.group_starts,
                                                     b.shared_lens)]
        calls.append((b.dev.cache, q, out, arrays, w, Stream()))
    hints = dict(max_shared_len=1 << 30, max_own_len=int(batches[0].lens.max()), max_query_len=3)
    for _ in range(20):
        for cache, q, out, arrays, w, stream in calls:
            cache.attend_shared(q, out, *arrays, workspace=w, stream=stream, **hints)
    for (_, _, out, _, _, stream), want in zip(calls, alone):
        stream.synchronize()
        assert np.array_equal(out.download().view(np.uint16).reshape(want.shape), want)
