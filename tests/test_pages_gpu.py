"""Forks, copies of blocks and kept tokens moved together on the GPU, byte by byte against
numpy's, in all layers."""

import numpy as np
import pytest

from oracle import paged as oracle
from pegaflow_amd._lib import PegaFlowError
from pegaflow_amd.paged_cache import PagedLayers
from pegaflow_amd.runtime import DeviceArray, Stream, synchronize
from test_paged_cache_gpu import FORMS, DevicePages, device_array

pytestmark = pytest.mark.gpu


def cache_of(rng, form, layers, nb, pad=0, blocks_first=False):
    kind, rows, heads, dim, bs, head_major = form
    out = []
    for _ in range(layers):
        pages = oracle.Pages(nb, bs, heads, dim, kind, head_major, rows, pad=pad,
                             blocks_first=blocks_first)
        pages.bytes[:] = rng.integers(0, 256, pages.bytes.shape, np.uint8)
        out.append(DevicePages(pages))
    return out, PagedLayers([d.cache for d in out])


def copy_block(pages, a, b):
    """A block's values and scales, without what a segment has behind them."""
    used = oracle.Pages(1, pages.block_size, pages.heads, pages.dim, pages.kind,
                        rows=pages.rows).segment
    pages.seg()[:, b, :used] = pages.seg()[:, a, :used].copy()


def check(devs):
    for d in devs:
        assert np.array_equal(d.bytes(), d.host.bytes)


@pytest.mark.parametrize("n", [0, 1, 9, 40])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_copy_blocks(gpu, form, n):
    rng = np.random.default_rng(n)
    nb = 2 * n + 4
    devs, layers = cache_of(rng, form, 3, nb, pad=32 * (n % 2), blocks_first=n == 9)
    order = rng.permutation(nb).astype(np.int32)
    a, b = order[:n].copy(), order[n:2 * n].copy()
    if n > 5:
        a[1] = a[2]  # one block, to two
        a[3], b[4], a[5] = -1, nb, 1 << 30
    layers.copy_blocks(device_array(a, "int32"), device_array(b, "int32"))
    synchronize()
    for d in devs:
        for x, y in zip(a, b):
            if 0 <= x < nb and 0 <= y < nb:
                copy_block(d.host, x, y)
    check(devs)
    layers.close()


@pytest.mark.parametrize("children", [0, 1, 7, 50])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_fork(gpu, form, children):
    rng = np.random.default_rng(children + 1)
    bs, seqs, width = form[4], 5, 6
    nb = seqs * width + children
    devs, layers = cache_of(rng, form, 2, nb, blocks_first=children == 7)
    order = rng.permutation(nb).astype(np.int32)
    table = np.full((seqs, width + 3), 77, np.int32)  # rows of a wider table
    table[:, :width] = order[:seqs * width].reshape(seqs, width)
    lens = rng.integers(0, width * bs + 1, seqs).astype(np.int32)
    lens[0], lens[1], lens[2] = 0, width * bs, 2 * bs
    parents = rng.integers(0, seqs, children).astype(np.int32)
    new = order[seqs * width:].copy()
    if children > 5:
        parents[1], parents[2] = -1, seqs
        new[3], new[4] = -1, nb
        parents[3] = parents[4] = parents[5] = 3
        lens[3] = bs + bs // 2
    wide = device_array(table, "int32")
    out = np.full((children, width + 1), -7, np.int32)
    out_dev = device_array(out, "int32")
    layers.fork(DeviceArray((seqs, width), "int32", wide.buffer, 0, (width + 3, 1)),
                device_array(lens, "int32"), device_array(parents, "int32"),
                device_array(new, "int32"),
                DeviceArray((children, width), "int32", out_dev.buffer, 0, (width + 1, 1)))
    synchronize()
    for i, p in enumerate(parents):
        if not 0 <= p < seqs:
            continue
        out[i, :width] = table[p, :width]
        page = lens[p] // bs
        if page < width and 0 <= new[i] < nb:
            out[i, page] = new[i]
            if lens[p] % bs:
                for d in devs:
                    copy_block(d.host, table[p, page], new[i])
    got = out_dev.download().view(np.int32).reshape(out.shape) if children else out
    assert np.array_equal(got, out)
    check(devs)


class Moves:
    """A batch of sequences with kept tokens, and what moving them leaves."""

    def __init__(self, form, seed, counts, lengths, layers=2, in_place=True, first=True,
                 ordered=True):
        rng = np.random.default_rng(seed)
        self.bs = bs = form[4]
        seqs = len(counts)
        width = max(max(lengths) // bs + 1, 1)
        used = seqs * width
        self.nb = nb = 2 * used + 3
        self.devs, self.layers = cache_of(rng, form, layers, nb, blocks_first=seed % 2 == 1)
        order = rng.permutation(nb).astype(np.int32)
        self.table = order[:used].reshape(seqs, width).copy()
        self.out_table = self.table if in_place else order[used:2 * used].reshape(seqs, width).copy()
        self.kept, self.starts, self.first = [], [0], []
        for n, length in zip(counts, lengths):
            at = int(rng.integers(0, length - n + 1)) if first else 0
            self.first.append(at)
            self.kept += sorted(rng.choice(np.arange(at, length), n, replace=False).tolist())
            self.starts.append(self.starts[-1] + n)
        self.kept = np.array(self.kept, np.int32)
        self.starts = np.array(self.starts, np.int32)
        self.first = np.array(self.first, np.int32)
        self.in_place = in_place

    def run(self, with_first=True, **more):
        table = device_array(self.table, "int32")
        out = None if self.in_place else device_array(self.out_table, "int32")
        self.out_lens = device_array(np.full(len(self.first), -5, np.int32), "int32")
        self.layers.compact(table, device_array(self.kept, "int32"),
                            device_array(self.starts, "int32"),
                            first=device_array(self.first, "int32") if with_first else None,
                            out_table=out, out_lens=self.out_lens, **more)
        synchronize()

    def check(self):
        bs, nb = self.bs, self.nb
        room = self.table.shape[1] * bs
        for d in self.devs:
            pages = d.host
            was = oracle.Pages(nb, bs, pages.heads, pages.dim, pages.kind, pages.head_major,
                               pages.rows, blocks_first=pages.blocks_first)
            was.bytes = pages.bytes.copy()
            for i in range(len(self.first)):
                for j in range(self.starts[i], self.starts[i + 1]):
                    a, b = self.kept[j], self.first[i] + j - self.starts[i]
                    if not (0 <= a < room and b < room):
                        continue
                    x, y = self.table[i, a // bs], self.out_table[i, b // bs]
                    if not (0 <= x < nb and 0 <= y < nb):
                        continue
                    pages.values()[:, y, b % bs] = was.values()[:, x, a % bs]
                    if pages.kind in oracle.LARGEST:
                        pages.scales().view(np.uint32)[:, y, b % bs] = \
                            was.scales().view(np.uint32)[:, x, a % bs]
        check(self.devs)
        assert np.array_equal(self.out_lens.download().view(np.int32),
                              self.first + np.diff(self.starts))


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("counts,lengths", [((1,), (1,)), ((0,), (9,)), ((3, 0, 16, 5), (7, 4, 16, 24)),
                                            ((17, 130, 1), (30, 500, 3)), ((700,), (1100,))], ids=str)
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_compact(gpu, form, counts, lengths, in_place):
    """Few and many kept tokens, across several chunks, in place and to other blocks."""
    m = Moves(form, len(counts) + counts[0], counts, lengths, in_place=in_place)
    m.run()
    m.check()


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("hint", [0, 1, 5, 1 << 40])
def test_compact_whatever_the_hint_says(gpu, hint, in_place):
    m = Moves(FORMS[2], 3, (300, 20), (1000, 33), in_place=in_place)
    m.run(max_kept=hint)
    m.check()


def test_compact_everything_and_nothing(gpu):
    """A sequence that keeps all stays as it is; from position 0 without a list of firsts."""
    m = Moves(FORMS[0], 8, (50, 0), (50, 20), first=False)
    m.run(with_first=False)
    m.check()


@pytest.mark.parametrize("in_place", [True, False])
def test_compact_of_tokens_that_are_not_there(gpu, in_place):
    """Positions outside the table and blocks that do not exist do not move; starts that lie
    outside the list are cut to it."""
    m = Moves(FORMS[4], 9, (40, 6), (90, 20), in_place=in_place)
    m.kept[3] = -4
    m.kept[39] = 1 << 30
    m.table[0, 5] = -1
    m.table[0, 7] = m.nb
    m.out_table[1, 0] = -9
    m.run()
    m.check()
    starts = m.starts.copy()
    m.starts = np.array([40, 46, 1 << 30], np.int32)  # the second has none
    m.table, m.out_table = m.table[::-1].copy(), m.out_table[::-1].copy()
    if in_place:
        m.out_table = m.table
    m.first = m.first[::-1].copy()
    m.run()
    m.starts = np.array([40, 46, 46], np.int32)
    m.check()
    assert len(starts) == 3


def test_moves_again_on_another_stream(gpu):
    """A move in place takes what the one before it left."""
    m = Moves(FORMS[2], 12, (6, 3), (40, 30))
    s = Stream()
    for _ in range(3):
        m.run(stream=s)
        s.synchronize()
        m.check()


def test_refusals(gpu):
    rng = np.random.default_rng(0)
    devs, layers = cache_of(rng, FORMS[0], 2, 8)
    other, _ = cache_of(rng, FORMS[1], 1, 8)
    with pytest.raises(PegaFlowError, match="another shape"):
        PagedLayers([devs[0].cache, other[0].cache])
    with pytest.raises(ValueError, match="no layers"):
        PagedLayers([])
    table = device_array(np.zeros((2, 4), np.int32), "int32")
    one, two = (device_array(np.zeros(n, np.int32), "int32") for n in (1, 2))
    three = device_array(np.zeros(3, np.int32), "int32")
    with pytest.raises(ValueError, match="blocks to copy"):
        layers.copy_blocks(one, two)
    with pytest.raises(ValueError, match="int32"):
        layers.copy_blocks(device_array(np.zeros(2, np.int64), "int64"), two)
    with pytest.raises(ValueError, match="new blocks"):
        layers.fork(table, two, two, one, table)
    with pytest.raises(PegaFlowError, match="itself"):
        layers.fork(table, two, two, two, table)
    out = device_array(np.zeros((2, 4), np.int32), "int32")
    narrow = DeviceArray((2, 4), "int32", out.buffer, 0, (2, 1))
    with pytest.raises(PegaFlowError, match="overlap"):
        layers.fork(table, two, two, two, narrow)
    with pytest.raises(ValueError, match="starts of kept"):
        layers.compact(table, two, two)
    with pytest.raises(ValueError, match="max_kept"):
        layers.compact(table, two, three, max_kept=-1)
    with pytest.raises(ValueError, match="of first"):
        layers.compact(table, two, three, first=one)
    with pytest.raises(PegaFlowError, match="two strides"):
        layers.compact(table, two, three, out_table=_restrided(table))
    layers.close()
    with pytest.raises(PegaFlowError, match="null layers"):
        layers.copy_blocks(one, one)


def _restrided(table):
    """The table's address with rows further apart."""
    class View:
        shape, dtype = (2, 4), "int32"

        def data_ptr(self):
            return table.data_ptr()

        def stride(self):
            return (5, 1)
    return View()
