"""Rotary positions on the GPU against their definition (oracle/paged.py): queries turned, keys
turned and written, values written as ``write`` writes them."""

import numpy as np
import pytest

from oracle import paged as oracle
from pegaflow_amd._lib import PegaFlowError
from pegaflow_amd.paged_cache import RotaryPositions
from pegaflow_amd.runtime import DeviceBuffer, DeviceArray, Stream, synchronize
from test_paged_cache_gpu import FORMS, DevicePages, device_array, device_rows, values

pytestmark = pytest.mark.gpu

HALF = oracle.HALF_STEP
# The least step of a row type, halved.
LEAST = {"bf16": 2.0 ** -134, "fp16": 2.0 ** -25}


def check_rows(bits, want, bound, rows):
    got = oracle.from_bits(bits, rows).astype(np.float64)
    allowed = HALF[rows] * (np.abs(want) + bound) + bound + LEAST[rows]
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= allowed).all(), np.abs(got - want).max()


def check_codes(pages, kv, slots, want, bound):
    """8-bit codes and scales of turned rows [n, heads, dim] in 64 bits."""
    b, t = slots // pages.block_size, slots % pages.block_size
    s = pages.scales()[kv, b, t].astype(np.float64)
    largest = np.abs(want).max(-1)
    # 1 / L, the product: a half-step each.  Under 2^-126 numbers are held to 2^-149: a turned
    # value, three roundings, is off by another 2^-148 at most, a scale by 2^-150 of its own, and
    # a code times it by L times that.
    top = oracle.LARGEST[pages.kind]
    tiny = 2.0 ** -148
    assert (np.abs(s - largest / top)
            <= (largest * 2.0 ** -22 + bound.max(-1) + tiny) / top + 2.0 ** -150).all()
    held = oracle.decode(pages.values()[kv, b, t], pages.kind) * s[..., None]
    off = bound + 2.0 ** -22 * np.abs(want) + 2.0 ** -22 * largest[..., None]
    off = off + np.where(largest < 2.0 ** -110, 2 * tiny + top * 2.0 ** -149, 0)[..., None]
    if pages.kind == "int8":
        step = s[..., None] / 2 + off
    else:  # half a step of 3 bits behind the first, or of the least, 2^-9
        step = np.maximum(2.0 ** -4 * (np.abs(want) + off), s[..., None] * 2.0 ** -10) + off
    assert (np.abs(held - want) <= step).all()


def rotaries(dim):
    return [(dim, "half"), (dim, "interleaved"), (max(2, dim // 2), "half"), (2, "half"),
            (max(2, dim - 6), "half"), (max(2, dim // 4 * 2 - 2), "interleaved"),
            (max(16, dim // 16 * 8 // 16 * 16), "interleaved")]


@pytest.mark.parametrize("n", [0, 1, 3, 70])
@pytest.mark.parametrize("which", range(7))
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_write_rotated(gpu, form, which, n):
    """Every byte of the pages and every query row, of all forms, layouts and strides."""
    kind, rows, heads, dim, bs, head_major = form
    r, layout = rotaries(dim)[which]
    group = (which + heads) % 3 * 2 + 1
    rng = np.random.default_rng(100 * which + n + dim)
    nb = n // bs * 2 + 5
    pages = oracle.Pages(nb, bs, heads, dim, kind, head_major, rows, pad=16 * (n % 2),
                         blocks_first=n % 2 == 1 and bs % 2 == 0)
    pages.bytes[:] = rng.integers(0, 256, pages.bytes.shape, np.uint8)
    dev = DevicePages(pages)
    strides = ["contiguous", "fused", "heads_first", "odd"][(n + which) % 4]
    q = values(rng, (n, heads * group, dim), rows)
    k, v = values(rng, (n, heads, dim), rows), values(rng, (n, heads, dim), rows)
    slots = rng.permutation(nb * bs)[:n].astype(np.int64)
    if n > 10:
        slots[5], slots[6], slots[7], slots[8] = -1, nb * bs, -(1 << 40), 1 << 40
        k[0] = 0
        k[1, 0] = 1  # the least numbers
        v[2] = 0
    positions = rng.integers(0, 40000, n)
    factor = [1.0, 1.25][which % 2]
    rotary = RotaryPositions(r, layout=layout, frequencies=[
        500000.0 ** (-2 * i / r) for i in range(r // 2)], factor=factor)
    qd, _, _ = device_rows(q, strides, rows, offset=8 if strides != "odd" else 1)
    out, out_flat, out_view = device_rows(np.zeros_like(q), "fused", rows,
                                          offset=0 if which % 3 else 3)
    kd, _, _ = device_rows(k, strides, rows)
    vd, _, _ = device_rows(v, strides, rows)
    dev.cache.write_rotated(qd, out, kd, vd, device_array(positions, "int64"),
                            device_array(slots, "int64"), rotary)
    synchronize()
    want, bound = oracle.rotate(oracle.from_bits(q, rows), positions, rotary.frequencies, layout,
                                factor)
    got = out.buffer.download().view(np.uint16)
    inner = np.lib.stride_tricks.as_strided(got[out._offset // 2:], q.shape,
                                            [2 * s for s in out.stride()])
    check_rows(inner, want, bound, rows)
    assert np.array_equal(inner[..., r:], q[..., r:])
    inner[:] = 0
    assert np.array_equal(got, out_flat)  # nothing beside the rows

    turned, bound = oracle.rotate(oracle.from_bits(k, rows), positions, rotary.frequencies, layout,
                                  factor)
    keep = (slots >= 0) & (slots < nb * bs)
    at = slots[keep]
    mine = oracle.Pages(nb, bs, heads, dim, kind, head_major, rows,
                        pages.segment - oracle.Pages(nb, bs, heads, dim, kind).segment,
                        pages.blocks_first)
    mine.bytes = dev.bytes()
    b, t = at // bs, at % bs
    if kind in oracle.LARGEST:
        check_codes(mine, 0, at, turned[keep], bound[keep])
    else:
        held = mine.values()[0, b, t]
        check_rows(held, turned[keep], bound[keep], rows)
        assert np.array_equal(held[..., r:], k[keep][..., r:])
    # V as written, all else untouched.
    pages.set(slots, k, v)
    pages.values()[0, b, t] = mine.values()[0, b, t]
    if kind in oracle.LARGEST:
        pages.scales()[0, b, t] = mine.scales()[0, b, t]
    assert np.array_equal(mine.bytes, pages.bytes)
    rotary.close()


@pytest.mark.parametrize("strides", ["contiguous", "odd"])
@pytest.mark.parametrize("r,layout", [(128, "half"), (48, "interleaved"), (20, "half"),
                                      (90, "interleaved")])
def test_in_place(gpu, r, layout, strides):
    """Rows turned where they lie have the bits of those turned elsewhere, and back they are
    what they were, twice rounded."""
    rng = np.random.default_rng(r)
    x = values(rng, (37, 5, 128), "bf16")
    positions = rng.integers(0, 1 << 20, 37)
    rotary = RotaryPositions(r, layout=layout)
    here, _, _ = device_rows(x, strides, "bf16")
    there, _, _ = device_rows(np.zeros_like(x), "contiguous", "bf16")
    at = device_array(positions, "int64")
    rotary.rotate(here, there, at)
    rotary.rotate(here, here, at)
    synchronize()
    got = there.download().view(np.uint16).reshape(x.shape)

    def rows_of(a):
        return np.lib.stride_tricks.as_strided(a.buffer.download().view(np.uint16), x.shape,
                                               [2 * s for s in a.stride()]).copy()

    assert np.array_equal(rows_of(here), got)
    want, bound = oracle.rotate(oracle.from_bits(x, "bf16"), positions, rotary.frequencies, layout)
    check_rows(got, want, bound, "bf16")
    rotary.rotate(here, here, device_array(-positions, "int64"))
    synchronize()
    want, bound = oracle.rotate(oracle.from_bits(got, "bf16"), -positions, rotary.frequencies,
                                layout)
    check_rows(rows_of(here), want, bound, "bf16")


def test_far_and_negative_positions(gpu):
    """The angle of a position as far as 2^32, and of its negative, is as exact as of a near one."""
    rng = np.random.default_rng(9)
    positions = np.concatenate([[0, 1, -1, (1 << 31) - 1, 1 << 31, -(1 << 31), (1 << 32) - 1],
                                rng.integers(-(1 << 32) + 1, 1 << 32, 57)])
    x = values(rng, (len(positions), 3, 64), "fp16")
    for layout in ("half", "interleaved"):
        # 1 / 8 of a turn a position, and none, among ordinary ones.
        f = [10000.0 ** (-i / 32) for i in range(30)] + [np.pi / 4, 0.0]
        rotary = RotaryPositions(64, layout=layout, frequencies=f)
        rows, _, _ = device_rows(x, "contiguous", "fp16")
        out, _, _ = device_rows(x, "contiguous", "fp16")
        rotary.rotate(rows, out, device_array(positions, "int64"))
        synchronize()
        got = out.download().view(np.uint16).reshape(x.shape)
        want, bound = oracle.rotate(oracle.from_bits(x, "fp16"), positions, f, layout)
        check_rows(got, want, bound, "fp16")


def test_position_0_is_write(gpu):
    """At position 0 nothing turns: the pages have the bytes that ``write`` leaves."""
    rng = np.random.default_rng(4)
    rotary = RotaryPositions(128)
    for kind in ("bf16", "e4m3", "int8"):
        k, v = values(rng, (40, 8, 128), "bf16"), values(rng, (40, 8, 128), "bf16")
        slots = rng.permutation(80).astype(np.int64)[:40]
        both = []
        for turned in (False, True):
            dev = DevicePages(oracle.Pages(5, 16, 8, 128, kind))
            kd, _, _ = device_rows(k)
            vd, _, _ = device_rows(v)
            at = device_array(slots, "int64")
            if turned:
                dev.cache.write_rotated(None, None, kd, vd, device_array(np.zeros(40, np.int64),
                                                                         "int64"), at, rotary)
            else:
                dev.cache.write(kd, vd, at)
            synchronize()
            both.append(dev.bytes())
        assert np.array_equal(*both)


@pytest.mark.parametrize("kind", ["bf16", "e4m3", "int8"])
def test_odd_values(gpu, kind):
    """Infinities and NaN of a key spoil their pair (16 bits) or their row (codes), nothing else;
    tiny rows keep scales that hold."""
    rng = np.random.default_rng(5)
    k, v = values(rng, (8, 2, 64), "bf16"), values(rng, (8, 2, 64), "bf16")
    k[1, 0, 3] = 0x7f80
    k[2, 1, 40] = 0x7fc1
    k[3] = rng.integers(0, 4, (2, 64))  # the least subnormal numbers
    k[4] = 0x7f7f  # the largest: two of them reach infinity
    k[5] = rng.integers(0, 0x0880, (2, 64))  # up to 2^-110
    positions = np.array([5, 6, 7, 8, 12345, 9, 11, 0])
    dev = DevicePages(oracle.Pages(1, 16, 2, 64, kind))
    rotary = RotaryPositions(64)
    kd, _, _ = device_rows(k)
    vd, _, _ = device_rows(v)
    slots = np.arange(8)
    dev.cache.write_rotated(None, None, kd, vd, device_array(positions, "int64"),
                            device_array(slots, "int64"), rotary)
    synchronize()
    mine = oracle.Pages(1, 16, 2, 64, kind)
    mine.bytes = dev.bytes()
    want, bound = oracle.rotate(oracle.from_bits(k, "bf16"), positions, rotary.frequencies, "half")
    if kind == "bf16":
        got = oracle.from_bits(mine.values()[0, 0, :8], "bf16").astype(np.float64)
        spoilt = ~np.isfinite(want)
        assert spoilt.sum() == 4 and not np.isfinite(got[spoilt]).any()
        # A sum past the largest bf16 number, 2^128 (1 - 2^-9) from halfway on, is infinite.
        ok = ~spoilt & (np.abs(want) < 2.0 ** 128 * (1 - 2.0 ** -8))
        allowed = HALF["bf16"] * (np.abs(want) + bound) + bound + LEAST["bf16"]
        assert (np.abs(got - want)[ok] <= allowed[ok]).all()
        return
    spoilt = ~np.isfinite(want).all(-1) | (np.abs(want).max(-1) > 2.0 ** 128 * (1 - 2.0 ** -20))
    scales = mine.scales()[0, 0, :8]
    assert np.array_equal(np.isnan(scales), spoilt) and spoilt[1, 0] and spoilt[2, 1]
    assert (mine.values()[0, 0, :8][spoilt] == 0).all()
    # A scale under 2^-126 is held to 2^-149 only, and so are the products that are turned.
    held = oracle.decode(mine.values()[0, 0, :8], kind) * scales.astype(np.float64)[..., None]
    top = oracle.LARGEST[kind]
    for i in range(8):
        for h in range(2):
            if spoilt[i, h]:
                continue
            coarse = top * 2.0 ** -149 + 2.0 ** -147
            step = scales[i, h] / 2 if kind == "int8" else np.maximum(
                2.0 ** -4 * np.abs(want[i, h]), scales[i, h] * 2.0 ** -10)
            off = 2 * bound[i, h] + 2.0 ** -20 * np.abs(want[i, h]).max()
            assert (np.abs(held[i, h] - want[i, h]) <= step * (1 + 2.0 ** -8) + off + coarse).all()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("r", [2, 20, 32, 46])
def test_values_behind_the_turned_ones(gpu, r, layout):
    """They pass bit by bit, NaN of any payload included, and spoil no pair beside them."""
    rng = np.random.default_rng(r)
    x = values(rng, (9, 3, 64), "bf16")
    x[:, :, r:] = rng.integers(0x7f80, 0x8000, (9, 3, 64 - r)) | rng.integers(0, 2, (9, 3, 64 - r)) << 15
    positions = rng.integers(0, 10 ** 6, 9)
    rotary = RotaryPositions(r, layout=layout)
    xd, _, _ = device_rows(x)
    out, _, _ = device_rows(x)
    rotary.rotate(xd, out, device_array(positions, "int64"))
    pages = DevicePages(oracle.Pages(1, 16, 3, 64, "bf16"))
    pages.cache.write_rotated(None, None, xd, xd, device_array(positions, "int64"),
                              device_array(np.arange(9), "int64"), rotary)
    synchronize()
    got = out.download().view(np.uint16).reshape(9, 3, 64)
    mine = oracle.Pages(1, 16, 3, 64, "bf16")
    mine.bytes = pages.bytes()
    want, bound = oracle.rotate(oracle.from_bits(x[..., :r], "bf16"), positions, rotary.frequencies,
                                layout)
    for bits in (got, np.asarray(mine.values()[0, 0, :9])):
        assert np.array_equal(bits[..., r:], x[..., r:])
        check_rows(bits[..., :r], want, bound, "bf16")


def test_refusals(gpu):
    rotary = RotaryPositions(64)
    dev = DevicePages(oracle.Pages(2, 16, 2, 64, "bf16"))
    x = np.zeros((4, 2, 64), np.uint16)
    rows, _, _ = device_rows(x)
    other, _, _ = device_rows(x, rows="fp16")
    at = device_array(np.zeros(4, np.int64), "int64")
    wide, _, _ = device_rows(np.zeros((4, 2, 48), np.uint16))
    with pytest.raises(PegaFlowError, match="64 turned values of heads of 48"):
        rotary.rotate(wide, wide, at)
    with pytest.raises(PegaFlowError, match="one type"):
        rotary.rotate(rows, other, at)
    with pytest.raises(PegaFlowError, match="one type"):
        dev.cache.write_rotated(other, other, rows, rows, at, at, rotary)
    with pytest.raises(PegaFlowError, match="rows' own type"):
        dev.cache.write_rotated(None, None, other, other, at, at, rotary)
    short = DeviceArray((4, 2, 64), "bf16", DeviceBuffer(4 * 2 * 64 * 2), 0)
    short._strides = (1 << 20, 64, 1)
    with pytest.raises(PegaFlowError, match="not inside"):
        rotary.rotate(rows, short, at)
    overlapping = DeviceArray((4, 2, 64), "bf16", DeviceBuffer(1 << 12), 0, (32, 64, 1))
    with pytest.raises(PegaFlowError, match="overlap"):
        rotary.rotate(rows, overlapping, at)
    with pytest.raises(ValueError, match="positions"):
        rotary.rotate(rows, rows, device_array(np.zeros(3, np.int64), "int64"))
    with pytest.raises(ValueError, match="int64"):
        rotary.rotate(rows, rows, device_array(np.zeros(4, np.int32), "int32"))
    with pytest.raises(ValueError, match="together"):
        dev.cache.write_rotated(rows, None, rows, rows, at, at, rotary)
    rotary.close()
    with pytest.raises(PegaFlowError, match="null rotary"):
        rotary.rotate(rows, rows, at)
    # On a stream of its own, and of no rows.
    rotary = RotaryPositions(64)
    stream = Stream()
    rotary.rotate(rows, rows, at, stream=stream)
    stream.synchronize()
    none, _, _ = device_rows(np.zeros((0, 2, 64), np.uint16))
    rotary.rotate(none, none, device_array(np.zeros(0, np.int64), "int64"))
