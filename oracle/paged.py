"""The paged-cache operators from their definitions, in numpy: 64 bits where values are
computed, the defined 32-bit steps where codes and scales are.

TEST INFRASTRUCTURE ONLY, as the rest of this package."""

import numpy as np

LARGEST = {"e4m3": 448.0, "int8": 127.0}
# Largest relative error of one rounding to a row type.
HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}


def to_bits(x, rows):
    """float32 values rounded to bf16 or fp16, as uint16."""
    x = np.asarray(x, np.float32)
    if rows == "fp16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16).view(np.uint16)
    b = np.ascontiguousarray(x).view(np.uint32)
    r = ((b.astype(np.uint64) + 0x7fff + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7fc0), r)


def from_bits(bits, rows):
    bits = np.asarray(bits, np.uint16)
    if rows == "fp16":
        return bits.view(np.float16).astype(np.float32)
    return (bits.astype(np.uint32) << 16).view(np.float32)


def _e4m3_table():
    c = np.arange(256)
    m, e = (c & 7).astype(np.float64), (c >> 3) & 15
    v = np.where(e > 0, (8 + m) * 2.0 ** (e - 10.0), m * 2.0 ** -9)
    v[(c & 127) == 127] = np.nan
    return np.where(c >= 128, -v, v)


E4M3 = _e4m3_table()


def to_e4m3(x):
    """Nearest code of each float32, ties to the even code; 448 < |x| < 464 give 448."""
    size = np.abs(np.asarray(x, np.float64))
    levels = E4M3[:127]
    hi = np.clip(np.searchsorted(levels, size), 0, 126)
    lo = np.maximum(hi - 1, 0)
    below, above = size - levels[lo], levels[hi] - size
    code = np.where(below < above, lo, np.where(below > above, hi, np.where(lo % 2 == 0, lo, hi)))
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def encode(x, kind):
    """(codes as uint8, scales) of float32 rows [..., dim]."""
    m = np.abs(x).max(-1)
    ok = np.isfinite(x).all(-1)
    with np.errstate(all="ignore"):
        s = (m * (np.float32(1) / np.float32(LARGEST[kind]))).astype(np.float32)
        q = np.where(s[..., None] > 0, x / s[..., None], np.float32(0)).astype(np.float32)
        q = np.where(ok[..., None], q, np.float32(0))
    codes = to_e4m3(q) if kind == "e4m3" else np.rint(q).astype(np.int8).view(np.uint8)
    zero = ~ok | (m == 0)
    codes[zero] = 0
    return codes, np.where(ok, s, np.float32(np.nan))


def decode(codes, kind):
    return E4M3[codes] if kind == "e4m3" else codes.view(np.int8).astype(np.float64)


class Pages:
    """A layer's blocks on the host: [2, num_blocks, segment bytes] (or blocks-first, K and
    V halves of each block)."""

    def __init__(self, num_blocks, block_size, heads, dim, kind, head_major=False, rows="bf16",
                 pad=0, blocks_first=False):
        self.num_blocks, self.block_size, self.heads, self.dim = num_blocks, block_size, heads, dim
        self.kind, self.head_major, self.blocks_first = kind, head_major, blocks_first
        self.rows = kind if kind in HALF_STEP else rows
        n = block_size * heads * dim
        self.codes = n if kind in LARGEST else 2 * n
        size = n + 4 * block_size * heads if kind in LARGEST else 2 * n
        self.segment = -(-size // 16) * 16 + pad
        shape = (num_blocks, 2, self.segment) if blocks_first else (2, num_blocks, self.segment)
        self.bytes = np.zeros(shape, np.uint8)

    def seg(self):
        return self.bytes.swapaxes(0, 1) if self.blocks_first else self.bytes

    def values(self):
        """The held values [2, num_blocks, block_size, heads, dim], uint8 or uint16, a view."""
        v = self.seg()[..., :self.codes]
        if self.kind not in LARGEST:
            v = v.view(np.uint16)
        if self.head_major:
            return v.reshape(2, self.num_blocks, self.heads, self.block_size, self.dim).swapaxes(2, 3)
        return v.reshape(2, self.num_blocks, self.block_size, self.heads, self.dim)

    def scales(self):
        at = self.codes
        s = self.seg()[..., at:at + 4 * self.block_size * self.heads].view(np.float32)
        return s.reshape(2, self.num_blocks, self.heads, self.block_size).swapaxes(2, 3)

    def set(self, slots, k, v):
        """Rows [n, heads, dim] as uint16 bits into the slots that exist."""
        keep = (slots >= 0) & (slots < self.num_blocks * self.block_size)
        b, t = slots[keep] // self.block_size, slots[keep] % self.block_size
        both = np.stack([k[keep], v[keep]])
        if self.kind not in LARGEST:
            _put(self, "values", b, t, both)
            return
        codes, scales = encode(from_bits(both, self.rows), self.kind)
        _put(self, "values", b, t, codes)
        _put(self, "scales", b, t, scales)

    def get(self, slots):
        """K and V at ``slots`` in 64 bits [2, n, heads, dim], and in the defined 32 bits."""
        b, t = slots // self.block_size, slots % self.block_size
        raw = self.values()[:, b, t]
        if self.kind not in LARGEST:
            x = from_bits(raw, self.rows)
            return x.astype(np.float64), x
        c, s = decode(raw, self.kind), self.scales()[:, b, t][..., None]
        with np.errstate(invalid="ignore"):
            return c * s, (c.astype(np.float32) * s).astype(np.float32)


def _put(pages, which, b, t, x):
    view = getattr(pages, which)()
    assert np.shares_memory(view, pages.bytes)
    view[:, b, t] = x


def attend(pages, q, rows, table, lens, starts, scale, causal=True, window=0, weights=None,
           every=1, fine=()):
    """(out, lse, bound, lse bound) in 64 bits of query bits [n, heads, dim]: bound is how far each output
    of a kernel may be off that holds scores, statistics and sums in 32 bits, rounds each weight
    to ``weights`` and the output to ``rows``.  Only every ``every``-th row is computed.
    Of the sequences in ``fine`` a weight is two such numbers, the second the rounding of the first.

    A weight's rounding and the errors below scale with A = sum w |v| / sum w.  A score's
    32-bit sum of dim products is off by (dim + 4) half-steps of sum |q k| scale at most, the
    weight's exponential by that and 2^-21; l and o are sums of n terms, each addition off by
    half a step (n in all; also those of a join), l's errors counted again in the quotient.
    A weight under fp16's normal range is off by half its smallest step instead, 2^-25, where
    2^12 stands for the largest weight: by 2^-37 of that; one that carries the scale of a code by
    2^-25 where the largest such scale is 2^11 or more, so its products by 2^-36 of that scale
    times the code."""
    n, q_heads, dim = q.shape
    group = q_heads // pages.heads
    out = np.zeros((n, q_heads, dim))
    lse = np.full((n, q_heads), -np.inf)
    bound, lse_bound = np.zeros((n, q_heads, dim)), np.zeros((n, q_heads))
    x = from_bits(q, rows).astype(np.float64)
    bs = pages.block_size
    u = 2.0 ** -24
    for i in range(len(lens)):
        a, e = starts[i], starts[i + 1]
        length = min(max(int(lens[i]), 0), table.shape[1] * bs)
        t = np.arange(length)
        block = table[i][t // bs]
        there = (block >= 0) & (block < pages.num_blocks)
        slots = np.where(there, block, 0).astype(np.int64) * bs + t % bs
        kv = pages.get(slots)[0]
        v_scale = pages.scales()[1, slots // bs, slots % bs] if pages.kind in LARGEST else None
        for r in range(a + -a % every, e, every):
            p = length - (e - a) + (r - a)
            see = there & ((t <= p) if causal else True)
            if window:
                see = see & (t > p - window)
            if not see.any():
                continue
            for h in range(q_heads):
                k, v = kv[0][see, h // group], kv[1][see, h // group]
                with np.errstate(all="ignore"):
                    z = scale * (k @ x[r, h])
                    dz = u * (dim + 4) * np.abs(scale) * (np.abs(k) @ np.abs(x[r, h])).max()
                    m = z.max()
                    w = np.exp(z - m)
                    l = w.sum()
                    out[r, h] = (w @ v) / l
                    lse[r, h] = m + np.log(l)
                    size = (w @ np.abs(v)) / l
                off = 2 * dz + 2.0 ** -20 + 2 * (len(z) + 8) * u
                step = HALF_STEP[weights or rows] ** (2 if i in fine else 1)
                bound[r, h] = size * (step + off) + (
                    HALF_STEP[rows] * np.abs(out[r, h]) + 2.0 ** -24)
                if (weights or rows) == "fp16":
                    least = 2.0 ** -37 * np.abs(v).sum(0)
                    if v_scale is not None:
                        s = v_scale[see, h // group].astype(np.float64)[:, None]
                        with np.errstate(all="ignore"):
                            codes = np.divide(np.abs(v), s, out=np.zeros_like(v), where=s > 0)
                            least = 2.0 ** -36 * s.max() * codes.sum(0)
                    bound[r, h] += least / l
                lse_bound[r, h] = dz + 2.0 ** -21 + (len(z) + 8) * u + 2.0 ** -22 * abs(lse[r, h])
    return out, lse, bound, lse_bound
