"""Attention over pages whose V holds infinities and NaN: they reach the rows that attend
their tokens, as what they are, and no others."""

import numpy as np
import pytest

from oracle import paged as oracle
from test_paged_cache_gpu import (FORMS, INF16, LLAMA, NAN16, Batch,  # noqa: F401
                                  workspace)

pytestmark = pytest.mark.gpu

E4M3_NAN = 0x7f
FP16_80 = ("fp16", "fp16", 2, 80, 8, True)


def put(b, seq, token, head, d, bits):
    """V's value d of a sequence's token and KV head."""
    bs = b.pages.block_size
    b.pages.values()[1, b.table[seq][token // bs], token % bs, head, d] = bits


def check(b, got, lse):
    """Batch.check, and every output that is not finite."""
    out, want_lse, bound, lse_bound = oracle.attend(
        b.pages, b.q, b.rows, b.table, b.lens, b.starts, b.scale,
        fine=np.flatnonzero(np.diff(b.starts) * b.group <= 16))
    x = oracle.from_bits(got, b.rows).astype(np.float64)
    fine = np.isfinite(out)
    assert not fine.all()
    assert np.array_equal(np.where(fine, 0, out), np.where(np.isfinite(x), 0, x), equal_nan=True)
    assert (np.abs(x - out)[fine] <= bound[fine]).all()
    assert (np.abs(lse - want_lse) <= lse_bound).all()


@pytest.mark.parametrize("form,group", [(LLAMA, 4), (FORMS[1], 1), (FORMS[2], 4), (FORMS[4], 5),
                                        (FP16_80, 3)], ids=str)
@pytest.mark.parametrize("new,cached", [((1, 1), (400, 390)), ((100, 30), (400, 350)),
                                        ((1,), (3000,)), ((40,), (3000,))], ids=str)
def test_beside_missing_blocks(gpu, workspace, form, group, new, cached):
    """Tokens 112 to 127 have no block: what the tokens beside them hold is attended still."""
    b = Batch(new, cached, form, group, seed=40)
    bs, heads = b.pages.block_size, b.pages.heads
    codes = b.kind in oracle.LARGEST
    for i in range(len(new)):
        put(b, i, 100, 0, 3, E4M3_NAN if codes else INF16[b.rows])
        put(b, i, 103, heads - 1, b.pages.dim - 1, E4M3_NAN if codes else NAN16[b.rows])
        b.table[i, 112 // bs:128 // bs] = (-1, b.pages.num_blocks)[i % 2]
    b.dev.upload()
    for w in (None, workspace):
        check(b, *b.run(workspace=w))


@pytest.mark.parametrize("sharp", [1.0, 20.0, 60.0])
@pytest.mark.parametrize("form,group", [(LLAMA, 4), (FORMS[1], 1), (FP16_80, 3)], ids=str)
@pytest.mark.parametrize("new,cached", [((1, 1), (400, 390)), ((100, 30), (400, 350)),
                                        ((3,), (3000,)), ((40,), (3000,))], ids=str)
def test_infinities_keep_their_sign(gpu, workspace, form, group, new, cached, sharp):
    """In tiles that every row attends whole: an infinity stays one however small its weight is,
    and only two of both signs, or a NaN, make NaN."""
    b = Batch(new, cached, form, group, seed=41, sharp=sharp)
    inf, minus = INF16[b.rows], INF16[b.rows] | 0x8000
    for i in range(len(new)):
        for token, d, bits in ((40, 0, inf), (75, 1, minus), (41, 2, inf), (300, 2, inf),
                               (42, 3, inf), (290, 3, minus), (220, 4, NAN16[b.rows]),
                               (43, 17, minus)):
            put(b, i, token, 0, d, bits)
    b.dev.upload()
    for w in (None, workspace):
        check(b, *b.run(workspace=w))


@pytest.mark.parametrize("bad", ["inf", "nan"])
@pytest.mark.parametrize("form,group", [(LLAMA, 4), (FORMS[2], 4), (FP16_80, 3)], ids=str)
@pytest.mark.parametrize("new,cached", [((1, 1), (400, 390)), ((100, 30), (400, 350))], ids=str)
def test_nothing_but_such_values(gpu, workspace, form, group, new, cached, bad):
    """Every value of V from a token on, in every head but the last."""
    b = Batch(new, cached, form, group, seed=42)
    codes = b.kind in oracle.LARGEST
    bits = E4M3_NAN if codes else INF16[b.rows] if bad == "inf" else NAN16[b.rows]
    for i, n in enumerate(b.lens):
        for token in range(150, int(n)):
            put(b, i, token, slice(0, b.pages.heads - 1), slice(None), bits)
    b.dev.upload()
    for w in (None, workspace):
        check(b, *b.run(workspace=w))
