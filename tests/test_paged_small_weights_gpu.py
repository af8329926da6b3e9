"""Attention whose outputs are made of many small weights beside one large one: what each is
rounded to for the product with V must not lose their sum."""

import numpy as np
import pytest

from oracle import paged as oracle
from test_paged_cache_gpu import Batch, workspace  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,rows", [("fp16", "fp16"), ("bf16", "bf16"), ("e4m3", "fp16"),
                                       ("int8", "fp16")])
@pytest.mark.parametrize("new,cached", [((1,), (30000,)), ((3,), (30000,)), ((40,), (30000,)),
                                        ((1, 40), (5000, 20000))], ids=str)
def test_one_token_takes_most_of_the_weight(gpu, workspace, kind, rows, new, cached):
    """A token whose V is 0 lies 15 to 20 above all others in natural units: the outputs are
    the others' share, some 1e-3 and less."""
    dim = 64
    b = Batch(new, cached, (kind, rows, 1, dim, 16, False), 1, seed=50)
    rng = np.random.default_rng(51)
    u = rng.choice([-1.0, 1.0], dim)  # q . k of a row below: its gap
    gaps = rng.uniform(15, 20, len(b.q))
    b.q = oracle.to_bits((u * gaps[:, None, None] / 4).astype(np.float32), rows)
    bs = b.pages.block_size
    for i, n in enumerate(b.lens):
        t = np.arange(n)
        k = np.zeros((n, 1, dim))
        k[5] = u / 2
        v = rng.uniform(0.5, 1.5, (n, 1, dim))
        v[5] = 0
        b.pages.set(b.table[i][t // bs].astype(np.int64) * bs + t % bs,
                    oracle.to_bits(k.astype(np.float32), rows),
                    oracle.to_bits(v.astype(np.float32), rows))
    b.dev.upload()
    for w in (None, workspace):
        b.check(*b.run(workspace=w))


@pytest.mark.parametrize("kind,rows", [("e4m3", "fp16"), ("int8", "fp16"), ("int8", "bf16"),
                                       ("fp16", "fp16")])
@pytest.mark.parametrize("new,cached", [((4,) * 90, (20,) * 90), ((300,), (0,))], ids=str)
def test_log_sum_exps_beside_small_values(gpu, workspace, kind, rows, new, cached):
    """V of 2^-60 does not show in the statistics of the scores."""
    b = Batch(new, cached, (kind, rows, 2, 16, 16, False), 2, seed=52, sharp=0.01)
    if kind in oracle.LARGEST:
        held = b.pages.scales()[1]
        held[np.isfinite(held)] = 2.0 ** -60
    b.dev.upload()
    for window in (1, 2, 3, 5):
        b.check(*b.run(workspace=workspace, window=window), window=window)


@pytest.mark.parametrize("rows", ["bf16", "fp16"])
def test_the_largest_weight_is_held_as_it_is(gpu, workspace, rows):
    """A token of a later tile lies 2^3.5 to 2^7.5 above the first ones and all others far below:
    its V is the output, but for the output's own rounding and a share of the first's."""
    dim, n, late = 64, 40, 200
    b = Batch((n,), (300,), (rows, rows, 1, dim, 16, False), 1, seed=53)
    rng = np.random.default_rng(54)
    u = rng.choice([-1.0, 1.0], dim)
    b.q = oracle.to_bits(np.repeat(u[None, None], n, 0).astype(np.float32), rows)
    bs, t = b.pages.block_size, np.arange(b.lens[0])
    v = rng.uniform(0.5, 1.5, (len(t), 1, dim)) * rng.choice([-1.0, 1.0], (len(t), 1, dim))
    for gap in np.linspace(3.5, 7.5, 9):
        # scale * q . k = 8 |k| along u: 0 for the token, -gap for the first, -40 for others.
        k = np.full(len(t), -40.0)
        k[5], k[late] = -gap, 0.0
        k = k * np.log(2) / (dim * b.scale)
        b.pages.set(b.table[0][t // bs].astype(np.int64) * bs + t % bs,
                    oracle.to_bits((k[:, None, None] * u).astype(np.float32), rows),
                    oracle.to_bits(v.astype(np.float32), rows))
        b.dev.upload()
        want = oracle.attend(b.pages, b.q, rows, b.table, b.lens, b.starts, b.scale)[0]
        for w in (None, workspace):
            got = oracle.from_bits(b.run(workspace=w)[0], rows).astype(np.float64)
            half = oracle.HALF_STEP[rows]
            # The first's weight is 2^-gap, but for its key's rounding, and rounded to half a step
            # of |V| <= 1.5; 2^-16 stands for the others and for 32-bit sums.
            bound = half * np.abs(want) + half * 2.0 ** -(gap - 0.25) * 1.5 + 2.0 ** -16
            assert (np.abs(got - want) <= bound).all(), gap
