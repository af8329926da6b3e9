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
