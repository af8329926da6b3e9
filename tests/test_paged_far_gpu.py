"""Rotary writes, forks, copies, moves of kept tokens and shared attention in layers of 9 GiB: the
same bits as in small ones."""

import numpy as np
import pytest

from pegaflow_amd.paged_cache import (SHARE_ANYWAY, PagedKVCache, PagedLayers, RotaryPositions,
                                      segment_bytes)
from pegaflow_amd.runtime import DeviceBuffer, synchronize
from pegaflow_amd.transfer import KVCacheRegistration
from test_paged_cache_gpu import device_array, device_rows, values, workspace  # noqa: F401

pytestmark = pytest.mark.gpu

BS, HEADS, GROUP, DIM, LAYERS = 16, 8, 4, 128, 2
PROMPT, CHILDREN, DRAFTS = 100, 3, 2


def int32(x):
    return device_array(np.asarray(x, np.int32), "int32")


def int64(x):
    return device_array(np.asarray(x, np.int64), "int64")


def life(kind, blocks, num_blocks, workspace, seed):
    """What a prompt's blocks (``blocks``, of a layer of ``num_blocks``) hold and answer after a
    fork, drafts, a copy and moves."""
    rng = np.random.default_rng(seed)
    blocks = np.asarray(blocks)
    seg = segment_bytes(BS, HEADS, DIM, kind)
    buffers = [DeviceBuffer(2 * num_blocks * seg) for _ in range(LAYERS)]
    caches = [PagedKVCache(KVCacheRegistration.create(b.ptr, b.nbytes, num_blocks, seg,
                                                      num_blocks * seg, 2), BS, HEADS, DIM, kind)
              for b in buffers]
    layers, rotary = PagedLayers(caches), RotaryPositions(DIM)
    zero = device_rows(np.zeros((12 * BS, HEADS, DIM), np.uint16))[0]
    everything = int64((blocks[:, None].astype(np.int64) * BS + np.arange(BS)).reshape(-1))
    for c in caches:
        c.write(zero, zero, everything)

    def write(table, sequences, first, n):
        at = first + np.arange(n)
        slots = np.concatenate([table[s][at // BS].astype(np.int64) * BS + at % BS
                                for s in sequences])
        out = []
        for c in caches:
            count = len(slots)
            q = device_rows(values(rng, (count, HEADS * GROUP, DIM), "bf16"))[0]
            k, v = (device_rows(values(rng, (count, HEADS, DIM), "bf16"))[0] for _ in range(2))
            c.write_rotated(q, q, k, v, int64(np.tile(at, len(sequences))), int64(slots), rotary)
            synchronize()
            out.append(q)
        return out

    prompt = np.concatenate([blocks[:7], [-1]])[None]
    write(prompt, [0], 0, PROMPT)
    children = device_array(np.zeros((CHILDREN, 8), np.int32), "int32")
    layers.fork(int32(prompt), int32([PROMPT]), int32([0] * CHILDREN), int32(blocks[7:10]), children)
    synchronize()
    table = children.download().view(np.int32).reshape(CHILDREN, 8)
    queries = write(table, range(CHILDREN), PROMPT, DRAFTS)
    answers = []
    for c, q in zip(caches, queries):
        out = device_rows(np.zeros((CHILDREN * DRAFTS, HEADS * GROUP, DIM), np.uint16))[0]
        c.attend_shared(q, out, children, int32([PROMPT + DRAFTS] * CHILDREN),
                        int32(np.arange(CHILDREN + 1) * DRAFTS), int32([0, CHILDREN]),
                        int32([PROMPT // BS * BS]), max_shared_len=SHARE_ANYWAY,
                        max_own_len=BS, max_query_len=DRAFTS, workspace=workspace)
        synchronize()
        answers.append(out.download())
    layers.copy_blocks(int32(blocks[6:7]), int32(blocks[10:11]))
    layers.compact(int32(table[:1]), int32([3, 50, 97, 101]), int32([0, 4]), first=int32([1]))
    layers.compact(int32(table[1:2]), int32([20, 99, 100]), int32([0, 3]),
                   out_table=int32(np.concatenate([blocks[11:], [-1] * 7])[None]))
    synchronize()
    for c in caches:
        k, v = (device_rows(np.zeros((12 * BS, HEADS, DIM), np.uint16))[0] for _ in range(2))
        c.read(everything, k, v)
        synchronize()
        answers += [k.download(), v.download()]
    layers.close()
    rotary.close()
    rank = {int(b): i for i, b in enumerate(blocks)}
    return [np.array([[rank.get(int(b), -1) for b in row] for row in table])] + answers


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_offsets_past_32_bits(gpu, workspace, kind):
    """Blocks on both sides of 4 GiB of a segment, the last one among them."""
    near = life(kind, np.arange(12)[::-1], 12, workspace, seed=1)
    nb = (9 << 30) // (2 * segment_bytes(BS, HEADS, DIM, kind))
    far = [nb - 1, nb - 2, nb // 2, nb - 40, 5, nb - 3, nb - 77, nb - 5, nb // 2 + 1, nb - 8, nb - 30,
           nb - 9]
    assert len(set(far)) == 12
    for a, b in zip(near, life(kind, far, nb, workspace, seed=1)):
        assert np.array_equal(a, b) and np.any(a)
