"""The search of paged_more_torch_steps.py against attention's definition, output by output, in a
process of its own.  Run by tests/test_paged_more_bounds_gpu.py."""

import math
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from oracle import paged as oracle  # noqa: E402
from paged_more_torch_steps import (BLOCKS, BS, CHILDREN, DIM, DRAFTS, GROUP, HEADS, LAYERS,  # noqa: E402
                                    PROMPT, Search)
from pegaflow_amd.paged_cache import AttentionWorkspace  # noqa: E402

# Queries sharp enough that single tokens count, and drafts that are larger than the prompt.
SHARP, KEYS, VALUES = 6.0, 2.0, 8.0


def mistakes(table, lens):
    """(name, table, lengths, causal) of attention that leaves tokens out, or takes too many."""
    own = table.copy()
    own[:, PROMPT // BS:] = -1
    yield "without the own tokens", own, lens, True
    yield "without the drafts", table, lens - DRAFTS, False
    yield "without the mask", table, lens, False
    yield "each row without itself", table, lens - 1, True
    tile = table.copy()
    tile[:, 20:20 + 64 // BS] = -1
    yield "without a tile of the prompt", tile, lens, True
    mixed = table.copy()
    mixed[:, PROMPT // BS] = np.roll(table[:, PROMPT // BS], 1)
    yield "with the last tokens of another child", mixed, lens, True


def main(kind):
    search = Search(kind, AttentionWorkspace())
    gen = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(search.x.shape, device="cuda", generator=gen)
    q_heads = HEADS * GROUP
    x[:, :, :q_heads] *= SHARP
    x[:, :, q_heads:q_heads + HEADS] *= KEYS
    x[:, :, q_heads + HEADS:] *= VALUES
    search.set(x.to(torch.bfloat16), search.kept)
    search.layers.compact = lambda *args, **kw: None  # what the cache holds stays as attended
    search.run()
    table, lens = search.children.cpu().numpy(), search.lens.cpu().numpy()
    starts = search.starts.cpu().numpy()
    scale = 1 / math.sqrt(DIM)
    for i in range(LAYERS):
        q = (search.x[i] * 0.5)[:, :q_heads].contiguous()  # as run() has it
        search.rotary.rotate(q, q, search.positions)
        bits = q.view(torch.int16).cpu().numpy().view(np.uint16)
        pages = oracle.Pages(BLOCKS, BS, HEADS, DIM, kind)
        pages.bytes = search.memory[i].cpu().numpy()
        got = search.out[i].double().cpu().numpy()
        want, _, bound, _ = oracle.attend(pages, bits, "bf16", table, lens, starts, scale)
        off = np.abs(got - want) / bound
        assert off.max() <= 1, f"layer {i}: {off.max()}"
        for name, t, n, causal in mistakes(table, lens):
            wrong = oracle.attend(pages, bits, "bf16", t, n, starts, scale, causal)[0]
            seen = (np.abs(got - wrong) > bound).reshape(CHILDREN, -1).any(1)
            assert seen.all(), f"{name} would pass: {seen}"
        print(f"{kind}: layer {i}, {off.max():.3f} of the bound", flush=True)
    print("ok", flush=True)


if __name__ == "__main__":
    main(sys.argv[1])
