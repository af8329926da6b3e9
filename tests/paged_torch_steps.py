"""Steps of a model runner with torch tensors, in a process of their own: torch comes first,
and the library then runs on torch's HIP runtime.  Run by tests/test_paged_torch_gpu.py."""

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from pegaflow_amd.paged_cache import (AttentionWorkspace, PagedKVCache,  # noqa: E402
                                      segment_bytes)
from pegaflow_amd.transfer import KVCacheRegistration  # noqa: E402

HEADS, GROUP, DIM, BS, BLOCKS = 2, 4, 128, 16, 300
CACHED = 2500
BLOCK_LIST = torch.randperm(BLOCKS, generator=torch.Generator().manual_seed(1))[:200].to("cuda")


class Step:
    """One token behind CACHED ones: its K and V written, attended and read back."""

    def __init__(self, kind):
        seg = segment_bytes(BS, HEADS, DIM, kind)
        self.layer = torch.zeros(2, BLOCKS, seg, dtype=torch.uint8, device="cuda")
        self.cache = PagedKVCache(KVCacheRegistration.create(
            self.layer.data_ptr(), self.layer.numel(), BLOCKS, seg, BLOCKS * seg, 2), BS, HEADS,
            DIM, kind)
        self.workspace = AttentionWorkspace()
        rows = dict(dtype=torch.bfloat16, device="cuda")
        self.x = torch.zeros(1, HEADS * (GROUP + 2), DIM, **rows)
        self.out = torch.zeros(1, HEADS * GROUP, DIM, **rows)
        self.k, self.v = (torch.zeros(1, HEADS, DIM, **rows) for _ in range(2))
        self.slots = torch.zeros(1, dtype=torch.int64, device="cuda")
        self.table = BLOCK_LIST.to(torch.int32)[None]
        self.lens = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.starts = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
        gen = torch.Generator(device="cuda").manual_seed(2)
        kv = torch.randn(2, CACHED, HEADS, DIM, device="cuda", generator=gen).to(torch.bfloat16)
        t = torch.arange(CACHED, device="cuda")
        self.cache.write(kv[0], kv[1], BLOCK_LIST[t // BS] * BS + t % BS)
        torch.cuda.synchronize()

    def set(self, i, x):
        self.x.copy_(x)
        self.slots.copy_(BLOCK_LIST[(CACHED + i) // BS, None] * BS + (CACHED + i) % BS)
        self.lens.fill_(CACHED + i + 1)

    def run(self):
        qkv = self.x * 0.5  # what a layer before would do
        q, k, v = qkv.split([HEADS * GROUP, HEADS, HEADS], 1)
        self.cache.write(k, v, self.slots)
        self.cache.attend(q, self.out, self.table, self.lens, self.starts, max_query_len=1,
                          workspace=self.workspace)
        self.cache.read(self.slots, self.k, self.v)

    def results(self):
        return [t.clone() for t in (self.out, self.k, self.v, self.layer)]


def main(kind):
    eager, side, captured = Step(kind), Step(kind), Step(kind)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    gen = torch.Generator(device="cuda").manual_seed(3)
    inputs = torch.randn(5, *eager.x.shape, device="cuda", generator=gen).to(torch.bfloat16)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured.run()
    for i, x in enumerate(inputs):
        eager.set(i, x)
        eager.run()
        want = eager.results()
        assert want[0].abs().sum() > 0
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            torch.cuda._sleep(20_000_000)  # the inputs come late
            side.set(i, x)
            side.run()
            got = side.results()
        stream.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got)), f"stream, step {i}"
        captured.set(i, x)
        graph.replay()
        got = captured.results()
        assert all(torch.equal(a, b) for a, b in zip(want, got)), f"graph, step {i}"
        print(f"{kind}: step {i}", flush=True)
    print("ok", flush=True)


if __name__ == "__main__":
    main(sys.argv[1])
