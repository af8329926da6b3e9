"""A search over branches with torch tensors, in a process of its own: a prompt is turned and
written, forked into children, which draft tokens behind the shared prompt, attend over it
together, and keep the accepted ones.  Run by tests/test_paged_more_torch_gpu.py."""

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from pegaflow_amd.paged_cache import (AttentionWorkspace, PagedKVCache, PagedLayers,  # noqa: E402
                                      RotaryPositions, segment_bytes)
from pegaflow_amd.transfer import KVCacheRegistration  # noqa: E402

LAYERS, HEADS, GROUP, DIM, BS, BLOCKS = 2, 2, 4, 128, 16, 240
PROMPT, CHILDREN, DRAFTS = 1003, 6, 5
WIDTH = PROMPT // BS + 4
I32 = dict(dtype=torch.int32, device="cuda")


class Search:
    def __init__(self, kind, workspace):
        gen = torch.Generator(device="cuda").manual_seed(1)
        order = torch.randperm(BLOCKS, device="cuda", generator=gen).to(torch.int32)
        seg = segment_bytes(BS, HEADS, DIM, kind)
        self.memory = torch.zeros(LAYERS, 2, BLOCKS, seg, dtype=torch.uint8, device="cuda")
        self.caches = [PagedKVCache(KVCacheRegistration.create(
            m.data_ptr(), m.numel(), BLOCKS, seg, BLOCKS * seg, 2), BS, HEADS, DIM, kind)
            for m in self.memory]
        self.layers = PagedLayers(self.caches)
        self.rotary = RotaryPositions(DIM, base=500000.0, scaling={
            "type": "yarn", "factor": 4, "original_max_position": 512})
        self.workspace = workspace
        self.table = torch.full((1, WIDTH), -1, **I32)
        pages = -(-PROMPT // BS)
        self.table[0, :pages] = order[:pages]
        self.own = order[pages:pages + 3 * CHILDREN].view(CHILDREN, 3)
        self.prompt_len = torch.tensor([PROMPT], **I32)
        self.parents = torch.zeros(CHILDREN, **I32)
        self.children = torch.zeros(CHILDREN, WIDTH, **I32)
        rows = dict(dtype=torch.bfloat16, device="cuda")
        self.prompt = torch.randn(LAYERS, PROMPT, 2, HEADS, DIM, device="cuda",
                                  generator=gen).to(torch.bfloat16)
        self.x = torch.zeros(LAYERS, CHILDREN * DRAFTS, HEADS * (GROUP + 2), DIM, **rows)
        self.out = torch.zeros(LAYERS, CHILDREN * DRAFTS, HEADS * GROUP, DIM, **rows)
        self.kept = torch.zeros(CHILDREN * 2, **I32)  # two accepted drafts of each
        self.kept_starts = torch.arange(0, 2 * CHILDREN + 1, 2, **I32)
        self.first = torch.full((CHILDREN,), PROMPT, **I32)
        self.lens = torch.full((CHILDREN,), PROMPT + DRAFTS, **I32)
        self.starts = torch.arange(0, CHILDREN * DRAFTS + 1, DRAFTS, **I32)
        self.group_starts = torch.tensor([0, CHILDREN], **I32)
        self.shared = torch.tensor([PROMPT // BS * BS], **I32)
        self.new_lens = torch.zeros(CHILDREN, **I32)
        self.at = PROMPT + torch.arange(DRAFTS, device="cuda")
        self.positions = self.at.repeat(CHILDREN)

    def set(self, x, kept):
        self.x.copy_(x)
        self.kept.copy_(kept)

    def run(self):
        t = torch.arange(PROMPT, device="cuda")
        slots = self.table[0, t // BS].long() * BS + t % BS
        for cache, kv in zip(self.caches, self.prompt):
            cache.write_rotated(None, None, kv[:, 0], kv[:, 1], t, slots, self.rotary)
        self.layers.fork(self.table, self.prompt_len, self.parents, self.own[:, 0].contiguous(),
                         self.children)
        first = PROMPT // BS
        self.children[:, first + 1:first + 3] = self.own[:, 1:]
        slots = (self.children[:, self.at // BS].long() * BS + self.at % BS).flatten()
        for i, cache in enumerate(self.caches):
            qkv = self.x[i] * 0.5  # what a layer before would do
            q, k, v = qkv.split([HEADS * GROUP, HEADS, HEADS], 1)
            cache.write_rotated(q, q, k, v, self.positions, slots, self.rotary)
            cache.attend_shared(q, self.out[i], self.children, self.lens, self.starts,
                                self.group_starts, self.shared, max_shared_len=1 << 30,
                                max_own_len=BS + DRAFTS, max_query_len=DRAFTS,
                                workspace=self.workspace)
        self.layers.compact(self.children, self.kept, self.kept_starts, first=self.first,
                            out_lens=self.new_lens)

    def results(self):
        return [t.clone() for t in (self.out, self.children, self.new_lens, self.memory)]

    def check(self, before):
        """The last layer's outputs against attend's, whose bound is the same (2^-8 of the weighted
        mean of |v| for weights, as much for the output, twice), and the kept tokens' bytes."""
        q = (self.x[-1] * 0.5)[:, :HEADS * GROUP].contiguous()
        self.rotary.rotate(q, q, self.positions)
        want = torch.empty_like(self.out[-1])
        now = self.memory.clone()
        self.memory.copy_(before)
        self.caches[-1].attend(q, want, self.children, self.lens, self.starts,
                               max_query_len=DRAFTS, workspace=self.workspace)
        k = torch.empty(CHILDREN, 2, HEADS, DIM, dtype=torch.bfloat16, device="cuda")
        moved = []
        for memory, at in ((before, self.kept.view(CHILDREN, 2)),
                           (now, PROMPT + torch.arange(2, device="cuda").expand(CHILDREN, 2))):
            self.memory.copy_(memory)
            slots = self.children.gather(1, at.long() // BS).long() * BS + at % BS
            v = torch.empty_like(k)
            for cache in self.caches:
                cache.read(slots.flatten(), k.view(-1, HEADS, DIM), v.view(-1, HEADS, DIM))
                moved.append((k.clone(), v.clone()))
        self.memory.copy_(now)
        top = torch.cat([self.prompt[-1, :, 1].float().abs().amax()[None],
                         self.x[-1].float().abs().amax()[None]]).amax()
        assert (self.out[-1].float() - want.float()).abs().amax() <= 2.0 ** -6 * top
        for a, b in zip(moved[:LAYERS], moved[LAYERS:]):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and a[1].abs().sum() > 0
        assert self.new_lens.tolist() == [PROMPT + 2] * CHILDREN


def main(kind):
    workspace = AttentionWorkspace()
    eager, side = Search(kind, workspace), Search(kind, AttentionWorkspace())
    # Two captured searches share a workspace: their replays are ordered.
    together = AttentionWorkspace()
    captured = [Search(kind, together), Search(kind, together)]
    stream = torch.cuda.Stream()
    graphs = [torch.cuda.CUDAGraph() for _ in captured]
    gen = torch.Generator(device="cuda").manual_seed(3)
    inputs = []
    for _ in range(4):
        x = torch.randn(eager.x.shape, device="cuda", generator=gen).to(torch.bfloat16)
        kept = torch.stack([torch.randperm(DRAFTS - 1, device="cuda", generator=gen)[:2].sort()[0]
                            for _ in range(CHILDREN)]) + PROMPT + 1
        inputs.append((x, kept.flatten().to(torch.int32)))
    torch.cuda.synchronize()
    for search, graph in zip(captured, graphs):
        with torch.cuda.graph(graph):
            search.run()
    for i, x in enumerate(inputs):
        eager.set(*x)
        eager.run()
        want = eager.results()
        assert want[0].abs().sum() > 0
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            torch.cuda._sleep(20_000_000)  # the inputs come late
            side.set(*x)
            side.run()
            got = side.results()
        stream.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got)), f"stream, step {i}"
        for search, graph in zip(captured, graphs):
            search.set(*x)
            graph.replay()
        for search in captured:
            assert all(torch.equal(a, b) for a, b in zip(want, search.results())), f"graph, {i}"
        # Without the move, what the cache held before it.
        keep = eager.layers.compact
        eager.layers.compact = lambda *args, **kw: None
        eager.run()
        before = eager.memory.clone()
        eager.layers.compact = keep
        eager.run()
        eager.check(before)
        print(f"{kind}: step {i}", flush=True)
    print("ok", flush=True)


if __name__ == "__main__":
    main(sys.argv[1])
