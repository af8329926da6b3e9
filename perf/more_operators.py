"""More operators on the paged cache, case by case: rotary positions with the write of
new tokens, forks of sequences, kept tokens moved together, and attention of a batch
that shares a long prefix.

A case is one call as a model runner makes it between the transfers that save and
restore the layers' blocks.  The layer tensors are the runner's, K and V segments of
``num_blocks`` blocks; the positions, slots, block tables, lengths and kept tokens are
what it holds for the step.  With ``own`` false the operators are computed in their
plain form, in 32 bits (angles in 64); with it true by the package.

``op`` of a case:
  * ``rotate``   one layer: new tokens' queries and keys are turned to their positions,
                 queries into a buffer, keys and values into the pages;
  * ``fork``     all layers: children of sequences get block tables of their own and
                 copies of their parents' last, part-filled blocks;
  * ``compact``  all layers: the tokens of a sequence that are kept move together, in
                 place or to other blocks;
  * ``shared``   one layer: new tokens of a batch of sequences attend over all pages of
                 their sequences, whose first tokens lie in the same blocks.

``kind`` is what the pages hold: ``rows`` (the rows' own type), ``e4m3`` or ``int8``.
"""

import math
import random

import torch

own = False

ROWS = {"bf16": torch.bfloat16, "fp16": torch.float16}
LARGEST = {"e4m3": 448.0, "int8": 127.0}


def _case(name, op, kind, rows, heads, dim, **more):
    c = {"op": op, "kind": kind, "rows": rows, "heads": heads, "dim": dim, "block_size": 16,
         "head_major": False, "mix": 0, **more}
    return {"name": name, **c} if name else c


def _rotate(name, kind, rows, heads, dim, *, group, tokens, context, seqs, rotary,
            layout="half", base=10000.0, scaling="none", factor=1.0, original=8192, **more):
    """``tokens`` new tokens a sequence at positions up to ``context`` + ``tokens``; the
    first ``rotary`` values of a head are turned."""
    return _case(name, "rotate", kind, rows, heads, dim, group=group, tokens=tokens,
                 context=context, seqs=seqs, rotary=rotary, layout=layout, base=base,
                 scaling=scaling, factor=factor, original=original, **more)


def _fork(name, kind, rows, heads, dim, *, layers, parents, children, context, **more):
    """``children`` of each of ``parents`` sequences of up to ``context`` tokens."""
    return _case(name, "fork", kind, rows, heads, dim, layers=layers, parents=parents,
                 children=children, context=context, **more)


def _compact(name, kind, rows, heads, dim, *, layers, seqs, tokens, kept, drafts, **more):
    """Of each sequence about ``kept`` tokens move together: of its last ``drafts``, in
    place, or (``drafts`` 0) of all its ``tokens``, to other blocks."""
    return _case(name, "compact", kind, rows, heads, dim, layers=layers, seqs=seqs,
                 tokens=tokens, kept=kept, drafts=drafts, **more)


def _shared(name, kind, rows, heads, dim, *, group, groups, seqs, shared, context, tokens=1,
            alone=0, **more):
    """``groups`` groups of ``seqs`` sequences in all that share up to ``shared`` tokens,
    each up to ``context`` cached tokens of its own and ``tokens`` new ones; ``alone``
    sequences more share nothing."""
    return _case(name, "shared", kind, rows, heads, dim, group=group, groups=groups, seqs=seqs,
                 shared=shared, context=context, tokens=tokens, alone=alone, **more)


def listed():
    return [
        # A decode step of five requests on a small model (12 heads of 64 in fp16), half of
        # a head turned.
        _rotate("rotate_5_tokens_fp16", "rows", "fp16", 12, 64, group=1, tokens=1, context=300,
                seqs=5, rotary=32, layout="interleaved"),
        # A decode step of a full batch, frequencies stretched for long contexts, 8-bit cache.
        _rotate("rotate_64_tokens_e4m3", "e4m3", "bf16", 8, 128, group=4, tokens=1,
                context=16000, seqs=64, rotary=128, base=500000.0, scaling="llama3", factor=8.0),
        # A whole prompt of 10,000 tokens.
        _rotate("rotate_10000_tokens", "rows", "bf16", 8, 128, group=4, tokens=10000, context=0,
                seqs=1, rotary=128, base=500000.0),
        # A request of a small model sampled four ways.
        _fork("fork_4_children_fp16", "rows", "fp16", 12, 64, layers=12, parents=1, children=4,
              context=300),
        # Eight searches that branch eightfold, 8-bit cache.
        _fork("fork_64_children_e4m3", "e4m3", "bf16", 8, 128, layers=32, parents=8, children=8,
              context=1000),
        # The accepted branches of 32 draft trees of 24 tokens.
        _compact("compact_32_drafts", "rows", "bf16", 8, 128, layers=32, seqs=32, tokens=200,
                 kept=4, drafts=24),
        # Half of a 5,000-token prefix that others hold too is dropped, the rest packed anew.
        _compact("compact_5000_tokens", "rows", "bf16", 8, 128, layers=32, seqs=1, tokens=5000,
                 kept=2500, drafts=0),
        # A decode step of eight short chats on a small model behind one instruction.
        _shared("shared_8_fp16", "rows", "fp16", 12, 64, group=1, groups=1, seqs=8, shared=1000,
                context=200, mix=1),
        # A decode step of a full batch of questions about one document of 10,000 tokens.
        _shared("shared_64_after_10000", "rows", "bf16", 8, 128, group=4, groups=1, seqs=64,
                shared=10000, context=500, mix=2),
        # Three tools' instructions, drafts of up to five tokens, a head-major int8 cache.
        _shared("shared_drafts_int8", "int8", "fp16", 8, 128, group=4, groups=3, seqs=29,
                shared=4100, context=701, tokens=5, alone=2, head_major=True, mix=3),
        # 64 chats behind one long instruction, on an 8-bit cache.
        _shared("shared_64_e4m3", "e4m3", "bf16", 8, 128, group=4, groups=1, seqs=64,
                shared=16000, context=2000, mix=4),
        # Many branches of one search over a long document.
        _shared("shared_256_after_30000", "rows", "bf16", 8, 128, group=4, groups=1, seqs=256,
                shared=30000, context=300, mix=5),
    ]


def draw(rng):
    """Any such call: 1 to 16,384 rotated tokens, forks and moves of up to 48 layers,
    prefixes of up to 32,768 tokens, head sizes 64 to 256, pages of 8 to 64 tokens, up to
    the work of the largest listed case."""
    op = rng.choice(("rotate", "fork", "compact", "shared", "shared"))
    kind = rng.choice(("rows", "e4m3", "int8"))
    rows = rng.choice(("bf16", "bf16", "fp16"))
    heads = rng.choice((1, 2, 4, 8, 12))
    group = rng.choice((1, 2, 3, 4, 5, 7, 8)) if heads <= 8 else 1
    dim = rng.choice((64, 80, 96, 128, 128, 128, 192, 256))
    other = {"block_size": rng.choice((8, 16, 16, 16, 32, 64)), "head_major": rng.random() < 0.3,
             "mix": rng.randrange(1 << 16)}
    per_token = 2 * heads * dim * 2  # bytes of K and V at 16 bits
    if op == "rotate":
        # A code of int8 next to a border may be either of two, so that codes are no whole
        # numbers to be equal: that kind is left to tests.
        kind = rng.choice(("rows", "e4m3"))
        seqs = rng.choice((1, 1, rng.randint(2, 64)))
        tokens = max(1, min(round(16384 ** rng.random()),
                            200_000_000 // (seqs * heads * (group + 1) * dim * 4)))
        return _rotate(None, kind, rows, heads, dim, group=group, tokens=tokens,
                       context=round(100_000 ** rng.random()), seqs=seqs,
                       rotary=rng.choice((dim, dim, dim // 2, 16 * rng.randint(1, dim // 16),
                                          2 * rng.randint(1, dim // 2))),
                       layout=rng.choice(("half", "half", "interleaved")),
                       base=rng.choice((10000.0, 500000.0)),
                       scaling=rng.choice(("none", "linear", "ntk", "llama3", "yarn")),
                       factor=rng.choice((2.0, 4.0, 8.0)), original=rng.choice((2048, 8192)),
                       **other)
    layers = rng.choice((1, 12, 32, round(48 ** rng.random())))
    if op == "fork":
        parents, children = round(16 ** rng.random()), round(8 ** rng.random())
        while layers * parents * children * other["block_size"] * per_token > 150_000_000:
            layers = (layers + 1) // 2
            children = (children + 1) // 2
        return _fork(None, kind, rows, heads, dim, layers=layers, parents=parents,
                     children=children, context=rng.randint(1, 2000), **other)
    if op == "compact":
        drafts = rng.choice((0, rng.randint(2, 64)))
        seqs = round(64 ** rng.random())
        tokens = max(drafts, round(8192 ** rng.random()))
        kept = rng.randint(1, max(1, drafts // 2 if drafts else tokens))
        while layers * seqs * (tokens + kept) * per_token > 900_000_000:
            if seqs > 1:
                seqs = (seqs + 1) // 2
            elif layers > 1:
                layers = (layers + 1) // 2
            else:
                tokens = (tokens + 1) // 2
                drafts, kept = min(drafts, tokens), min(kept, max(1, tokens // 2))
        return _compact(None, kind, rows, heads, dim, layers=layers, seqs=seqs, tokens=tokens,
                        kept=kept, drafts=drafts, **other)
    groups = rng.choice((1, 1, 1, 2, 3, 5))
    seqs = max(groups, round(256 ** rng.random()))
    tokens = rng.choice((1, 1, 1, 2, 5, 8))
    shared, context = round(32768 ** rng.random()), round(4096 ** rng.random())
    while True:  # within the largest case, and the plain form within memory
        pairs = seqs * heads * group * tokens * (shared + context)
        if (4 * dim * pairs <= 10 ** 11 and pairs <= 5 * 10 ** 8
                and (seqs * (context + tokens) + groups * shared) * heads * dim <= 3 * 10 ** 8):
            break
        if seqs > groups:
            seqs = max(groups, seqs // 2)
        shared, context = (shared + 1) // 2, (context + 1) // 2
    return _shared(None, kind, rows, heads, dim, group=group, groups=groups, seqs=seqs,
                   shared=shared, context=context, tokens=tokens, alone=rng.choice((0, 0, 1, 3)),
                   **other)


def _segment_bytes(c):
    """Bytes of one block's K (or V): values, then for 8-bit kinds the scales of each head
    and token, padded to 16."""
    n = c["block_size"] * c["heads"] * c["dim"]
    return 2 * n if c["kind"] == "rows" else -(-(n + 4 * c["block_size"] * c["heads"]) // 16) * 16


def _values(c, segments):
    """The values held in ``segments`` [..., num_blocks, bytes] as [..., num_blocks,
    block_size, heads, dim], a view."""
    bs, heads, dim = c["block_size"], c["heads"], c["dim"]
    if c["kind"] == "rows":
        values = segments.view(ROWS[c["rows"]])
    else:
        values = segments[..., :bs * heads * dim]
        values = values.view(torch.float8_e4m3fn if c["kind"] == "e4m3" else torch.int8)
    if c["head_major"]:
        return values.unflatten(-1, (heads, bs, dim)).transpose(-3, -2)
    return values.unflatten(-1, (bs, heads, dim))


def _scales(c, segments):
    """The scales held in ``segments`` as [..., num_blocks, block_size, heads], a view."""
    bs, heads = c["block_size"], c["heads"]
    at = bs * heads * c["dim"]
    scales = segments[..., at:at + 4 * bs * heads].view(torch.float32)
    return scales.unflatten(-1, (heads, bs)).transpose(-1, -2)


def _vectors(n, c, generator):
    """Rows of K or V as projections give them: a few channels run larger than the rest."""
    x = torch.randn((n, c["heads"], c["dim"]), device="cuda", generator=generator)
    channel = torch.randn((c["heads"], c["dim"]), device="cuda", generator=generator)
    return x.mul_(torch.exp(0.5 * channel))


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _shuffled(n, generator):
    return torch.randperm(n, device="cuda", generator=generator).to(torch.int32)


def _cache(c, segments):
    """What a runner makes once of a layer's tensor [2, num_blocks, bytes]."""
    from pegaflow_amd.paged_cache import PagedKVCache
    from pegaflow_amd.transfer import KVCacheRegistration
    nb, seg = segments.shape[1:]
    reg = KVCacheRegistration.create(segments.data_ptr(), segments.numel(), nb, seg, nb * seg, 2)
    return PagedKVCache(reg, c["block_size"], c["heads"], c["dim"],
                        c["rows"] if c["kind"] == "rows" else c["kind"],
                        head_major=c["head_major"])


def _encode(c, x):
    """Codes and scales of 32-bit rows."""
    scales = x.abs().amax(-1) / LARGEST[c["kind"]]
    codes = torch.where(scales[..., None] > 0, x / scales[..., None], 0.0)
    if c["kind"] == "int8":
        return codes.round().to(torch.int8), scales
    return codes.to(torch.float8_e4m3fn), scales


def _put(c, segments, k, v, slots):
    """32-bit rows of K and V into the pages."""
    block, offset = slots // c["block_size"], slots % c["block_size"]
    x = torch.stack((k, v))
    if c["kind"] == "rows":
        _values(c, segments)[:, block, offset] = x.to(ROWS[c["rows"]])
        return
    codes, scales = _encode(c, x)
    _scales(c, segments)[:, block, offset] = scales
    _values(c, segments).view(torch.uint8)[:, block, offset] = codes.view(torch.uint8)


# --- rotary positions, and the write ---------------------------------------------------


def _frequencies(c):
    """(radians a position of each pair, factor of the turned values)."""
    r, s, base, n0 = c["rotary"], c["factor"], c["base"], c["original"]
    i = torch.arange(r // 2, dtype=torch.float64)
    if c["scaling"] == "ntk" and r > 2:
        base = base * s ** (r / (r - 2))
    f = base ** (-2 * i / r)
    if c["scaling"] == "linear":
        return f / s, 1.0
    if c["scaling"] == "llama3":
        # Short waves stay, long ones are stretched, with a ramp between.
        turns = n0 * f / (2 * math.pi)  # over the original context
        keep = ((turns - 1) / (4 - 1)).clamp(0, 1)
        return keep * f + (1 - keep) * f / s, 1.0
    if c["scaling"] == "yarn":
        def index(turns):
            return r * math.log(n0 / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(index(32)), 0), min(math.ceil(index(1)), r - 1)
        ramp = ((i - low) / (high - low if high != low else 0.001)).clamp(0, 1)
        return f / s * ramp + f * (1 - ramp), 0.1 * math.log(s) + 1 if s > 1 else 1.0
    return f, 1.0


def _scaling(c):
    """The same for the package, by its names."""
    if c["scaling"] == "none":
        return None
    s = {"type": c["scaling"], "factor": c["factor"]}
    if c["scaling"] in ("llama3", "yarn"):
        s["original_max_position"] = c["original"]
    return s


def _prepare_rotate(c, generator):
    rng = random.Random(c["mix"])
    bs, n = c["block_size"], c["tokens"]
    total = c["seqs"] * n
    first = [c["context"]] + [rng.randint(0, c["context"]) for _ in range(c["seqs"] - 1)]
    positions = (_ints(first, torch.int64)[:, None] + torch.arange(n, device="cuda")).flatten()
    # Each sequence's new tokens in blocks of their own, from its place in the first.
    pages = [-(-(a % bs + n) // bs) for a in first]
    used = sum(pages)
    num_blocks = used + used // 4 + 3
    order = _shuffled(num_blocks, generator).to(torch.int64)
    at = _ints([sum(pages[:i]) * bs + a % bs for i, a in enumerate(first)], torch.int64)
    at = (at[:, None] + torch.arange(n, device="cuda")).flatten()
    rows = ROWS[c["rows"]]
    q_heads = c["heads"] * c["group"]
    # One projection's output.
    qkv = torch.randn((total, q_heads + 2 * c["heads"], c["dim"]), device="cuda",
                      generator=generator).to(rows)
    qkv[:, q_heads:q_heads + c["heads"]] = _vectors(total, c, generator)
    q, k, v = qkv.split([q_heads, c["heads"], c["heads"]], 1)
    f, factor = _frequencies(c)
    segments = torch.zeros((2, num_blocks, _segment_bytes(c)), dtype=torch.uint8, device="cuda")
    s = {"segments": segments, "q": q, "k": k, "v": v, "positions": positions,
         "slots": order[at // bs] * bs + at % bs, "frequencies": f.cuda(), "factor": factor,
         "q_out": torch.empty((total, q_heads, c["dim"]), dtype=rows, device="cuda")}
    if own:
        from pegaflow_amd.paged_cache import RotaryPositions
        s["cache"] = _cache(c, segments)
        s["rotary"] = RotaryPositions(c["rotary"], base=c["base"], layout=c["layout"],
                                      scaling=_scaling(c))
    return s


def _turned(c, s, x):
    """Rows in 32 bits, turned to their positions."""
    r = c["rotary"]
    angle = (s["positions"].double()[:, None] * s["frequencies"])[:, None]
    cos, sin = (angle.cos() * s["factor"]).float(), (angle.sin() * s["factor"]).float()
    y = x.float()
    if c["layout"] == "half":
        a, b = y[..., :r // 2], y[..., r // 2:r]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = y[..., 0:r:2], y[..., 1:r:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((turned, y[..., r:]), -1)


def _run_rotate(c, s):
    if own:
        s["cache"].write_rotated(s["q"], s["q_out"], s["k"], s["v"], s["positions"], s["slots"],
                                 s["rotary"])
    else:
        s["q_out"].copy_(_turned(c, s, s["q"]))
        _put(c, s["segments"], _turned(c, s, s["k"]), s["v"].float(), s["slots"])
    held = {"q": s["q_out"], "values": _values(c, s["segments"])}
    if c["kind"] != "rows":
        held["scales"] = _scales(c, s["segments"])
    return held


def _exact_rotate(c, s):
    r = c["rotary"]
    turn = torch.polar(torch.full_like(s["frequencies"], s["factor"]).expand(len(s["slots"]), -1),
                       torch.outer(s["positions"].double(), s["frequencies"]))[:, None]

    def turned(x):
        x = x.double()
        if c["layout"] == "half":
            z = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous()) * turn
            x[..., :r // 2], x[..., r // 2:r] = z.real, z.imag
        else:
            z = torch.complex(x[..., 0:r:2].contiguous(), x[..., 1:r:2].contiguous()) * turn
            x[..., 0:r:2], x[..., 1:r:2] = z.real, z.imag
        return x

    both = torch.stack((turned(s["k"]), s["v"].double()))
    at = (slice(None), s["slots"] // c["block_size"], s["slots"] % c["block_size"])
    held = torch.zeros(_values(c, s["segments"]).shape, dtype=torch.float64, device="cuda")
    out = {"q": turned(s["q"]), "values": held}
    if c["kind"] == "rows":
        held[at] = both
        return out
    out["scales"] = torch.zeros(held.shape[:-1], dtype=torch.float64, device="cuda")
    out["scales"][at] = torch.linalg.vector_norm(both, ord=math.inf, dim=-1) / LARGEST[c["kind"]]
    held[at] = both / out["scales"][at][..., None].clamp(min=1e-300)
    return out


# --- forks, and moves of kept tokens ---------------------------------------------------


def _layers(c, num_blocks, generator):
    """All layers' tensors [layers, 2, num_blocks, bytes], filled with any bits: these
    operators move them as they are."""
    shape = (c["layers"], 2, num_blocks, _segment_bytes(c))
    return torch.randint(0, 256, shape, dtype=torch.uint8, device="cuda", generator=generator)


def _paged_layers(c, segments):
    from pegaflow_amd.paged_cache import PagedLayers
    return PagedLayers([_cache(c, layer) for layer in segments])


def _prepare_fork(c, generator):
    rng = random.Random(c["mix"])
    bs, parents = c["block_size"], c["parents"]
    lens = [c["context"]] + [rng.randint(1, c["context"]) for _ in range(parents - 1)]
    width = -(-c["context"] // bs) + 1
    new = parents * c["children"]
    # Parents hold many of their blocks together; their last ones are their own.
    num_blocks = min(parents * width, 2 * parents + 32) + new
    order = _shuffled(num_blocks, generator)
    table = order[torch.randint(parents, num_blocks - new, (parents, width), device="cuda",
                                generator=generator)]
    table[torch.arange(parents, device="cuda"), _ints(lens).long() // bs] = order[:parents]
    segments = _layers(c, num_blocks, generator)
    s = {"segments": segments, "table": table.contiguous(), "lens": _ints(lens),
         "parents": torch.arange(parents, device="cuda").repeat_interleave(
             c["children"]).to(torch.int32),
         "new_blocks": order[num_blocks - new:].contiguous(),
         "out_table": torch.zeros((new, width), dtype=torch.int32, device="cuda")}
    if own:
        s["layers"] = _paged_layers(c, segments)
    return s


def _run_fork(c, s):
    if own:
        s["layers"].fork(s["table"], s["lens"], s["parents"], s["new_blocks"], s["out_table"])
    else:
        parents, new = s["parents"].long(), s["new_blocks"].long()
        s["out_table"].copy_(s["table"][parents])
        page = s["lens"][parents].long() // c["block_size"]
        child = torch.arange(len(parents), device="cuda")
        last = s["out_table"][child, page].long()
        s["out_table"][child, page] = s["new_blocks"]
        # A parent that ends with its block leaves nothing to copy.
        last = torch.where(s["lens"][parents] % c["block_size"] > 0, last, new)
        for layer in s["segments"]:
            layer[:, new] = layer[:, last]
    return {"segments": s["segments"].view(torch.int32), "table": s["out_table"]}


def _prepare_compact(c, generator):
    rng = random.Random(c["mix"])
    bs, seqs, drafts = c["block_size"], c["seqs"], c["drafts"]
    kept, counts, first, lens = [], [], [], []
    for i in range(seqs):
        n = c["tokens"] if i == 0 else rng.randint(max(drafts, (c["tokens"] + 1) // 2), c["tokens"])
        if drafts:
            # The accepted branch lies behind the ones that were drafted before it.
            count = rng.randint(1, min(c["kept"], drafts // 2))
            at = sorted(rng.sample(range(n - drafts + count, n), count))
            first.append(n - drafts)
        else:
            count = min(c["kept"], n)
            at = sorted(rng.sample(range(n), count))
            first.append(0)
        kept += at
        counts.append(count)
        lens.append(n)
    pages = [-(-n // bs) for n in lens]
    out_pages = [0 if drafts else -(-n // bs) for n in counts]
    used = sum(pages) + sum(out_pages)
    num_blocks = used + used // 8 + 3
    order = _shuffled(num_blocks, generator)
    width = max(pages)

    def tables(sizes, base):
        starts = _ints([base + sum(sizes[:i]) for i in range(seqs)], torch.int64)
        at = starts[:, None] + torch.arange(width, device="cuda")
        inside = torch.arange(width, device="cuda") < _ints(sizes, torch.int64)[:, None]
        return torch.where(inside, order[at.clamp(max=num_blocks - 1)], -1).contiguous()

    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    segments = _layers(c, num_blocks, generator)
    table = tables(pages, 0)
    s = {"segments": segments, "table": table, "kept": _ints(kept), "starts": _ints(starts),
         "first": _ints(first), "out_table": table if drafts else tables(out_pages, sum(pages)),
         "out_lens": torch.zeros(seqs, dtype=torch.int32, device="cuda"), "most": max(counts)}
    if own:
        s["layers"] = _paged_layers(c, segments)
    return s


def _run_compact(c, s):
    if own:
        s["layers"].compact(s["table"], s["kept"], s["starts"], first=s["first"],
                            out_table=s["out_table"], out_lens=s["out_lens"], max_kept=s["most"])
    else:
        bs = c["block_size"]
        starts, kept = s["starts"].long(), s["kept"].long()
        j = torch.arange(len(kept), device="cuda")
        seq = torch.searchsorted(starts[1:], j, right=True)
        to = s["first"].long()[seq] + j - starts[seq]
        a = (s["table"][seq, kept // bs].long(), kept % bs)
        b = (s["out_table"][seq, to // bs].long(), to % bs)
        for layer in s["segments"]:
            values = _values(c, layer)
            if c["kind"] != "rows":
                scales = _scales(c, layer).view(torch.int32)
                scales[:, b[0], b[1]] = scales[:, a[0], a[1]]
                values = values.view(torch.uint8)
            values[:, b[0], b[1]] = values[:, a[0], a[1]]
        s["out_lens"].copy_(s["first"] + (starts[1:] - starts[:-1]).to(torch.int32))
    return {"segments": s["segments"].view(torch.int32), "lens": s["out_lens"]}


# --- attention behind shared prefixes --------------------------------------------------


def _batch(c):
    """(sequences of each group, shared tokens of each group, cached tokens of its own and
    new ones of each sequence)."""
    rng = random.Random(c["mix"])
    cuts = sorted(rng.sample(range(1, c["seqs"]), c["groups"] - 1)) if c["groups"] > 1 else []
    sizes = [b - a for a, b in zip([0] + cuts, cuts + [c["seqs"]])]
    bs = c["block_size"]
    shared = [c["shared"] // bs * bs]
    shared += [rng.randint(0, c["shared"]) // bs * bs for _ in sizes[1:]]
    n = c["seqs"] + c["alone"]
    cached = [c["context"]] + [rng.randint(0, c["context"]) for _ in range(n - 1)]
    new = [c["tokens"]] + [rng.randint(1, c["tokens"]) for _ in range(n - 1)]
    return sizes, shared, cached, new


def _prefix_of(c):
    """Shared tokens of each sequence."""
    sizes, shared, _, _ = _batch(c)
    return [n for size, n in zip(sizes, shared) for _ in range(size)] + [0] * c["alone"]


def _prepare_shared(c, generator):
    bs = c["block_size"]
    sizes, shared, cached, new = _batch(c)
    prefix = _prefix_of(c)
    seqs = len(new)
    lens = [p + a + b for p, a, b in zip(prefix, cached, new)]
    width = max(-(-n // bs) for n in lens)
    own_pages = [-(-(a + b) // bs) for a, b in zip(cached, new)]
    used = sum(n // bs for n in shared) + sum(own_pages)
    num_blocks = used + used // 8 + 3
    order = _shuffled(num_blocks, generator)
    rows, at = [], sum(n // bs for n in shared)
    shared_at = [sum(n // bs for n in shared[:g]) for g in range(len(shared))]
    group_of = [g for g, size in enumerate(sizes) for _ in range(size)] + [0] * c["alone"]
    slots = []  # of every token that the cache holds, once
    for g, n in enumerate(shared):
        t = torch.arange(n, device="cuda")
        slots.append(order[shared_at[g] + t // bs].long() * bs + t % bs)
    for i in range(seqs):
        g, n = group_of[i], prefix[i] // bs
        row = torch.zeros(width, dtype=torch.int32, device="cuda")
        row[:n] = order[shared_at[g]:shared_at[g] + n]
        row[n:n + own_pages[i]] = order[at:at + own_pages[i]]
        t = torch.arange(cached[i] + new[i], device="cuda")
        slots.append(order[at + t // bs].long() * bs + t % bs)
        at += own_pages[i]
        rows.append(row)
    slots = torch.cat(slots)
    segments = torch.zeros((2, num_blocks, _segment_bytes(c)), dtype=torch.uint8, device="cuda")
    k, v = (_vectors(len(slots), c, generator).to(ROWS[c["rows"]]) for _ in range(2))
    _put(c, segments, k.float(), v.float(), slots)
    del k, v
    q_heads, total = c["heads"] * c["group"], sum(new)
    width_q = (q_heads + 2 * c["heads"]) * c["dim"]
    qkv = torch.randn((total, width_q), device="cuda", generator=generator).to(ROWS[c["rows"]])
    ends, firsts = [0], [0]
    for n in new:
        ends.append(ends[-1] + n)
    for n in sizes:
        firsts.append(firsts[-1] + n)
    s = {"segments": segments, "table": torch.stack(rows), "lengths": _ints(lens),
         "starts": _ints(ends), "group_starts": _ints(firsts), "shared_lens": _ints(shared),
         "q": qkv[:, :q_heads * c["dim"]].view(total, q_heads, c["dim"]),
         "out": torch.empty((total, q_heads, c["dim"]), dtype=ROWS[c["rows"]], device="cuda"),
         "scale": 1 / math.sqrt(c["dim"]), "most_new": max(new), "longest": max(lens),
         "most_shared": max(shared), "most_own": max(a + b for a, b in zip(cached, new)),
         "batch": (sizes, shared), "prefix": _ints(prefix)}
    if own:
        from pegaflow_amd.paged_cache import AttentionWorkspace
        s["cache"] = _cache(c, segments)
        s["workspace"] = AttentionWorkspace()
    return s


def _held_rows(c, segments, slots):
    """K and V at ``slots`` in 32 bits: [2, *slots.shape, heads, dim]."""
    block, offset = slots // c["block_size"], slots % c["block_size"]
    if c["kind"] == "rows":
        return _values(c, segments)[:, block, offset].float()
    codes = _values(c, segments).view(torch.uint8)[:, block, offset]
    codes = codes.view(torch.float8_e4m3fn if c["kind"] == "e4m3" else torch.int8).float()
    return codes * _scales(c, segments)[:, block, offset][..., None]


def _plain_shared(c, s):
    total, q_heads, dim = s["q"].shape
    heads, group, bs = c["heads"], c["group"], c["block_size"]
    starts, lens = s["starts"].long(), s["lengths"].long()
    seqs = len(lens)
    row = torch.arange(total, device="cuda")
    seq = torch.searchsorted(starts[1:], row, right=True)
    index = row - starts[seq]
    new = starts[1:] - starts[:-1]
    x = s["q"].float() * s["scale"]
    # Scores over the sequences' own tokens, of a padded batch.
    q = torch.zeros((seqs, s["most_new"], q_heads, dim), device="cuda")
    q[seq, index] = x
    q = q.view(seqs, -1, heads, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs, heads, -1, dim)
    j = torch.arange(s["most_own"], device="cuda")
    t = s["prefix"].long()[:, None] + j
    page = (t // bs).clamp(max=s["table"].shape[1] - 1)
    k, v = _held_rows(c, s["segments"], s["table"].long().gather(1, page) * bs + t % bs)
    z = q @ k.permute(0, 2, 3, 1).contiguous()
    z = z.view(seqs, heads, -1, group, len(j)).permute(0, 2, 1, 3, 4)[seq, index]
    p = (lens - new)[seq] + index
    hidden = t[seq] > p[:, None]  # [rows, own tokens]
    z = z.masked_fill(hidden[:, None, None], -math.inf)  # [rows, heads, group, own tokens]
    m = z.amax(-1)
    # Scores over the shared ones, group by group.
    parts, first = [], 0
    for size, shared in zip(*s["batch"]):
        if shared:
            t = torch.arange(shared, device="cuda")
            kp, vp = _held_rows(c, s["segments"], s["table"][first, t // bs].long() * bs + t % bs)
            mine = (seq >= first) & (seq < first + size)
            qp = (x * mine[:, None, None]).view(total, heads, group, dim).permute(1, 0, 2, 3)
            zp = qp.reshape(heads, -1, dim) @ kp.permute(1, 2, 0).contiguous()
            zp = zp.view(heads, total, group, shared).permute(1, 0, 2, 3)
            zp = torch.where(mine[:, None, None, None], zp, -math.inf)
            m = torch.maximum(m, zp.amax(-1))
            parts.append((zp, vp))
        first += size
    w = torch.exp(z - m[..., None])
    l = w.sum(-1)
    padded = torch.zeros((seqs, s["most_new"], heads, group, len(j)), device="cuda")
    padded[seq, index] = w
    padded = padded.permute(0, 2, 1, 3, 4).reshape(seqs, heads, -1, len(j))
    o = padded @ v.permute(0, 2, 1, 3).contiguous()
    o = o.view(seqs, heads, -1, group, dim).permute(0, 2, 1, 3, 4)[seq, index]
    for zp, vp in parts:
        w = torch.exp(zp - m[..., None])
        l += w.sum(-1)
        w = w.permute(1, 0, 2, 3).reshape(heads, total * group, -1)
        op = w @ vp.permute(1, 0, 2).contiguous()
        o += op.view(heads, total, group, dim).permute(1, 0, 2, 3)
    s["out"].copy_((o / l[..., None]).reshape(total, q_heads, dim))


def _run_shared(c, s):
    if own:
        s["cache"].attend_shared(s["q"], s["out"], s["table"], s["lengths"], s["starts"],
                                 s["group_starts"], s["shared_lens"], scale=s["scale"],
                                 max_shared_len=s["most_shared"], max_own_len=s["most_own"],
                                 max_query_len=s["most_new"], workspace=s["workspace"])
    else:
        _plain_shared(c, s)
    return s["out"]


def _exact_value(c, raw):
    """64-bit values of the raw bytes (8-bit kinds) or 16-bit values."""
    if c["kind"] == "rows":
        return raw.double()
    b = raw.long()
    if c["kind"] == "int8":
        return (b - 256 * (b >= 128)).double()
    mantissa, exponent = (b & 7).double(), (b >> 3) & 15
    size = torch.where(exponent > 0, (8 + mantissa) * torch.exp2((exponent - 10).double()),
                       mantissa * 2.0 ** -9)
    return torch.where(b >= 128, -size, size)


def _exact_sequence(c, segments, table, length, kv):
    """K (0) or V (1) of one sequence in 64 bits: [heads, length, dim]."""
    bs, heads, dim = c["block_size"], c["heads"], c["dim"]
    pages = segments[kv][table[:-(-length // bs)].long()]
    n = bs * heads * dim
    raw = pages.view(ROWS[c["rows"]]) if c["kind"] == "rows" else pages[:, :n]
    if c["head_major"]:
        raw = raw.reshape(-1, heads, bs, dim).transpose(0, 1)
    else:
        raw = raw.reshape(-1, bs, heads, dim).permute(2, 0, 1, 3)
    x = _exact_value(c, raw)
    if c["kind"] != "rows":
        scales = pages[:, n:n + 4 * bs * heads].contiguous().view(torch.float32)
        x = x * scales.view(-1, heads, bs).transpose(0, 1).double()[..., None]
    return x.reshape(heads, -1, dim)[:, :length]


def _exact_shared(c, s):
    """Each sequence by itself, over its whole block table."""
    _, _, _, new = _batch(c)
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    heads, group, dim = c["heads"], c["group"], c["dim"]
    for i, n in enumerate(new):
        first, length = int(s["starts"][i]), int(s["lengths"][i])
        k, v = (_exact_sequence(c, s["segments"], s["table"][i], length, kv) for kv in (0, 1))
        q = s["q"][first:first + n].double().view(n, heads, group, dim).permute(1, 0, 2, 3)
        z = torch.matmul(q.reshape(heads, n * group, dim), k.transpose(1, 2).contiguous())
        z = z.mul_(s["scale"]).view(heads, n, group, length)
        t = torch.arange(length, device="cuda")
        hidden = t > (length - n + torch.arange(n, device="cuda"))[:, None]
        z.masked_fill_(hidden[:, None], -math.inf)
        z.sub_(torch.logsumexp(z, -1, keepdim=True)).exp_()
        o = torch.matmul(z.view(heads, n * group, length), v.contiguous())
        out[first:first + n] = o.view(heads, n, group, dim).permute(1, 0, 2, 3).reshape(n, -1, dim)
    return out


PREPARE = {"rotate": _prepare_rotate, "fork": _prepare_fork, "compact": _prepare_compact,
           "shared": _prepare_shared}
RUN = {"rotate": _run_rotate, "fork": _run_fork, "compact": _run_compact, "shared": _run_shared}


def prepare(case, seed):
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    state = PREPARE[case["op"]](case, generator)
    state["case"] = case
    torch.cuda.synchronize()
    return state


def run(state):
    return RUN[state["case"]["op"]](state["case"], state)


def work(case):
    """Rows, positions and tables, and the pages' bytes of every token (of a fork: block)
    that moves or that a row attends to, once."""
    c = case
    held = 2 * c["heads"] * (2 * c["dim"] if c["kind"] == "rows" else c["dim"] + 4)
    if c["op"] == "rotate":
        n, q_heads = c["seqs"] * c["tokens"], c["heads"] * c["group"]
        return {"bytes": n * (held + 4 * c["heads"] * c["dim"] + 4 * q_heads * c["dim"] + 16),
                "flops": n * (q_heads + c["heads"]) * c["rotary"] * 3}
    if c["op"] == "fork":
        rng = random.Random(c["mix"])
        lens = [c["context"]] + [rng.randint(1, c["context"]) for _ in range(c["parents"] - 1)]
        n = sum(length % c["block_size"] > 0 for length in lens) * c["children"]
        row = 4 * (-(-c["context"] // c["block_size"]) + 1)
        return {"bytes": n * c["layers"] * 4 * _segment_bytes(c)
                + row * c["parents"] * (1 + c["children"]), "flops": 0}
    if c["op"] == "compact":
        rng = random.Random(c["mix"])
        moved = 0
        for i in range(c["seqs"]):
            drafts, kept = c["drafts"], c["kept"]
            n = c["tokens"] if i == 0 else rng.randint(max(drafts, (c["tokens"] + 1) // 2),
                                                       c["tokens"])
            if drafts:
                count = rng.randint(1, min(kept, drafts // 2))
                rng.sample(range(n - drafts + count, n), count)
            else:
                count = min(kept, n)
                rng.sample(range(n), count)
            moved += count
        return {"bytes": moved * (c["layers"] * 2 * held + 4), "flops": 0}
    sizes, shared, cached, new = _batch(c)
    prefix = _prefix_of(c)
    seen = sum(shared) + sum(cached) + sum(new)
    pairs = sum(n * (p + a) + n * (n + 1) // 2 for p, a, n in zip(prefix, cached, new))
    q_heads = c["heads"] * c["group"]
    return {"bytes": seen * held + 4 * sum(new) * q_heads * c["dim"],
            "flops": 4 * c["dim"] * q_heads * pairs}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotate":
        return _exact_rotate(case, s)
    if case["op"] == "shared":
        return _exact_shared(case, s)
    return None  # bits that move as they are: the plain form's have to be equal
