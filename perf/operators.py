"""The paged cache's operators, case by case: rows of K and V written into a layer's
pages, read back from them, and attended over.

A case is one call for one layer, as a model runner makes it between the transfers
that save and restore the layer's blocks.  The layer tensor is the runner's, K and V
segments of ``num_blocks`` blocks; the slots, block tables and lengths are what it
holds for the step.  With ``own`` false the operators are computed in their plain
form, in 32 bits; with it true by the package.

``op`` of a case:
  * ``write``   K and V of new tokens into the pages, at 16 bits or as 8-bit codes with
                a scale for each token and head;
  * ``read``    the rows of cached tokens back at 16 bits;
  * ``attend``  new tokens of a batch of sequences over all pages of their sequences:
                chunks of a prompt, or one token each.

``kind`` is what the pages hold: ``rows`` (the rows' own type), ``e4m3`` or ``int8``.
"""

import math
import random

import torch

own = False

ROWS = {"bf16": torch.bfloat16, "fp16": torch.float16}
LARGEST = {"e4m3": 448.0, "int8": 127.0}


def _case(name, op, kind, rows, heads, dim, *, group=1, seqs=1, tokens=1, context=0, ragged=False,
          block_size=16, head_major=False, window=0, mix=0):
    """``seqs`` sequences of ``tokens`` new (or cached, for a read) tokens behind
    ``context`` cached ones; ``ragged``: those are the longest of a batch.  ``heads`` KV
    heads, each shared by ``group`` query heads."""
    c = {"op": op, "kind": kind, "rows": rows, "heads": heads, "dim": dim, "group": group,
         "seqs": seqs, "tokens": tokens, "context": context, "ragged": ragged,
         "block_size": block_size, "head_major": head_major, "window": window, "mix": mix}
    return {"name": name, **c} if name else c


def listed():
    return [
        # A decode step of five requests on a small model (12 heads of 64 in fp16).
        _case("write_5_tokens_fp16", "write", "rows", "fp16", 12, 64, seqs=5, context=300,
              ragged=True),
        # A decode step of a full batch: 64 tokens quantised into 64 different blocks.
        _case("write_64_tokens_e4m3", "write", "e4m3", "bf16", 8, 128, seqs=64, context=2000,
              ragged=True),
        # A whole prompt of 10,000 tokens quantised as it is written.
        _case("write_10000_tokens_int8", "write", "int8", "bf16", 8, 128, tokens=10000),
        # The last, part-filled block of a prefix read back.
        _case("read_9_tokens_e4m3", "read", "e4m3", "bf16", 8, 128, tokens=9),
        # A 10,000-token prefix read back at 16 bits.
        _case("read_10000_tokens_e4m3", "read", "e4m3", "bf16", 8, 128, tokens=10000),
        # One user's next token behind the 10,000-token prompt.
        _case("decode_1_after_10000", "attend", "rows", "bf16", 8, 128, group=4, context=10000),
        # A decode step of 32 chats on a small model without shared heads.
        _case("decode_32_fp16", "attend", "rows", "fp16", 12, 64, seqs=32, context=1000,
              ragged=True, mix=1),
        # A decode step of a full batch, prompts of up to 16,000 tokens, 8-bit cache.
        _case("decode_64_e4m3", "attend", "e4m3", "bf16", 8, 128, group=4, seqs=64,
              context=16000, ragged=True, mix=2),
        # A follow-up turn: 500 tokens behind a restored 10,000-token prefix in 8 bits.
        _case("chunk_500_after_10000_e4m3", "attend", "e4m3", "bf16", 8, 128, group=4,
              tokens=500, context=10000),
        # A step that mixes chunks of several prompts and single tokens, odd lengths.
        _case("chunks_mixed_int8", "attend", "int8", "fp16", 8, 128, group=4, seqs=9, tokens=701,
              context=4100, ragged=True, head_major=True, mix=3),
        # A prompt with no cached prefix.
        _case("prompt_8192", "attend", "rows", "bf16", 8, 128, group=4, tokens=8192),
        # A chunk of a long document.
        _case("chunk_2048_after_30000", "attend", "rows", "bf16", 8, 128, group=4, tokens=2048,
              context=30000),
    ]


def draw(rng):
    """Any such call: 1 to 16,384 new tokens, contexts up to 32,768, head sizes 64 to 256,
    pages of 8 to 64 tokens, up to the work of the largest listed case."""
    op = rng.choice(("write", "read", "attend", "attend", "attend"))
    kind = rng.choice(("rows", "e4m3", "int8"))
    rows = rng.choice(("bf16", "bf16", "fp16"))
    heads = rng.choice((1, 2, 4, 8, 12))
    group = rng.choice((1, 2, 3, 4, 5, 7, 8, 16)) if heads <= 8 else 1
    dim = rng.choice((64, 80, 96, 128, 128, 128, 192, 256))
    other = {"block_size": rng.choice((8, 16, 16, 16, 32, 64)), "head_major": rng.random() < 0.3,
             "mix": rng.randrange(1 << 16)}
    if op != "attend":
        seqs = rng.choice((1, 1, rng.randint(2, 64)))
        tokens = max(1, min(round(16384 ** rng.random()), 100_000_000 // (seqs * heads * dim)))
        return _case(None, op, kind, rows, heads, dim, seqs=seqs, tokens=tokens,
                     context=rng.randint(0, 2000) if op == "write" else 0,
                     ragged=seqs > 1, **other)
    window = rng.choice((0, 0, 0, round(2 ** rng.uniform(4, 12))))
    if rng.random() < 0.5:  # single tokens
        seqs, tokens = round(128 ** rng.random()), 1
    else:
        seqs, tokens = rng.choice((1, 1, 2, 5, 9)), round(8192 ** rng.random())
    context = round(32768 ** rng.random())
    while True:  # within the largest case, and the plain form within memory
        longest = tokens + context
        pairs = seqs * heads * group * tokens * longest
        if (4 * dim * pairs <= 10 ** 12 and pairs <= 2 * 10 ** 9
                and seqs * longest * heads * dim <= 10 ** 9):
            break
        if tokens > 1 and tokens * 8 > context:
            tokens = (tokens + 1) // 2
        else:
            context = context // 2
    return _case(None, op, kind, rows, heads, dim, group=group, seqs=seqs, tokens=tokens,
                 context=context, ragged=seqs > 1, window=window, **other)


def _lengths(c):
    """(new, cached) tokens of each sequence."""
    if not c["ragged"]:
        return [c["tokens"]] * c["seqs"], [c["context"]] * c["seqs"]
    rng = random.Random(c["mix"])
    new = [c["tokens"]] + [rng.randint(1, c["tokens"]) for _ in range(c["seqs"] - 1)]
    cached = [c["context"]] + [rng.randint(0, c["context"]) for _ in range(c["seqs"] - 1)]
    return new, cached


def _segment_bytes(c):
    """Bytes of one block's K (or V): values, then for 8-bit kinds the scales of each head
    and token, padded to 16."""
    n = c["block_size"] * c["heads"] * c["dim"]
    return 2 * n if c["kind"] == "rows" else -(-(n + 4 * c["block_size"] * c["heads"]) // 16) * 16


def _tables(c, generator):
    """Block tables of all sequences in a cache with a quarter of its blocks to spare."""
    new, cached = _lengths(c)
    pages = [-(-(a + b) // c["block_size"]) for a, b in zip(new, cached)]
    used = sum(pages)
    num_blocks = used + used // 4 + 3
    order = torch.randperm(num_blocks, device="cuda", generator=generator).to(torch.int32)
    width = max(pages)
    starts = torch.tensor([sum(pages[:i]) for i in range(len(pages))], device="cuda")
    at = starts[:, None] + torch.arange(width, device="cuda")
    table = order[at.clamp(max=used - 1)]
    valid = torch.arange(width, device="cuda") < torch.tensor(pages, device="cuda")[:, None]
    return torch.where(valid, table, 0).contiguous(), num_blocks


def _vectors(n, c, generator):
    """Rows of K or V as projections give them: a few channels run larger than the rest."""
    x = torch.randn((n, c["heads"], c["dim"]), device="cuda", generator=generator)
    channel = torch.randn((c["heads"], c["dim"]), device="cuda", generator=generator)
    return x.mul_(torch.exp(0.5 * channel))


def _values(c, segments):
    """The values held in ``segments`` [2, num_blocks, bytes] as [2, num_blocks, block_size,
    heads, dim], a view."""
    nb, bs, heads, dim = segments.shape[1], c["block_size"], c["heads"], c["dim"]
    if c["kind"] == "rows":
        values = segments.view(ROWS[c["rows"]])
    else:
        values = segments[..., :bs * heads * dim]
        values = values.view(torch.float8_e4m3fn if c["kind"] == "e4m3" else torch.int8)
    if c["head_major"]:
        return values.view(2, nb, heads, bs, dim).transpose(2, 3)
    return values.view(2, nb, bs, heads, dim)


def _scales(c, segments):
    """The scales held in ``segments`` as [2, num_blocks, block_size, heads], a view."""
    nb, bs, heads = segments.shape[1], c["block_size"], c["heads"]
    at = bs * heads * c["dim"]
    scales = segments[..., at:at + 4 * bs * heads].view(torch.float32)
    return scales.view(2, nb, heads, bs).transpose(2, 3)


def _slots(c, table, first, count):
    """Slots of ``count[i]`` tokens of each sequence from its token ``first[i]`` on."""
    seq = torch.tensor([i for i, n in enumerate(count) for _ in range(n)], device="cuda")
    pos = torch.cat([torch.arange(a, a + n, device="cuda") for a, n in zip(first, count)])
    bs = c["block_size"]
    return table[seq, pos // bs].to(torch.int64) * bs + pos % bs


def prepare(case, seed):
    c = case
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    new, cached = _lengths(c)
    table, num_blocks = _tables(c, generator)
    segments = torch.zeros((2, num_blocks, _segment_bytes(c)), dtype=torch.uint8, device="cuda")
    rows = ROWS[c["rows"]]
    total = sum(new)
    state = {"case": c, "segments": segments}
    if c["op"] == "write":
        # K and V as slices of one projection's output.
        qkv = torch.empty((total, 3, c["heads"], c["dim"]), dtype=rows, device="cuda")
        qkv[:, 1] = _vectors(total, c, generator)
        qkv[:, 2] = _vectors(total, c, generator)
        state.update(k=qkv[:, 1], v=qkv[:, 2], slots=_slots(c, table, cached, new))
    else:
        # The cache holds what writes of its tokens left.
        lengths = [a + b for a, b in zip(new, cached)]
        slots = _slots(c, table, [0] * len(lengths), lengths)
        k, v = (_vectors(sum(lengths), c, generator).to(rows) for _ in range(2))
        _plain_write(c, segments, k, v, slots)
        if c["op"] == "read":
            state.update(slots=slots, k=torch.empty_like(k), v=torch.empty_like(v))
        else:
            q_heads = c["heads"] * c["group"]
            width = (q_heads + 2 * c["heads"]) * c["dim"]
            qkv = torch.randn((total, width), device="cuda", generator=generator).to(rows)
            ends = [0]
            for n in new:
                ends.append(ends[-1] + n)
            state.update(
                q=qkv[:, :q_heads * c["dim"]].view(total, q_heads, c["dim"]),
                out=torch.empty((total, q_heads, c["dim"]), dtype=rows, device="cuda"),
                table=table, starts=torch.tensor(ends, dtype=torch.int32, device="cuda"),
                lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                longest=max(lengths), most_new=max(new), scale=1 / math.sqrt(c["dim"]))
    if own:
        # What a runner makes once: the layer's registration and page shape, and a
        # workspace for its stream.
        from pegaflow_amd.paged_cache import AttentionWorkspace, PagedKVCache
        from pegaflow_amd.transfer import KVCacheRegistration
        seg = _segment_bytes(c)
        reg = KVCacheRegistration.create(segments.data_ptr(), segments.numel(), num_blocks, seg,
                                         num_blocks * seg, 2)
        state["cache"] = PagedKVCache(reg, c["block_size"], c["heads"], c["dim"],
                                      c["rows"] if c["kind"] == "rows" else c["kind"],
                                      head_major=c["head_major"])
        if c["op"] == "attend":
            state["workspace"] = AttentionWorkspace()
    torch.cuda.synchronize()
    return state


def _plain_write(c, segments, k, v, slots):
    block, offset = slots // c["block_size"], slots % c["block_size"]
    values = _values(c, segments)
    x = torch.stack((k, v))
    if c["kind"] == "rows":
        values[:, block, offset] = x
        return
    x = x.float()
    scales = x.abs().amax(-1) / LARGEST[c["kind"]]
    codes = torch.where(scales[..., None] > 0, x / scales[..., None], 0.0)
    _scales(c, segments)[:, block, offset] = scales
    if c["kind"] == "int8":
        values[:, block, offset] = codes.round().to(torch.int8)
    else:
        values.view(torch.uint8)[:, block, offset] = codes.to(torch.float8_e4m3fn).view(torch.uint8)


def _plain_rows(c, segments, slots):
    """K and V at ``slots`` in 32 bits: [2, *slots.shape, heads, dim]."""
    block, offset = slots // c["block_size"], slots % c["block_size"]
    values = _values(c, segments)
    if c["kind"] == "rows":
        return values[:, block, offset].float()
    if c["kind"] == "e4m3":
        codes = values.view(torch.uint8)[:, block, offset].view(torch.float8_e4m3fn)
    else:
        codes = values[:, block, offset]
    return codes.float() * _scales(c, segments)[:, block, offset][..., None]


def _plain_attend(c, s):
    total, q_heads, dim = s["q"].shape
    heads, group, seqs = c["heads"], c["group"], c["seqs"]
    starts, lengths = s["starts"].long(), s["lengths"].long()
    new = starts[1:] - starts[:-1]
    # Rows of the packed batch as (sequence, index) of a padded one.
    row = torch.arange(total, device="cuda")
    seq = torch.searchsorted(starts[1:], row, right=True)
    index = row - starts[seq]
    q = torch.zeros((seqs, s["most_new"], q_heads, dim), device="cuda")
    q[seq, index] = s["q"].float()
    q = q.view(seqs, -1, heads, group, dim).permute(0, 2, 1, 3, 4)
    t = torch.arange(s["longest"], device="cuda")
    slots = s["table"][:, t // c["block_size"]].long() * c["block_size"] + t % c["block_size"]
    k, v = _plain_rows(c, s["segments"], slots)  # [seqs, longest, heads, dim]
    k = k.permute(0, 2, 3, 1).contiguous()
    v = v.permute(0, 2, 1, 3).contiguous()
    z = q.reshape(seqs, heads, -1, dim) @ k * s["scale"]
    z = z.view(seqs, heads, -1, group, s["longest"])
    p = (lengths - new)[:, None] + torch.arange(s["most_new"], device="cuda")  # positions
    allowed = (t <= p[..., None]) & (t < lengths[:, None, None])
    if c["window"]:
        allowed &= t > p[..., None] - c["window"]
    allowed = allowed[:, None, :, None]
    z = z.masked_fill(~allowed, -math.inf)
    w = torch.exp(z - z.amax(-1, keepdim=True).clamp(min=-1e30))
    l = w.sum(-1)
    o = (w.view(seqs, heads, -1, s["longest"]) @ v).view(seqs, heads, -1, group, dim)
    o = o / l.clamp(min=1e-30)[..., None]
    o = o.permute(0, 2, 1, 3, 4).reshape(seqs, -1, q_heads, dim)
    s["out"].copy_(o[seq, index])


def _held(s):
    """What a write leaves: the values that the pages hold, and their scales."""
    c = s["case"]
    values = _values(c, s["segments"])
    return values if c["kind"] == "rows" else {"codes": values, "scales": _scales(c, s["segments"])}


def run(state):
    s, c = state, state["case"]
    if c["op"] == "write":
        if own:
            s["cache"].write(s["k"], s["v"], s["slots"])
        else:
            _plain_write(c, s["segments"], s["k"], s["v"], s["slots"])
        return _held(s)
    if c["op"] == "read":
        if own:
            s["cache"].read(s["slots"], s["k"], s["v"])
        else:
            rows = _plain_rows(c, s["segments"], s["slots"])
            s["k"].copy_(rows[0])
            s["v"].copy_(rows[1])
        return {"k": s["k"], "v": s["v"]}
    if own:
        s["cache"].attend(s["q"], s["out"], s["table"], s["lengths"], s["starts"],
                          scale=s["scale"], window=c["window"], max_seq_len=s["longest"],
                          max_query_len=s["most_new"], workspace=s["workspace"])
    else:
        _plain_attend(c, s)
    return s["out"]


def work(case):
    """Rows, and the pages' bytes of every token that a row attends to or that moves, once."""
    c = case
    new, cached = _lengths(c)
    held = 2 * c["heads"] * (2 * c["dim"] if c["kind"] == "rows" else c["dim"] + 4)
    if c["op"] != "attend":
        return {"bytes": sum(new) * (held + 4 * c["heads"] * c["dim"] + 8), "flops": 0}
    seen = pairs = 0
    for n, past in zip(new, cached):
        w = c["window"] or n + past
        seen += n + past - max(0, past + 1 - w)
        grow = max(0, min(n, w - past))  # rows that see everything up to themselves
        pairs += grow * past + grow * (grow + 1) // 2 + (n - grow) * w
    q_heads = c["heads"] * c["group"]
    return {"bytes": seen * held + 4 * sum(new) * q_heads * c["dim"],
            "flops": 4 * c["dim"] * q_heads * pairs}


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


def _exact_head(c, segments, table, length, kv, head):
    """K (0) or V (1) of one sequence and head in 64 bits: [length, dim]."""
    bs, heads, dim = c["block_size"], c["heads"], c["dim"]
    pages = segments[kv][table[:-(-length // bs)].long()]
    n = bs * heads * dim
    raw = pages.view(ROWS[c["rows"]]) if c["kind"] == "rows" else pages[:, :n]
    if c["head_major"]:
        raw = raw.reshape(-1, heads, bs, dim)[:, head]
    else:
        raw = raw.reshape(-1, bs, heads, dim)[:, :, head]
    x = _exact_value(c, raw)
    if c["kind"] != "rows":
        scales = pages[:, n:n + 4 * bs * heads].contiguous().view(torch.float32)
        x = x * scales.view(-1, heads, bs)[:, head].double()[..., None]
    return x.reshape(-1, dim)[:length]


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["op"] == "write":
        x = torch.stack((s["k"], s["v"])).double()
        at = (slice(None), s["slots"] // c["block_size"], s["slots"] % c["block_size"])
        held = torch.zeros(_values(c, s["segments"]).shape, dtype=torch.float64, device="cuda")
        if c["kind"] == "rows":
            held[at] = x
            return held
        scales = torch.zeros(held.shape[:-1], dtype=torch.float64, device="cuda")
        scales[at] = torch.linalg.vector_norm(x, ord=math.inf, dim=-1) / LARGEST[c["kind"]]
        if c["kind"] == "int8":  # whole numbers
            return {"codes": None, "scales": scales}
        held[at] = x / scales[at][..., None].clamp(min=1e-300)
        return {"codes": held, "scales": scales}
    if c["op"] == "read":
        bs = c["block_size"]
        order = torch.arange(s["segments"].shape[1], device="cuda")
        both = [torch.stack([_exact_head(c, s["segments"], order, len(order) * bs, kv, h)[s["slots"]]
                             for h in range(c["heads"])], 1) for kv in (0, 1)]
        return {"k": both[0], "v": both[1]}
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    group = c["group"]
    for i, (n, past) in enumerate(zip(*_lengths(c))):
        first = int(s["starts"][i])
        t = torch.arange(n + past, device="cuda")
        p = past + torch.arange(n, device="cuda")[:, None]
        hidden = (t > p) | (t <= p - c["window"]) if c["window"] else t > p
        for h in range(c["heads"]):
            k, v = (_exact_head(c, s["segments"], s["table"][i], n + past, kv, h) for kv in (0, 1))
            q = s["q"][first:first + n, h * group:(h + 1) * group].double().transpose(0, 1)
            z = torch.matmul(q.reshape(-1, c["dim"]), k.T.contiguous()).view(group, n, -1)
            z.mul_(s["scale"]).masked_fill_(hidden, -math.inf)
            z.sub_(torch.logsumexp(z, -1, keepdim=True)).exp_()
            o = torch.matmul(z.view(group * n, -1), v).view(group, n, -1)
            out[first:first + n, h * group:(h + 1) * group] = o.transpose(0, 1)
    return out
