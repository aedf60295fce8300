"""A paged KV cache held in 4 bits, the attention that reads it, and moving a cache's pages.

A serving rank that holds its cache in 4 bits (MXFP4: E2M1 codes, one power-of-two scale for 32
dims) uses the operators at three places, and the cases follow them:

- **rows** (``rows``): a step's new K and V rows are rounded to 4 bits and written at their slots,
  and rows are read back at full width (what a prefill that reuses a prefix attends over);
- **attention** (``attend``): single tokens of many sequences, chunks of prompts, and both in one
  batch, over the 4-bit pages their block tables name;
- **pages** (``fork``, ``compact``): pages copied for sequences that part, and a cache whose used
  pages are packed to its front, with every block table rewritten, so that the rest is free.

A half-row (the K or the V of one slot and head) of head size d is d/2 bytes of codes (dim j in the
low half of byte j/2 where j is even), then one scale byte for each 32 dims (2^(byte-127); 255: the
group holds no number), then zeros up to a multiple of 4 bytes. The caches have the three layouts
that the snapshot and the restore know, with the half-row's bytes in the place of the head dim.

Moved bytes are compared as whole numbers, attention and rows read back as values.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
LAYOUTS = ("kv_first", "blocks_first", "combined")
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # E2M1's magnitudes by code
GROUP = 32


def listed():
    return [
        # one decode step of 64 sequences, a layer's new rows (8 KV heads of 128): latency
        dict(name="rows_decode", kind="rows", layout="kv_first", dtype="bf16", heads=8,
             head_dim=128, block_size=16, count=64, read=64, padding=0.0),
        # a prompt's chunk written, and the whole context before it read back
        dict(name="rows_prompt", kind="rows", layout="combined", dtype="bf16", heads=8,
             head_dim=128, block_size=16, count=8192, read=32768, padding=0.0),
        # rows from a wider fused tensor, head sizes off 32, a ragged list with padding
        dict(name="rows_odd", kind="rows", layout="blocks_first", dtype="f16", heads=6,
             head_dim=120, block_size=16, count=5001, read=7003, padding=0.02),
        # one short sequence's single token, 14 heads on 2 (the smallest model here): latency
        dict(name="attend_one", kind="attend", layout="kv_first", dtype="bf16", q_heads=14,
             heads=2, head_dim=64, block_size=16, seqs=1, min_len=600, max_len=600, queries=1,
             chunked=0, lse=False),
        # a decode step of 64 sequences, 32 heads on 8, contexts of up to 8 Ki
        dict(name="attend_decode", kind="attend", layout="kv_first", dtype="bf16", q_heads=32,
             heads=8, head_dim=128, block_size=16, seqs=64, min_len=1024, max_len=8192, queries=1,
             chunked=0, lse=False),
        # four long contexts on a rank that holds one KV head of eight
        dict(name="attend_long", kind="attend", layout="combined", dtype="bf16", q_heads=8,
             heads=1, head_dim=128, block_size=64, seqs=4, min_len=100000, max_len=131072,
             queries=1, chunked=0, lse=True),
        # small odd things: pages of 24, head size 80, an empty sequence and one of one token
        dict(name="attend_odd", kind="attend", layout="blocks_first", dtype="f16", q_heads=12,
             heads=4, head_dim=80, block_size=24, seqs=9, min_len=0, max_len=3001, queries=3,
             chunked=9, lse=True),
        # the last chunk of four prompts
        dict(name="attend_chunk", kind="attend", layout="kv_first", dtype="bf16", q_heads=32,
             heads=8, head_dim=128, block_size=16, seqs=4, min_len=4096, max_len=8192,
             queries=1024, chunked=4, lse=False),
        # a mixed batch: 14 single tokens and two prompts' chunks
        dict(name="attend_mixed", kind="attend", layout="combined", dtype="bf16", q_heads=32,
             heads=8, head_dim=128, block_size=16, seqs=16, min_len=512, max_len=4001,
             queries=257, chunked=2, lse=False),
        # 64 sequences part: the last page of each copied in every layer
        dict(name="fork_step", kind="fork", layout="kv_first", dtype="bf16", layers=32, heads=8,
             head_dim=128, block_size=16, num_blocks=512, count=64),
        # a fragmented bf16 cache packed to its front
        dict(name="compact_cache", kind="compact", layout="blocks_first", dtype="bf16", layers=8,
             heads=8, head_dim=128, block_size=16, num_blocks=2048, seqs=64, used=0.55),
        # the same of a 4-bit cache with many small pages
        dict(name="compact_fp4", kind="compact", layout="combined", dtype="fp4", layers=16,
             heads=2, head_dim=96, block_size=16, num_blocks=16384, seqs=200, used=0.4),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rows", "rows", "attend", "attend", "attend", "attend", "fork", "compact"])
    layout, heads = rng.choice(LAYOUTS), rng.choice([1, 2, 3, 4, 8])
    d = rng.choice([64, 80, 96, 112, 120, 128, 128, 128, 192, 256])
    if kind == "rows":
        count = _log_int(rng, 1, 16384)
        return dict(kind=kind, layout=layout, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                    heads=heads, head_dim=d, block_size=rng.choice([16, 16, 24, 32, 64]),
                    count=count, read=min(32768, _log_int(rng, count, 2 * count + 64)),
                    padding=rng.choice([0.0, 0.0, 0.02]))
    if kind == "attend":
        shared = rng.choice([1, 2, 4, 4, 7, 8])
        bs = rng.choice([16, 16, 16, 24, 32, 64, 128])
        form = rng.choice(["single", "single", "few", "chunk", "mixed"])
        if form == "chunk":
            seqs, queries, top = rng.randrange(1, 5), _log_int(rng, 16, 1024), 8192
            top = max(queries, _log_int(rng, 128, top))
        elif form == "mixed":
            seqs, queries, top = rng.randrange(3, 33), _log_int(rng, 8, 512), 4096
            top = max(queries, _log_int(rng, 256, top))
        else:
            seqs = _log_int(rng, 1, 128)
            queries = 1 if form == "single" else rng.randrange(2, 9)
            top = _log_int(rng, 1, min(131072, max(64, (1 << 22) // (seqs * heads))))
        # the plain form's padded keys and scores stay under those of the largest listed cases
        while seqs * top * heads * d > 64 * 8192 * 8 * 128 or (
                seqs * heads * shared * queries * top > 4 * 32 * 1024 * 8192):
            if seqs > 1:
                seqs = (seqs + 1) // 2
            else:
                top = max(1, top // 2)
                queries = min(queries, top)
        low = min(top, rng.choice([0, 1, top, max(1, top // 2), max(1, top // 16)]))
        chunked = {"single": 0, "few": seqs, "chunk": seqs}.get(form, max(1, seqs // 8))
        return dict(kind=kind, layout=layout, dtype=rng.choice(["bf16", "bf16", "f16"]),
                    q_heads=heads * shared, heads=heads, head_dim=d, block_size=bs, seqs=seqs,
                    min_len=low, max_len=top, queries=queries, chunked=chunked,
                    lse=rng.random() < 0.3)
    dtype = rng.choice(["bf16", "f16", "fp4", "fp4"])
    case = dict(kind=kind, layout=layout, dtype=dtype, layers=rng.choice([1, 4, 16, 24, 32, 36]),
                heads=heads, head_dim=d, block_size=rng.choice([16, 16, 24, 32]))
    page = case["layers"] * _page_bytes(case)
    case["num_blocks"] = _log_int(rng, 64, max(96, min(16384, (1 << 30) // page)))
    if kind == "fork":
        case["count"] = _log_int(rng, 1, case["num_blocks"] // 4)
    else:
        case["seqs"] = _log_int(rng, 1, 256)
        case["used"] = rng.choice([0.2, 0.4, 0.5, 0.7, 0.9])
    return case


# ---------------------------------------------------------------- sizes
def _row_bytes(d):
    return (d // 2 + -(-d // GROUP) + 3) // 4 * 4


def _half_bytes(case):
    d = case["head_dim"]
    return _row_bytes(d) if case["dtype"] == "fp4" else 2 * d


def _page_bytes(case):
    return 2 * case["block_size"] * case["heads"] * _half_bytes(case)


def _lens(case):
    """Context lengths, evenly spread from the shortest to the longest (an empty range starts with
    0 and 1): the seed only shuffles them."""
    n, lo, hi = case["seqs"], case["min_len"], case["max_len"]
    if n == 1:
        return [hi]
    got = [lo + (hi - lo) * i // (n - 1) for i in range(n)]
    if lo == 0 and n > 2:
        got[1] = min(1, hi)
    return got


def _queries(case):
    """New tokens of each sequence, before the shuffle: the longest contexts hold the chunks, the
    last of them a ragged one, and every other sequence one token."""
    n, chunked = case["seqs"], case["chunked"]
    got = [1] * n
    for i in range(n - chunked, n):
        got[i] = case["queries"]
    if chunked > 1:
        got[n - chunked] = max(1, case["queries"] - case["queries"] // 3)
    return got


def work(case):
    kind = case["kind"]
    if kind == "rows":
        wide = 2 * case["head_dim"] * (4 if case["dtype"] == "f32" else 2)
        held = 2 * (case["head_dim"] // 2 + -(-case["head_dim"] // GROUP))
        each = (wide + held) * case["heads"]
        return {"bytes": each * (case["count"] + case["read"]) + 8 * (case["count"] + case["read"]),
                "flops": 0}
    if kind == "attend":
        d, rows = case["head_dim"], 0
        held = 2 * (d // 2 + -(-d // GROUP)) * case["heads"]
        tokens = pairs = 0
        for n, q in zip(_lens(case), _queries(case)):
            rows += q
            tokens += n
            seen = min(q, n)  # queries that see something; the last one sees all n
            pairs += seen * n - seen * (seen - 1) // 2
        return {"bytes": tokens * held + 4 * rows * case["q_heads"] * d
                + 4 * -(-tokens // case["block_size"]) + (4 * rows * case["q_heads"] if case["lse"] else 0),
                "flops": 4 * pairs * case["q_heads"] * d}
    if kind == "fork":
        return {"bytes": 2 * case["count"] * case["layers"] * _page_bytes(case), "flops": 0}
    used = _used(case)
    moved = int(used * (1 - used / case["num_blocks"]))  # pages past the front, on average
    entries = _entries(case)
    return {"bytes": 2 * moved * case["layers"] * _page_bytes(case) + 8 * entries, "flops": 0}


def _used(case):
    return max(1, int(case["used"] * case["num_blocks"]))


def _width(case):
    """Entries of a block table's row: twice a sequence's mean, and one for each shared page."""
    return max(2, -(-2 * _used(case) // case["seqs"]) + 1)


def _entries(case):
    return case["seqs"] * _width(case)


# ---------------------------------------------------------------- inputs
def _shape(layout, blocks, block_size, heads, half):
    return {"kv_first": (2, blocks, block_size, heads, half),
            "blocks_first": (blocks, 2, block_size, heads, half),
            "combined": (blocks, heads, block_size, 2 * half)}[layout]


def _canonical(cache, layout):
    """A view of a cache as [blocks, block_size, heads, 2, half-row]."""
    if layout == "kv_first":
        return cache.permute(1, 2, 3, 0, 4)
    if layout == "blocks_first":
        return cache.permute(0, 2, 3, 1, 4)
    return cache.unflatten(3, (2, -1)).permute(0, 2, 1, 3, 4)


def _encode(x):
    """Rows of values [..., d] -> the half-rows' bytes [..., row_bytes], uint8.

    A group's scale is the power of two that puts its largest magnitude at 7 or below, where 6 is
    the largest code and 7 half a step past it; codes are the nearest, ties to the even code. A
    group that holds an infinity or a NaN holds no number."""
    x = x.float()
    d = x.shape[-1]
    groups = -(-d // GROUP)
    lead = x.shape[:-1]
    g = torch.nn.functional.pad(x, (0, groups * GROUP - d)).reshape(*lead, groups, GROUP)
    most = g.abs().amax(-1)
    good = torch.isfinite(g).all(-1)
    mantissa, exponent = torch.frexp(torch.where(good, most, torch.ones_like(most)))
    # most = mantissa * 2^exponent, mantissa in [0.5, 1): 7 * 2^(exponent - 3) is 0.875 * 2^exponent
    scale = exponent - 3 + (mantissa > 0.875)
    scale = torch.where(most > 0, scale, torch.full_like(scale, -126)).clamp(-126, 125)
    y = torch.ldexp(g, -scale.unsqueeze(-1)).abs()
    code = ((y > 0.25).to(torch.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5)
            + (y >= 3.5) + (y > 5.0)) | (torch.signbit(g).to(torch.uint8) << 3)
    code = torch.where(good.unsqueeze(-1), code, torch.zeros_like(code)).reshape(*lead, -1)[..., :d]
    byte = torch.where(good, scale + 127, torch.full_like(scale, 255)).to(torch.uint8)
    out = torch.zeros(*lead, _row_bytes(d), dtype=torch.uint8, device=x.device)
    out[..., :d // 2] = code[..., 0::2] | (code[..., 1::2] << 4)
    out[..., d // 2:d // 2 + groups] = byte
    return out


def _decode(half, d):
    """The half-rows' bytes [..., row_bytes] -> their values [..., d], float32."""
    grid = torch.tensor(GRID + tuple(-v for v in GRID), dtype=torch.float32, device=half.device)
    codes, byte = half[..., :d // 2], half[..., d // 2:d // 2 + -(-d // GROUP)].int()
    value = grid[torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()]
    scale = torch.ldexp(torch.ones_like(byte, dtype=torch.float32), byte - 127)
    scale = torch.where(byte == 255, torch.full_like(scale, math.nan), scale)
    return value * scale.repeat_interleave(GROUP, -1)[..., :d]


def _randn(shape, g, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=g)


def _keys(n, heads, d, g):
    """K and V rows [n, heads, 2, d]: a few of K's channels are several times the others."""
    x = _randn((n, heads, 2, d), g)
    x[:, :, 0] *= 1 + 4 * (torch.rand((heads, d), generator=g, device="cuda") > 0.95)
    return x


def _fill(cache, layout, heads, d, g):
    """Every page of a 4-bit cache, from rows as a model makes them."""
    view = _canonical(cache, layout)
    blocks, bs = view.shape[:2]
    step = max(1, (1 << 26) // (bs * heads * 2 * d))
    for b in range(0, blocks, step):
        e = min(blocks, b + step)
        rows = _keys((e - b) * bs, heads, d, g)
        view[b:e] = _encode(rows).reshape(e - b, bs, heads, 2, -1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, layout = case["kind"], case["layout"]
    state = dict(case=case)
    if kind in ("rows", "attend"):
        heads, d, bs = case["heads"], case["head_dim"], case["block_size"]
        if kind == "rows":
            count, read = case["count"], case["read"]
            blocks = -(-max(count, read) // bs) + 5
            order = torch.randperm(blocks, generator=g, device="cuda")
            slots = (order[:, None] * bs + torch.arange(bs, device="cuda")).reshape(-1)
            state["read"] = slots[:read].contiguous()
            state["slots"] = slots[max(0, read - count):][:count].contiguous()  # the newest rows
            if case["padding"]:
                for s in (state["read"], state["slots"]):
                    s[torch.rand(s.shape, generator=g, device="cuda") < case["padding"]] = -1
            rows = _keys(count, heads, d, g).to(DTYPES[case["dtype"]])
            # K and V are views of one tensor, as a fused projection leaves them
            fused = rows.transpose(1, 2).contiguous()
            state["key"], state["value"] = fused[:, 0], fused[:, 1]
        else:
            order = torch.randperm(case["seqs"], generator=g, device="cuda").tolist()
            lens, queries = _lens(case), _queries(case)
            lens, queries = [lens[i] for i in order], [queries[i] for i in order]
            pages = [-(-n // bs) for n in lens]
            blocks = sum(pages) + 3
            perm = torch.randperm(blocks, generator=g, device="cuda").int()
            width = max(1, max(pages))
            first = torch.tensor([sum(pages[:i]) for i in range(len(pages))], device="cuda")
            at = torch.arange(width, device="cuda")
            held = at < torch.tensor(pages, device="cuda")[:, None]
            index = (first[:, None] + at).clamp(max=blocks - 1)
            state["tables"] = torch.where(held, perm[index], torch.zeros_like(perm[index]))
            state["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
            starts = [sum(queries[:i]) for i in range(len(queries) + 1)]
            state["max_q"] = max(queries)
            state["starts"] = (torch.tensor(starts, dtype=torch.int32, device="cuda")
                               if max(queries) > 1 else None)
            q = _randn((starts[-1], case["q_heads"], d), g).mul_(1.5)
            state["q"] = q.to(DTYPES[case["dtype"]])
            state["scale"] = d ** -0.5
        cache = torch.zeros(_shape(layout, blocks, bs, heads, _row_bytes(d)), dtype=torch.uint8,
                            device="cuda")
        _fill(cache, layout, heads, d, g)
        state["cache"] = cache
        if own:
            from everserve_amd.state.fp4 import Fp4Cache
            state["held"] = Fp4Cache(cache, d)
        return state
    blocks, bs, layers = case["num_blocks"], case["block_size"], case["layers"]
    half = _half_bytes(case) if case["dtype"] == "fp4" else case["head_dim"]
    shape = (layers,) + _shape(layout, blocks, bs, case["heads"], half)
    # the bytes are moved, not read as numbers: any will do
    state["all"] = torch.randint(0, 256, shape if case["dtype"] == "fp4" else shape + (2,),
                                 dtype=torch.uint8, device="cuda", generator=g)
    if case["dtype"] != "fp4":
        state["all"] = state["all"].view(torch.int16)[..., 0]
    layers_of = list(state["all"].view(DTYPES.get(case["dtype"], torch.uint8)).unbind(0))
    perm = torch.randperm(blocks, generator=g, device="cuda").int()
    if kind == "fork":
        n = case["count"]
        state["src"], state["dst"] = perm[:n].contiguous(), perm[n:2 * n].contiguous()
    else:
        seqs, width, used = case["seqs"], _width(case), _used(case)
        # every used page is in some row, the first ones in a second row too (a shared prefix)
        tables = torch.full((seqs, width), -1, dtype=torch.int32, device="cuda")
        i = torch.arange(used, device="cuda")
        tables[i % seqs, i // seqs] = perm[:used]
        counts = ((used - torch.arange(seqs, device="cuda") + seqs - 1) // seqs).clamp(min=0)
        shared = perm[:1] if used else perm[:0]
        rows = torch.arange(0, seqs, 2, device="cuda")
        tables[rows, counts[rows]] = shared.expand(rows.numel())
        counts[rows] += 1
        state["tables"], state["counts"] = tables, counts.int()
    if own:
        from everserve_amd.state.pages import PageMover
        state["mover"] = PageMover(layers_of)
    return state


# ---------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "rows":
        if own:
            state["held"].write(state["slots"], state["key"], state["value"])
            return state["held"].read(state["read"], DTYPES[case["dtype"]])
        return _rows(state)
    if kind == "attend":
        if own:
            return state["held"].attend(state["q"], state["tables"], state["lens"],
                                        q_starts=state["starts"], max_q=state["max_q"],
                                        scale=state["scale"], return_lse=case["lse"])
        return _attend(state)
    if kind == "fork":
        if own:
            state["mover"].copy(state["src"], state["dst"])
        else:
            pages = _pages(state)
            pages[:, state["dst"].long()] = pages[:, state["src"].long()]
        return state["all"]
    if own:
        plan = state["mover"].compact(state["tables"], state["counts"])
        return plan.tables, plan.src, plan.dst, plan.sizes, state["all"]
    return _compact(state)


def _pages(state):
    """A view of every layer's cache with the pages second."""
    return state["all"].transpose(1, 2) if state["case"]["layout"] == "kv_first" else state["all"]


def _rows(state):
    case = state["case"]
    d, dtype = case["head_dim"], DTYPES[case["dtype"]]
    view, bs = _canonical(state["cache"], case["layout"]), case["block_size"]
    half = _encode(torch.stack((state["key"], state["value"]), 2))
    slots = state["slots"]
    kept = slots >= 0
    if case["padding"]:
        slots, half = slots[kept], half[kept]
    view[slots // bs, slots % bs] = half
    s = state["read"].clamp(min=0)
    x = _decode(view[s // bs, s % bs], d)  # [n, heads, 2, d]
    if case["padding"]:
        x = torch.where((state["read"] >= 0)[:, None, None, None], x, torch.zeros_like(x))
    x = x.to(dtype)
    return x[:, :, 0].contiguous(), x[:, :, 1].contiguous()


def _attend(state):
    case = state["case"]
    d, heads, bs = case["head_dim"], case["heads"], case["block_size"]
    q, tables, lens = state["q"], state["tables"].long(), state["lens"].long()
    seqs, top = case["seqs"], case["max_len"]
    shared, most = case["q_heads"] // heads, state["max_q"]
    if state["starts"] is None:
        starts = torch.arange(seqs + 1, device=q.device)
    else:
        starts = state["starts"].long()
    news = starts[1:] - starts[:-1]
    # keys and values of every sequence, padded to the longest: [seqs, heads, top, d]
    t = torch.arange(top, device=q.device)
    half = _canonical(state["cache"], case["layout"])[tables[:, t // bs], (t % bs).expand(seqs, top)]
    x = _decode(half, d)  # [seqs, top, heads, 2, d]
    key, value = x[..., 0, :].transpose(1, 2), x[..., 1, :].transpose(1, 2)
    # queries, padded to the most: [seqs, heads, shared * most, d]
    i = torch.arange(most, device=q.device)
    at = (starts[:-1, None] + i).clamp(max=q.shape[0] - 1)
    rows = q[at].float().reshape(seqs, most, heads, shared, d).permute(0, 2, 3, 1, 4)
    score = torch.matmul(rows.reshape(seqs, heads, shared * most, d),
                         key.transpose(-1, -2)).mul_(state["scale"])
    score = score.view(seqs, heads, shared, most, top)
    sees = (lens - news)[:, None] + i  # each query's own position: it sees it and all before
    seen = (t <= sees[..., None]) & (t < lens[:, None, None])  # [seqs, most, top]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top_score = score.amax(-1, keepdim=True)
    top_score = torch.where(top_score == -math.inf, torch.zeros_like(top_score), top_score)
    weight = score.sub_(top_score).exp_()
    total = weight.sum(-1, keepdim=True)
    value = torch.where((t < lens[:, None])[:, None, :, None], value, torch.zeros_like(value))
    out = torch.matmul(weight.view(seqs, heads, shared * most, top), value)
    out = out.view(seqs, heads, shared, most, d) / torch.where(total > 0, total,
                                                               torch.ones_like(total))
    out = out.permute(0, 3, 1, 2, 4).reshape(seqs, most, case["q_heads"], d)
    lse = (total.log() + top_score)[..., 0].permute(0, 3, 1, 2).reshape(seqs, most, -1)
    if most > 1:
        real = (i < news[:, None]).nonzero(as_tuple=True)
        out, lse = out[real], lse[real]
    else:
        out, lse = out[:, 0], lse[:, 0]
    out = out.to(q.dtype)
    return (out, lse) if case["lse"] else out


def _compact(state):
    tables, counts, blocks = state["tables"], state["counts"], state["case"]["num_blocks"]
    room = blocks // 2
    at = torch.arange(tables.shape[1], device=tables.device)
    valid = (at < counts[:, None]) & (tables >= 0) & (tables < blocks)
    used = torch.zeros(blocks + 1, dtype=torch.bool, device=tables.device)
    used[torch.where(valid, tables, torch.full_like(tables, blocks)).long()] = True
    used = used[:blocks]
    ids = torch.arange(blocks, device=tables.device)
    front = ids < used.sum()
    holes, movers = (front & ~used).nonzero()[:, 0], (~front & used).nonzero()[:, 0]
    new = ids.clone()
    new[movers] = holes
    moved = torch.where(valid, new[tables.clamp(0, blocks - 1).long()].int(), tables)
    src = torch.full((room,), -1, dtype=torch.int32, device=tables.device)
    dst = src.clone()
    src[:movers.numel()], dst[:holes.numel()] = movers.int(), holes.int()
    pages = _pages(state)
    pages[:, holes] = pages[:, movers]
    sizes = torch.stack((used.sum(), (~front & used).sum())).int()
    return moved, src, dst, sizes, state["all"]


# ---------------------------------------------------------------- in 64 bits
_STEPS = ((0.25, 0.5), (0.75, 1.0), (1.25, 1.5), (1.75, 2.0), (2.5, 3.0), (3.5, 4.0), (5.0, 6.0))


def _exact_values(x):
    """What rows [..., d] stand for once held in 4 bits, from the definition, in 64 bits."""
    d = x.shape[-1]
    out = torch.empty_like(x, dtype=torch.float64)
    for lo in range(0, d, GROUP):
        part = x[..., lo:lo + GROUP].double()
        most = part.abs().max(-1, keepdim=True).values
        power = torch.full_like(most, 2.0 ** -126)
        # the least power of two, from 2^-126 to 2^125, with most <= 7 * power
        low = torch.full_like(most, -126.0)
        need = torch.ceil(torch.log2((most / 7).clamp(min=1e-300)))
        need = torch.maximum(need, low)
        for shift in (-1, 0, 1):  # the logarithm may be off by a little next to a whole number
            p = torch.exp2((need + shift).clamp(-126, 125))
            power = torch.where((most <= 7 * p) & ((most > 3.5 * p) | (need + shift <= -126)), p, power)
        power = torch.where(most > 7 * 2.0 ** 125, torch.full_like(most, 2.0 ** 125), power)
        mag = part.abs() / power
        value = torch.zeros_like(mag)
        for k, (edge, code) in enumerate(_STEPS):
            up = mag > edge if k % 2 == 0 else mag >= edge
            value = torch.where(up, torch.full_like(mag, code), value)
        value = torch.copysign(value * power, part)
        bad = ~torch.isfinite(part).all(-1, keepdim=True)
        out[..., lo:lo + GROUP] = torch.where(bad, torch.full_like(value, math.nan), value)
    return out


def _exact_rows_of(half, d):
    """The values of half-rows' bytes in 64 bits, byte by byte."""
    out = torch.empty(half.shape[:-1] + (d,), dtype=torch.float64, device=half.device)
    for j in range(d):
        code = (half[..., j // 2].int() >> (4 * (j % 2))) & 15
        low, e = (code & 1).double(), ((code >> 1) & 3).double()
        mag = torch.where(e > 0, (1 + low / 2) * torch.exp2(e - 1), low / 2)
        power = torch.exp2(half[..., d // 2 + j // GROUP].double() - 127)
        power[half[..., d // 2 + j // GROUP] == 255] = math.nan
        out[..., j] = torch.where(code >= 8, -mag, mag) * power
    return out


def exact(case, seed):
    if case["kind"] not in ("rows", "attend"):
        return None  # moved bytes and page numbers: nothing is computed
    state = prepare(case, seed)
    d, bs, heads = case["head_dim"], case["block_size"], case["heads"]
    view = _canonical(state["cache"], case["layout"])
    if case["kind"] == "rows":
        read = state["read"]
        s = read.clamp(min=0)
        got = _exact_rows_of(view[s // bs, s % bs], d)  # [n, heads, 2, d]
        slots = state["slots"]
        where = torch.full((view.shape[0] * bs,), -1, dtype=torch.long, device=slots.device)
        kept = slots >= 0
        where[slots[kept]] = torch.arange(slots.numel(), device=slots.device)[kept]
        fresh = _exact_values(torch.stack((state["key"], state["value"]), 2))
        new = where[s]
        got = torch.where((new >= 0)[:, None, None, None], fresh[new.clamp(min=0)], got)
        got = torch.where((read >= 0)[:, None, None, None], got, torch.zeros_like(got))
        return got[:, :, 0], got[:, :, 1]
    outs, lses = [], []
    starts = (state["starts"].tolist() if state["starts"] is not None
              else list(range(case["seqs"] + 1)))
    shared = case["q_heads"] // heads
    for k, n in enumerate(state["lens"].tolist()):
        q = state["q"][starts[k]:starts[k + 1]].double()
        out = torch.zeros_like(q)
        lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
        if n:
            t = torch.arange(n, device=q.device)
            x = _exact_rows_of(view[state["tables"][k, t // bs].long(), t % bs], d)
            for h in range(heads):
                at = slice(h * shared, (h + 1) * shared)
                score = torch.tensordot(q[:, at], x[:, h, 0], dims=([2], [1])) * state["scale"]
                last = n - q.shape[0] + torch.arange(q.shape[0], device=q.device)
                score = score.masked_fill((t > last[:, None])[:, None], -math.inf)
                some = last >= 0
                lse[:, at] = torch.where(some[:, None], torch.logsumexp(score, -1), lse[:, at])
                share = torch.exp(score - torch.where(some[:, None], lse[:, at], 0.0)[..., None])
                out[:, at] = torch.tensordot(share, x[:, h, 1], dims=([2], [0]))
        outs.append(out)
        lses.append(lse)
    out = torch.cat(outs)
    return (out, torch.cat(lses)) if case["lse"] else out
