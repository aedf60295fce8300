"""Attention over full-width paged caches for batches that share a prefix, the weights that tokens
gather in it, and the eviction that goes by them.

A serving rank uses the operators at three places, and the cases follow them:

- **attention** (``attend``): single tokens, a few tokens and chunks of prompts over bf16 and f16
  pages, where groups of sequences share a prefix's pages (a system prompt, a document, the samples
  of one prompt), which are read once for all of them;
- **weights** (``weigh``): the same, and what each token of the cache got of its softmaxes' weight,
  summed over the queries and the heads that share a KV head, is added to the token's mass;
- **eviction** (``evict``): of each layer, sequence and KV head, the newest tokens and those with the
  most mass stay; their rows go to the sequence's new pages, in their order, and their mass with them.

The caches have the three layouts that the snapshot and the restore know. A sequence's own pages
follow its group's prefix; its queries are the last of its own tokens and see what lies before them.
Mass lies in float32 by page: [layers, pages, KV heads, tokens of a page].

Rows that are moved, and the choice of them, are compared as whole numbers.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
LAYOUTS = ("kv_first", "blocks_first", "combined")


def listed():
    return [
        # two samples of one short prompt, 14 heads on 2 (the smallest model here): latency
        dict(name="shared_one", kind="attend", layout="kv_first", dtype="bf16", q_heads=14, heads=2,
             head_dim=64, block_size=16, seqs=2, groups=1, prefix=600, min_len=5, max_len=40,
             queries=1, chunked=0, lse=False),
        # a decode step of 64 sequences behind one prompt of 8 Ki, 32 heads on 8
        dict(name="shared_decode", kind="attend", layout="kv_first", dtype="bf16", q_heads=32,
             heads=8, head_dim=128, block_size=16, seqs=64, groups=1, prefix=8192, min_len=1,
             max_len=1024, queries=1, chunked=0, lse=False),
        # 16 questions about one long document, on a rank that holds one KV head of eight
        dict(name="shared_long", kind="attend", layout="combined", dtype="bf16", q_heads=8, heads=1,
             head_dim=128, block_size=64, seqs=16, groups=1, prefix=131072, min_len=100,
             max_len=2001, queries=1, chunked=0, lse=True),
        # three groups, pages of 24, head size 80, a sequence with nothing of its own, a few queries
        dict(name="shared_odd", kind="attend", layout="blocks_first", dtype="f16", q_heads=12,
             heads=4, head_dim=80, block_size=24, seqs=11, groups=3, prefix=1501, min_len=0,
             max_len=301, queries=3, chunked=5, lse=True),
        # four prompts' chunks behind a prefix, beside single tokens of 12 others
        dict(name="shared_chunk", kind="attend", layout="blocks_first", dtype="bf16", q_heads=32,
             heads=8, head_dim=128, block_size=16, seqs=16, groups=2, prefix=4096, min_len=64,
             max_len=1024, queries=512, chunked=4, lse=False),
        # one short sequence's single token, its weights gathered: latency
        dict(name="weigh_one", kind="weigh", layout="kv_first", dtype="bf16", q_heads=14, heads=2,
             head_dim=64, block_size=16, seqs=1, groups=0, prefix=0, min_len=600, max_len=600,
             queries=1, chunked=0, lse=False),
        # a decode step of 64 sequences, weights gathered
        dict(name="weigh_decode", kind="weigh", layout="kv_first", dtype="bf16", q_heads=32, heads=8,
             head_dim=128, block_size=16, seqs=64, groups=0, prefix=0, min_len=1024, max_len=4096,
             queries=1, chunked=0, lse=False),
        # the last chunks of two prompts that share a prefix, weights gathered
        dict(name="weigh_chunk", kind="weigh", layout="combined", dtype="bf16", q_heads=32, heads=8,
             head_dim=128, block_size=16, seqs=2, groups=1, prefix=1000, min_len=1024, max_len=4001,
             queries=1024, chunked=2, lse=True),
        # one short sequence of the smallest model cut down: latency
        dict(name="evict_one", kind="evict", layout="kv_first", dtype="bf16", layers=24, heads=2,
             head_dim=64, block_size=16, seqs=1, min_len=600, max_len=600, budget=256, recent=32),
        # four sequences cut to 1,024 tokens, half of the layers of a rank with 8 KV heads
        dict(name="evict_cache", kind="evict", layout="kv_first", dtype="bf16", layers=16, heads=8,
             head_dim=128, block_size=16, seqs=4, min_len=2048, max_len=4096, budget=1024,
             recent=128),
        # two long contexts on a rank that holds one KV head of eight
        dict(name="evict_long", kind="evict", layout="blocks_first", dtype="bf16", layers=8, heads=1,
             head_dim=128, block_size=64, seqs=2, min_len=100000, max_len=131072, budget=16384,
             recent=1024),
        # a 4-bit cache, pages of 24, sequences of no token up to 3,001, all shorter ones kept whole
        dict(name="evict_odd", kind="evict", layout="combined", dtype="fp4", layers=5, heads=3,
             head_dim=96, block_size=24, seqs=9, min_len=0, max_len=3001, budget=701, recent=33),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "weigh", "weigh", "evict", "evict"])
    layout, heads = rng.choice(LAYOUTS), rng.choice([1, 2, 3, 4, 8])
    d = rng.choice([64, 80, 96, 112, 120, 128, 128, 128, 192, 256])
    bs = rng.choice([16, 16, 16, 24, 32, 64])
    if kind == "evict":
        layers, seqs = rng.choice([1, 4, 8, 16, 24, 32]), _log_int(rng, 1, 32)
        top = _log_int(rng, 64, max(64, min(131072, (10 << 24) // (layers * seqs * heads * d))))
        budget = _log_int(rng, 16, max(16, top // 2))
        return dict(kind=kind, layout=layout, dtype=rng.choice(["bf16", "bf16", "f16", "fp4"]),
                    layers=layers, heads=heads, head_dim=d, block_size=bs, seqs=seqs,
                    min_len=rng.choice([0, top // 2, top]), max_len=top, budget=budget,
                    recent=rng.choice([0, 1, budget // 8, budget // 2]))
    shared = rng.choice([1, 2, 4, 4, 7, 8])
    form = rng.choice(["single", "single", "few", "chunk", "mixed"])
    if form == "chunk":
        seqs, queries = rng.randrange(1, 5), _log_int(rng, 16, 1024)
    elif form == "mixed":
        seqs, queries = rng.randrange(3, 33), _log_int(rng, 8, 512)
    else:
        seqs, queries = _log_int(rng, 1, 128), 1 if form == "single" else rng.randrange(2, 9)
    groups = rng.choice([0, 1, 1, 1, 2, 3]) if kind == "weigh" else rng.choice([1, 1, 1, 2, 3])
    groups = min(groups, seqs)
    prefix = _log_int(rng, 16, 131072 if heads == 1 else 16384) if groups else 0
    top = _log_int(rng, max(1, queries), 4096)
    # the plain form's scores and padded keys stay under those of the largest listed cases
    while (seqs * heads * shared * queries * (top + prefix) > 2 * 32 * 1024 * 5001
           or (seqs * top + groups * prefix) * heads * d > 64 * 4096 * 8 * 128):
        if prefix > top:
            prefix = max(1, prefix // 2)
        elif seqs > max(1, groups):
            seqs = max(max(1, groups), seqs // 2)
        else:
            top = max(1, top // 2)
            queries = min(queries, top)
    low = min(top, rng.choice([0, 1, max(1, top // 2), top]))
    chunked = {"single": 0, "few": seqs, "chunk": seqs}.get(form, max(1, seqs // 8))
    return dict(kind=kind, layout=layout, dtype=rng.choice(["bf16", "bf16", "f16"]),
                q_heads=heads * shared, heads=heads, head_dim=d, block_size=bs, seqs=seqs,
                groups=groups, prefix=prefix, min_len=low, max_len=top, queries=queries,
                chunked=chunked, lse=rng.random() < 0.3)


# ---------------------------------------------------------------- sizes
def _lens(case):
    """Lengths of the sequences' own tokens, evenly spread from the shortest to the longest: the
    seed only shuffles them."""
    n, lo, hi = case["seqs"], case["min_len"], case["max_len"]
    if n == 1:
        return [hi]
    return [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _queries(case):
    """New tokens of each sequence, before the shuffle: the longest hold the chunks, the last of
    them a ragged one, and every other sequence one token."""
    n, chunked = case["seqs"], case["chunked"]
    got = [1] * (n - chunked) + [case["queries"]] * chunked
    if chunked > 1:
        got[n - chunked] = max(1, case["queries"] - case["queries"] // 3)
    return got


def _prefixes(case):
    """Lengths of the groups' prefixes: the first the longest."""
    return [max(1, case["prefix"] * (case["groups"] - i) // case["groups"])
            for i in range(case["groups"])]


def _group_starts(case):
    """Where the groups' sequences start: the groups are of unlike size."""
    g, n = case["groups"], case["seqs"]
    if 2 * n < g * (g + 1):
        return list(range(g)) + [n]
    return [n * i * (i + 1) // max(1, g * (g + 1)) for i in range(g + 1)]


def _half_bytes(case):
    d = case["head_dim"]
    return (d // 2 + -(-d // 32) + 3) // 4 * 4 if case["dtype"] == "fp4" else 2 * d


def _pages(lens, bs):
    return [-(-n // bs) for n in lens]


def work(case):
    heads, bs = case["heads"], case["block_size"]
    if case["kind"] == "evict":
        lens = _lens(case)
        kept = sum(min(n, case["budget"]) for n in lens)
        each = case["layers"] * heads
        # the list of kept tokens is as wide as the budget
        return {"bytes": each * (4 * kept * _half_bytes(case) + 4 * sum(lens) + 4 * kept
                                 + 4 * case["budget"] * case["seqs"]) + 4 * sum(_pages(lens, bs)),
                "flops": 0}
    d, rows, pairs = case["head_dim"], 0, 0
    lens, queries = _lens(case), _queries(case)
    held = sum(lens) + sum(_prefixes(case))
    starts, prefixes = _group_starts(case), _prefixes(case)
    for g, n in enumerate(prefixes):
        # the shuffle deals chunks to groups by chance: of each group its share on average
        pairs += n * sum(queries) * (starts[g + 1] - starts[g]) / case["seqs"]
    for n, q in zip(lens, queries):
        rows += q
        seen = min(q, n)
        pairs += seen * n - seen * (seen - 1) // 2
    more = 8 * held * heads if case["kind"] == "weigh" else 0
    return {"bytes": held * heads * 4 * d + 4 * rows * case["q_heads"] * d + 4 * -(-held // bs)
            + (4 * rows * case["q_heads"] if case["lse"] else 0) + more,
            "flops": 4 * pairs * case["q_heads"] * d}


# ---------------------------------------------------------------- inputs
def _shape(layout, blocks, block_size, heads, half):
    return {"kv_first": (2, blocks, block_size, heads, half),
            "blocks_first": (blocks, 2, block_size, heads, half),
            "combined": (blocks, heads, block_size, 2 * half)}[layout]


def _canonical(cache, layout):
    """A view of a cache as [..., blocks, block_size, heads, 2, half-row]."""
    if layout == "kv_first":
        return cache.movedim(-5, -2)
    if layout == "blocks_first":
        return cache.movedim(-4, -2)
    return cache.unflatten(-1, (2, -1)).transpose(-4, -3)


def _randn(shape, g, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=g)


def _mass(shape, g):
    """Weights that tokens have gathered: a few tokens have most of them, many the same little."""
    x = torch.empty(shape, dtype=torch.float32, device="cuda").uniform_(generator=g)
    return torch.where(x < 0.2, torch.floor(x * 40) / 64, x.pow(12) * 30)


def _tables(pages, width, perm, at):
    """Block tables [rows, width] from the permuted page ids, row by row from place `at` on."""
    first = torch.tensor([at + sum(pages[:i]) for i in range(len(pages))], dtype=torch.long)
    i = torch.arange(width)
    index = torch.where(i < torch.tensor(pages, dtype=torch.long)[:, None], first[:, None] + i,
                        torch.zeros(1, dtype=torch.long))
    return perm[index.reshape(-1).to(perm.device)].reshape(len(pages), width)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    layout, heads, d, bs = case["layout"], case["heads"], case["head_dim"], case["block_size"]
    state = dict(case=case)
    order = torch.randperm(case["seqs"], generator=g, device="cuda").tolist()
    lens = _lens(case)
    lens = [lens[i] for i in order]
    pages = _pages(lens, bs)
    ints = dict(dtype=torch.int32, device="cuda")
    if case["kind"] == "evict":
        budget = case["budget"]
        room = -(-budget // bs)
        blocks = sum(pages) + case["seqs"] * room + 3
        perm = torch.randperm(blocks, generator=g, device="cuda").int()
        state["tables"] = _tables(pages, max(1, max(pages)), perm, 0)
        state["new_tables"] = _tables([room] * case["seqs"], room, perm, sum(pages))
        state["lens"] = torch.tensor(lens, **ints)
        fp4 = case["dtype"] == "fp4"
        shape = (case["layers"],) + _shape(layout, blocks, bs, heads, _half_bytes(case) if fp4 else d)
        # the bytes are moved, not read as numbers: any will do
        if fp4:
            state["all"] = torch.randint(0, 256, shape, dtype=torch.uint8, device="cuda",
                                         generator=g)
        else:
            state["all"] = torch.randint(-32768, 32768, shape, dtype=torch.int16, device="cuda",
                                         generator=g)
        state["mass"] = _mass((case["layers"], blocks, heads, bs), g)
        if own:
            from everserve_amd.state.evict import Evictor
            layers = state["all"].view(DTYPES.get(case["dtype"], torch.uint8)).unbind(0)
            state["evictor"] = Evictor(list(layers), layout)
        return state
    queries = _queries(case)
    queries = [queries[i] for i in order]
    prefixes = _prefixes(case)
    before = _pages(prefixes, bs)
    blocks = sum(pages) + sum(before) + 3
    perm = torch.randperm(blocks, generator=g, device="cuda").int()
    state["tables"] = _tables(pages, max(1, max(pages)), perm, sum(before))
    state["lens"] = torch.tensor(lens, **ints)
    starts = [sum(queries[:i]) for i in range(len(queries) + 1)]
    state["max_q"] = max(queries)
    state["starts"] = torch.tensor(starts, **ints) if max(queries) > 1 else None
    if prefixes:
        state["prefix_tables"] = _tables(before, max(before), perm, 0)
        state["prefix_lens"] = torch.tensor(prefixes, **ints)
        state["group_starts"] = torch.tensor(_group_starts(case), **ints)
    dtype = DTYPES[case["dtype"]]
    cache = _randn(_shape(layout, blocks, bs, heads, d), g, dtype)
    # a few of K's channels are several times the others
    key = _canonical(cache, layout)[..., 0, :]
    key.mul_((1 + 4 * (torch.rand((heads, d), generator=g, device="cuda") > 0.95)).to(dtype))
    state["cache"] = cache
    state["q"] = _randn((starts[-1], case["q_heads"], d), g).mul_(1.5).to(dtype)
    state["scale"] = d ** -0.5
    if case["kind"] == "weigh":
        state["mass"] = _mass((blocks, heads, bs), g)
    if own:
        from everserve_amd.state.full import FullCache, SharedPrefix
        state["held"] = FullCache(cache, layout)
        state["prefix"] = SharedPrefix(state["prefix_tables"], state["prefix_lens"],
                                       state["group_starts"]) if prefixes else None
    return state


# ---------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if case["kind"] == "evict":
        if own:
            got = state["evictor"].evict(state["tables"], state["lens"], state["new_tables"],
                                         case["budget"], state["mass"], recent=case["recent"])
            return got.lens, got.kept, state["mass"], state["all"]
        return _evict(state)
    mass = state["mass"].clone() if case["kind"] == "weigh" else None
    if own:
        out = state["held"].attend(state["q"], state["tables"], state["lens"],
                                   q_starts=state["starts"], max_q=state["max_q"],
                                   scale=state["scale"], return_lse=case["lse"],
                                   prefix=state["prefix"], mass=mass)
    else:
        out = _attend(state, mass)
    return out if mass is None else (out, mass)


def _soft(score, seen, value):
    """Scores [..., rows, tokens] (kept) and values [..., tokens, d] to the rows' maxima, sums of
    weights and sums of weighted values."""
    score.masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    base = torch.where(top == -math.inf, torch.zeros_like(top), top)
    weight = (score - base).exp_()
    return top, weight.sum(-1, keepdim=True), torch.matmul(weight, value)


def _rows_of(cache, layout, tables, lens):
    """The keys and values [rows, heads, tokens, d] that tables name, in 32 bits, zeros past the
    lengths; which tokens there are [rows, tokens]; and their pages and offsets."""
    view = _canonical(cache, layout)
    bs, width = view.shape[1], tables.shape[1]
    t = torch.arange(width * bs, device=cache.device)
    page, off = tables.long()[:, t // bs], (t % bs).expand(tables.shape[0], -1)
    there = t < lens[:, None]
    x = torch.where(there[..., None, None, None], view[page, off].float(), 0.0)
    return x[:, :, :, 0].transpose(1, 2), x[:, :, :, 1].transpose(1, 2), there, page, off


def _attend(state, mass):
    case = state["case"]
    d, heads, seqs = case["head_dim"], case["heads"], case["seqs"]
    q, lens, most = state["q"], state["lens"].long(), state["max_q"]
    shared, dev = case["q_heads"] // heads, q.device
    if state["starts"] is None:
        starts = torch.arange(seqs + 1, device=dev)
    else:
        starts = state["starts"].long()
    news = starts[1:] - starts[:-1]
    # queries, padded to the most: [seqs, heads, shared * most, d]
    i = torch.arange(most, device=dev)
    at = (starts[:-1, None] + i).clamp(max=q.shape[0] - 1)
    rows = q[at].float().mul_(state["scale"]).reshape(seqs, most, heads, shared, d)
    rows = rows.permute(0, 2, 3, 1, 4).reshape(seqs, heads, shared * most, d)
    real = (i < news[:, None])[:, None, None, :].expand(seqs, heads, shared, most)
    real = real.reshape(seqs, heads, shared * most, 1)
    # their own tokens
    key, value, there, page, off = _rows_of(state["cache"], case["layout"], state["tables"], lens)
    t = torch.arange(key.shape[2], device=dev)
    seen = (t <= ((lens - news)[:, None] + i)[..., None]) & there[:, None]  # [seqs, most, tokens]
    seen = seen[:, None, None].expand(seqs, heads, shared, most, -1).reshape(
        seqs, heads, shared * most, -1) & real
    score = torch.matmul(rows, key.transpose(-1, -2))
    top, total, out = _soft(score, seen, value)
    del key, value
    if case["groups"]:
        # the prefixes, each once: their groups' rows side by side, padded to the largest group
        first = state["group_starts"].long()
        n = torch.arange(seqs, device=dev)
        group = (n[:, None] >= first[1:]).sum(1)
        per = seqs if case["groups"] == 1 else max(b - a for a, b in zip(
            _group_starts(case), _group_starts(case)[1:]))
        member = (first[:-1, None] + torch.arange(per, device=dev))
        inside = member < first[1:, None]
        member = member.clamp(max=seqs - 1)
        near = (case["groups"], heads, per * shared * most)
        pkey, pvalue, pthere, ppage, poff = _rows_of(state["cache"], case["layout"],
                                                     state["prefix_tables"],
                                                     state["prefix_lens"].long())
        prows = rows[member].transpose(1, 2).reshape(*near, d)
        preal = (real[member] & inside[:, :, None, None, None]).transpose(1, 2).reshape(*near, 1)
        pscore = torch.matmul(prows, pkey.transpose(-1, -2))
        parts = _soft(pscore, pthere[:, None, None] & preal, pvalue)
        del pkey, pvalue
        ptop, ptotal, pout = (x.reshape(case["groups"], heads, per, shared * most, -1)[
            group, :, n - first[group]] for x in parts)
        both = torch.maximum(top, ptop)
        base = torch.where(both == -math.inf, torch.zeros_like(both), both)
        f, pf = (top - base).exp(), (ptop - base).exp()
        top, total, out = both, total * f + ptotal * pf, out * f + pout * pf
    out = out / torch.where(total > 0, total, torch.ones_like(total))
    base = torch.where(top == -math.inf, torch.zeros_like(top), top)
    lse = total.log() + base
    if mass is not None:
        # a row that sees nothing has no weights
        cut = torch.where(lse == -math.inf, torch.full_like(lse, math.inf), lse)
        gave = (score - cut).exp_().sum(2)  # [seqs, heads, tokens]
        fresh = (t >= (lens - news)[:, None]) & there
        _give(mass, page, off, there, gave, fresh)
        if case["groups"]:
            pcut = cut[member].transpose(1, 2).reshape(*near, 1)
            _give(mass, ppage, poff, pthere, (pscore - pcut).exp_().sum(2), None)
    out = out.view(seqs, heads, shared, most, d).permute(0, 3, 1, 2, 4)
    out = out.reshape(seqs, most, case["q_heads"], d)
    lse = lse.view(seqs, heads, shared, most).permute(0, 3, 1, 2).reshape(seqs, most, -1)
    there = (i < news[:, None]).nonzero(as_tuple=True)
    out, lse = out[there].to(q.dtype), lse[there]
    return (out, lse) if case["lse"] else out


def _give(mass, page, off, there, gave, fresh):
    """Adds gave [rows, heads, tokens] to the mass of the tokens; fresh ones start from zero."""
    page, off = page[there], off[there]
    old = mass[page, :, off]
    if fresh is not None:
        old = torch.where(fresh[there][:, None], torch.zeros_like(old), old)
    mass[page, :, off] = old + gave.transpose(1, 2)[there]


def _evict(state):
    case = state["case"]
    bs, budget = case["block_size"], case["budget"]
    tables, lens, mass = state["tables"].long(), state["lens"].long(), state["mass"]
    dev = mass.device
    t = torch.arange(tables.shape[1] * bs, device=dev)
    there = t < lens[:, None]  # [seqs, tokens]
    newest = there & (t >= (lens - case["recent"])[:, None])
    # [layers, seqs, heads, tokens]: the newest before all others, tokens that are none after them
    key = mass[:, tables[:, t // bs], :, t % bs].permute(2, 0, 3, 1)
    key = torch.where(newest[:, None], torch.full_like(key, math.inf), key)
    key = torch.where(there[:, None], key, torch.full_like(key, -math.inf))
    order = key.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    short = budget - order.shape[-1]
    if short > 0:
        order = torch.nn.functional.pad(order, (0, short), value=t.numel())
    count = lens.clamp(max=budget)
    j = torch.arange(budget, device=dev)
    held = (j < count[:, None])[:, None]  # [seqs, 1, budget]
    kept = torch.where(held, order, torch.full_like(order, 1 << 30)).sort(-1).values
    held = held.expand(kept.shape)
    kept = torch.where(held, kept, torch.full_like(kept, -1))
    # where each kept row lies, and where it goes
    layer, seq, head, place = held.nonzero(as_tuple=True)
    token = kept[layer, seq, head, place]
    src, dst = tables[seq, token // bs], state["new_tables"].long()[seq, place // bs]
    rows = _canonical(state["all"], case["layout"])
    rows[layer, dst, place % bs, head] = rows[layer, src, token % bs, head]
    mass[layer, dst, head, place % bs] = mass[layer, src, head, token % bs]
    return count.int(), kept.int(), mass, state["all"]


# ---------------------------------------------------------------- in 64 bits
def exact(case, seed):
    if case["kind"] == "evict":
        return None  # rows are chosen and moved: nothing is computed
    state = prepare(case, seed)
    bs, heads, shared = case["block_size"], case["heads"], case["q_heads"] // case["heads"]
    view = _canonical(state["cache"], case["layout"])
    groups = _group_starts(case)
    starts = (state["starts"].tolist() if state["starts"] is not None
              else list(range(case["seqs"] + 1)))
    mass = state["mass"].double() if case["kind"] == "weigh" else None
    outs, lses = [], []

    def places(table, n):
        t = torch.arange(n, device=view.device)
        return table[t // bs].long(), t % bs

    if mass is not None:  # a call's new tokens start from nothing
        for k, n in enumerate(state["lens"].tolist()):
            page, off = places(state["tables"][k], n)
            new = max(0, n - (starts[k + 1] - starts[k]))
            mass[page[new:], :, off[new:]] = 0
    for k, n in enumerate(state["lens"].tolist()):
        page, off = places(state["tables"][k], n)
        before = 0
        for j in range(case["groups"]):
            if groups[j] <= k < groups[j + 1]:
                before = int(state["prefix_lens"][j])
                ppage, poff = places(state["prefix_tables"][j], before)
                page, off = torch.cat((ppage, page)), torch.cat((poff, off))
        q = state["q"][starts[k]:starts[k + 1]].double()
        out = torch.zeros_like(q)
        lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
        t = torch.arange(before + n, device=q.device)
        last = before + n - q.shape[0] + torch.arange(q.shape[0], device=q.device)
        last = torch.clamp(last, min=before - 1)  # all of the prefix is seen
        some = last >= 0
        for h in range(heads if before + n else 0):
            at = slice(h * shared, (h + 1) * shared)
            x = view[page, off, h].double()
            score = torch.tensordot(q[:, at], x[:, 0], dims=([2], [1])) * state["scale"]
            score = score.masked_fill((t > last[:, None])[:, None], -math.inf)
            lse[:, at] = torch.where(some[:, None], torch.logsumexp(score, -1), lse[:, at])
            share = torch.exp(score - torch.where(some[:, None], lse[:, at], 0.0)[..., None])
            out[:, at] = torch.tensordot(share, x[:, 1], dims=([2], [0]))
            if mass is not None:
                mass[page, h, off] += share.sum((0, 1))
        outs.append(out)
        lses.append(lse)
    out = torch.cat(outs)
    got = (out, torch.cat(lses)) if case["lse"] else out
    return got if mass is None else (got, mass)
