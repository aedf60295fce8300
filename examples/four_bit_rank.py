"""A rank's KV cache held in 4 bits, from prompts to a packed cache: run on one MI355X.

    python examples/four_bit_rank.py

Prompts are written in 4 bits and attended over by chunks, single tokens decode, two sequences part from
one that they share pages with, and the pages of a sequence that ended are packed away, with the
same answers after each move. Weights are random: the numbers are those of an attention layer's shapes.
"""

from __future__ import annotations

import sys
import time
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import torch

from everserve_amd.state.fp4 import Fp4Cache
from everserve_amd.state.pages import PageMover

LAYERS, HEADS, SHARED, DIM, PAGE, PAGES = 4, 8, 4, 128, 16, 2048
PROMPTS = [1500, 700, 2048, 90]


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def main() -> None:
    g = torch.Generator(device="cuda").manual_seed(1)
    caches = [Fp4Cache.empty(PAGES, PAGE, HEADS, DIM, "kv_first") for _ in range(LAYERS)]
    mover = PageMover([c.tensor for c in caches], "kv_first")
    free = torch.randperm(PAGES, generator=torch.Generator().manual_seed(1)).tolist()
    tables = torch.full((6, 256), -1, dtype=torch.int32)
    for s, n in enumerate(PROMPTS):
        for p in range(-(-n // PAGE)):
            tables[s, p] = free.pop()

    def rows(n, heads):
        return torch.randn(n, heads, DIM, device="cuda", generator=g).bfloat16()

    def slots_of(s, at):
        at = torch.as_tensor(at)
        return (tables[s, at // PAGE].long() * PAGE + at % PAGE).cuda()

    # the prompts, a chunk of up to 512 tokens of each at a time: written, then attended over
    done = [0] * 4
    while any(d < n for d, n in zip(done, PROMPTS)):
        news = [min(512, n - d) for d, n in zip(done, PROMPTS)]
        lens = [d + k for d, k in zip(done, news)]
        slots = torch.cat([slots_of(s, torch.arange(d, d + k))
                           for s, (d, k) in enumerate(zip(done, news))])
        starts = [sum(news[:i]) for i in range(5)]
        for c in caches:
            c.write(slots, rows(len(slots), HEADS), rows(len(slots), HEADS))
            c.attend(rows(len(slots), HEADS * SHARED), tables[:4].cuda(), ints(lens),
                     q_starts=ints(starts), max_q=max(news), max_len=max(lens))
        done = lens

    # sequences 4 and 5 part from sequence 0: they share its whole pages and copy its last one
    last = (PROMPTS[0] - 1) // PAGE
    for s in (4, 5):
        tables[s] = tables[0]
        tables[s, last] = free.pop()
    mover.copy(tables[[0, 0], last].contiguous().cuda(), tables[[4, 5], last].contiguous().cuda())
    lens = PROMPTS + [PROMPTS[0]] * 2

    # 40 single tokens of each
    q = rows(6, HEADS * SHARED)
    torch.cuda.synchronize()
    start = time.perf_counter()
    for _ in range(40):
        for s in range(6):
            if lens[s] % PAGE == 0:
                tables[s, lens[s] // PAGE] = free.pop()
        lens = [n + 1 for n in lens]
        dev, n = tables.cuda(), ints(lens)
        slots = torch.cat([slots_of(s, [lens[s] - 1]) for s in range(6)])
        for c in caches:
            c.write(slots, rows(6, HEADS), rows(6, HEADS))
            out = c.attend(q, dev, n, max_len=max(lens))
    torch.cuda.synchronize()
    print(f"decoded 40 tokens of 6 sequences in {1e3 * (time.perf_counter() - start):.1f} ms, "
          f"{LAYERS} layers")

    # sequence 2 ends; what is left is packed to the front
    kept = [0, 1, 3, 4, 5]
    dev, n = tables[kept].contiguous().cuda(), ints([lens[s] for s in kept])
    counts = ints([-(-lens[s] // PAGE) for s in kept])
    want = [c.attend(q[:5], dev, n, max_len=max(lens)) for c in caches]
    plan = mover.compact(dev, counts)
    for c, w in zip(caches, want):
        assert torch.equal(c.attend(q[:5], plan.tables, n, max_len=max(lens)), w)
    used, moved = plan.sizes.tolist()
    print(f"packed {used} pages to the front by moving {moved}: pages from {used} on are free, "
          f"every answer is as it was")
    assert torch.isfinite(out).all()


if __name__ == "__main__":
    main()
