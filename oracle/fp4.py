"""The 4-bit cache, its attention and the moves of pages, restated plainly: the tests' oracle.

Everything is computed in 64 bits on the CPU from the definitions in ``include/everserve_mi355x.h``:
codes by comparing with every value a code can hold, attention row by row, page moves one at a time.
"""

from __future__ import annotations

import math

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
GROUP = 32


def row_bytes(d: int) -> int:
    return (d // 2 + -(-d // GROUP) + 3) // 4 * 4


def encode_group(x) -> tuple[int, np.ndarray]:
    """A group's scale byte and codes: ``x`` float64, at most 32 values."""
    if not np.all(np.isfinite(x)):
        return 255, np.zeros(len(x), dtype=np.uint8)
    most = float(np.max(np.abs(x)))
    e = -126
    while e < 125 and most > 7 * 2.0 ** e:
        e += 1
    codes = np.empty(len(x), dtype=np.uint8)
    for j, v in enumerate(np.abs(x) / 2.0 ** e):
        off = np.abs(GRID - v)
        near = np.flatnonzero(off == off.min())
        codes[j] = near[0] if len(near) == 1 else [c for c in near if c % 2 == 0][0]
    return e + 127, codes | (np.signbit(x).astype(np.uint8) << 3)


def encode(x) -> np.ndarray:
    """Half-rows' bytes [..., row_bytes] of values [..., d]."""
    x = np.asarray(x, dtype=np.float64)
    d = x.shape[-1]
    out = np.zeros(x.shape[:-1] + (row_bytes(d),), dtype=np.uint8)
    for at in np.ndindex(*x.shape[:-1]):
        for g in range(-(-d // GROUP)):
            lo, hi = g * GROUP, min(d, (g + 1) * GROUP)
            byte, codes = encode_group(x[at][lo:hi])
            out[at][lo // 2:hi // 2] = codes[0::2] | (codes[1::2] << 4)
            out[at][d // 2 + g] = byte
    return out


def decode(half, d: int) -> np.ndarray:
    """Values [..., d], float64, of half-rows' bytes."""
    half = np.asarray(half)
    codes = np.stack((half[..., :d // 2] & 15, half[..., :d // 2] >> 4), -1)
    codes = codes.reshape(half.shape[:-1] + (d,))
    value = np.where(codes & 8, -1.0, 1.0) * GRID[codes & 7]
    byte = half[..., d // 2:d // 2 + -(-d // GROUP)].astype(np.float64)
    scale = np.where(byte == 255, math.nan, 2.0 ** (byte - 127))
    return value * np.repeat(scale, GROUP, -1)[..., :d]


def canonical(cache: np.ndarray, layout: str) -> np.ndarray:
    """A view of a cache as [pages, slots in page, heads, K/V, bytes]."""
    if layout == "kv_first":
        return cache.transpose(1, 2, 3, 0, 4)
    if layout == "blocks_first":
        return cache.transpose(0, 2, 3, 1, 4)
    b, h, s, w = cache.shape
    return cache.reshape(b, h, s, 2, w // 2).transpose(0, 2, 1, 3, 4)


def attend(q, view, d: int, tables, lens, starts, scale: float):
    """Attention of ``q`` float64 [tokens, q_heads, d] over a canonical 4-bit cache.

    Returns ``(out, lse, reach, worst)``: ``reach`` [tokens, q_heads, d] is the weights' mean of
    the magnitudes of V, ``worst`` [tokens, q_heads] the largest sum of |q_j k_j| * scale over the
    seen tokens, which the tests derive tolerances from."""
    pages, bs, heads = view.shape[:3]
    shared = q.shape[1] // heads
    out, reach = np.zeros(q.shape), np.zeros(q.shape)
    lse, worst = np.full(q.shape[:2], -math.inf), np.zeros(q.shape[:2])
    for s in range(len(lens)):
        n, nq = int(lens[s]), int(starts[s + 1] - starts[s])
        at = [(t, int(tables[s][t // bs])) for t in range(n)]
        at = [(t, p) for t, p in at if 0 <= p < pages]
        if not at:
            continue
        t = np.array([x[0] for x in at])
        rows = decode(view[[x[1] for x in at], t % bs], d)  # [tokens, heads, 2, d]
        for i in range(nq):
            seen = t <= n - nq + i
            if not seen.any():
                continue
            for h in range(q.shape[1]):
                k, v = rows[seen, h // shared, 0], rows[seen, h // shared, 1]
                x = q[starts[s] + i, h]
                score = (k * x).sum(-1) * scale
                top = score.max()
                w = np.exp(score - top)
                row = starts[s] + i, h
                out[row] = (w[:, None] * v).sum(0) / w.sum()
                reach[row] = (w[:, None] * np.abs(v)).sum(0) / w.sum()
                lse[row] = top + math.log(w.sum())
                worst[row] = (np.abs(k * x).sum(-1) * scale).max()
    return out, lse, reach, worst


def plan_compaction(tables, counts, num_blocks: int):
    """``(tables, moves, used)``: the rewritten tables, the (src, dst) moves, the pages in use."""
    used = set()
    for row, n in zip(tables, counts):
        used |= {int(p) for p in row[:max(0, int(n))] if 0 <= p < num_blocks}
    u = len(used)
    holes = [p for p in range(u) if p not in used]
    movers = sorted(p for p in used if p >= u)
    moves = list(zip(movers, holes))
    new = dict(moves)
    out = [[new.get(int(p), int(p)) if c < int(n) else int(p) for c, p in enumerate(row)]
           for row, n in zip(tables, counts)]
    return out, moves, u
