"""Attention over full-width pages behind shared prefixes, the weights that tokens get, and eviction
by them, restated plainly: the tests' oracle.

Everything is computed in 64 bits on the CPU from the definitions in ``include/everserve_mi355x.h``:
attention head by head over the whole context, the choice of tokens by sorting.
"""

from __future__ import annotations

import math

import numpy as np


def canonical(cache, layout: str):
    """A view of a cache as [pages, slots in page, heads, K/V, elements] (numpy or torch)."""
    if layout == "kv_first":
        return cache.transpose(1, 2, 3, 0, 4)
    if layout == "blocks_first":
        return cache.transpose(0, 2, 3, 1, 4)
    b, h, s, w = cache.shape
    return cache.reshape(b, h, s, 2, w // 2).transpose(0, 2, 1, 3, 4)


def group_of(s: int, starts) -> int:
    """The group of sequence ``s``, -1 for none."""
    for g in range(len(starts) - 1):
        if starts[g] <= s < starts[g + 1]:
            return g
    return -1


def attend(q, view, tables, lens, starts, scale: float, prefix=None, mass=None):
    """Attention of ``q`` float64 [tokens, q_heads, d] over a canonical cache (float64).

    ``prefix`` is ``(tables, lens, starts)``. Returns a dict: ``out``, ``lse``; ``reach`` [tokens,
    q_heads, d], the weights' mean of the magnitudes of V; ``values`` [tokens, q_heads, d], the sum
    of those magnitudes; ``worst`` [tokens, q_heads], the largest sum of |q_j k_j| * scale over the
    seen tokens; and with ``mass`` (float64 [pages, heads, slots], changed in place) also
    ``gave`` and ``doubt`` of its shape: what a token got, and that times its rows' ``worst`` (at
    least 1)."""
    pages, bs, heads = view.shape[:3]
    shared = q.shape[1] // heads
    r = dict(out=np.zeros(q.shape), reach=np.zeros(q.shape), values=np.zeros(q.shape),
             lse=np.full(q.shape[:2], -math.inf), worst=np.zeros(q.shape[:2]))
    if mass is not None:
        r.update(gave=np.zeros(mass.shape), doubt=np.zeros(mass.shape))

    def places(table, n):
        return [(int(table[t // bs]), t % bs) for t in range(n)]

    for s in range(len(lens)):
        n, nq = int(lens[s]), int(starts[s + 1] - starts[s])
        g = -1 if prefix is None else group_of(s, prefix[2])
        ahead = [] if g < 0 else places(prefix[0][g], int(prefix[1][g]))
        at = [(p, o, -1) for p, o in ahead] + [(p, o, t) for t, (p, o) in
                                               enumerate(places(tables[s], n))]
        at = [x for x in at if 0 <= x[0] < pages]
        if mass is not None:
            for p, o, t in at:
                if t >= 0 and t >= n - nq:
                    mass[p, :, o] = 0
        if not at:
            continue
        page, off, pos = (np.array(x) for x in zip(*at))
        rows = view[page, off]  # [tokens, heads, 2, d]
        last = n - nq + np.arange(nq)
        seen = (pos[None] <= last[:, None]) | (pos < 0)[None]  # [queries, tokens]
        for h in range(q.shape[1]):
            k, v = rows[:, h // shared, 0], rows[:, h // shared, 1]
            x = q[starts[s]:starts[s + 1], h]
            for i in range(nq):
                see = seen[i]
                if not see.any():
                    continue
                part = k[see] * x[i]
                score = part.sum(-1) * scale
                top = score.max()
                w = np.exp(score - top)
                share = w / w.sum()
                row = starts[s] + i, h
                r["out"][row] = (share[:, None] * v[see]).sum(0)
                r["reach"][row] = (share[:, None] * np.abs(v[see])).sum(0)
                r["values"][row] = np.abs(v[see]).sum(0)
                r["lse"][row] = top + math.log(w.sum())
                r["worst"][row] = worst = (np.abs(part).sum(-1) * scale).max()
                if mass is not None:
                    for name, give in (("gave", share), ("doubt", share * max(1.0, worst))):
                        np.add.at(r[name], (page[see], h // shared, off[see]), give)
    if mass is not None:
        mass += r["gave"]
    return r


def order_of(x) -> tuple:
    """What sorts masses from the most to the least: no number first, -0 as 0."""
    return (0, 0.0) if math.isnan(x) else (1, -float(x) + 0.0)


def choose(mass, tables, n: int, budget: int, recent: int, pages: int):
    """The tokens of one sequence that stay, by the ``mass`` [pages, slots] of a layer and head."""
    bs = mass.shape[1]
    if n <= budget:
        return list(range(n))
    newest = n - recent

    def rank(t):
        p = int(tables[t // bs])
        return ((2, 0.0) if not 0 <= p < pages else order_of(mass[p, t % bs])), t

    others = sorted(range(newest), key=rank)[:budget - recent]
    return sorted(others) + list(range(newest, n))


def evict(views, mass, tables, lens, new_tables, budget: int, recent: int):
    """Cut sequences short in place: ``views`` are the layers' canonical caches, ``mass`` [layers,
    pages, heads, slots]. Returns ``(lens, kept)``."""
    layers, pages, heads, bs = mass.shape
    kept = np.full((layers, len(lens), heads, budget), -1, dtype=np.int32)
    old = [v.copy() for v in views], mass.copy()
    out = []
    for s, n in enumerate(lens):
        n = int(min(max(int(n), 0), tables.shape[1] * bs))
        out.append(min(n, budget))
        for la in range(layers):
            for h in range(heads):
                stay = choose(old[1][la, :, h], tables[s], n, budget, recent, pages)
                kept[la, s, h, :len(stay)] = stay
                for j, t in enumerate(stay):
                    a, b = int(tables[s][t // bs]), int(new_tables[s][j // bs])
                    if 0 <= a < pages and 0 <= b < pages:
                        views[la][b, j % bs, h] = old[0][la][a, t % bs, h]
                        mass[la, b, h, j % bs] = old[1][la, a, h, t % bs]
    return np.array(out, dtype=np.int32), kept
