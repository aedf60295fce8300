"""Sequences of a rank's caches cut to a budget of tokens, by the attention weight that they gathered.

Every layer and KV head keeps tokens of its own: the newest ones and, of the others, those with the
most mass, the weight that the attentions so far gave them
(:meth:`everserve_amd.state.full.FullCache.attend` with ``mass``). Their rows move to new pages, in
their order, so the sequence goes on as a shorter one: its length is the budget, its block table the
new pages, and the old pages are free, unless other sequences share them: they are only read.

Keys keep the positions that they were rotated for; ``Eviction.kept`` says which tokens a head holds.
The reference keeps whole contexts and has no counterpart.
"""

from __future__ import annotations

from dataclasses import dataclass

from everserve_amd.state.pages import PageMover, _kernels


@dataclass(frozen=True)
class Eviction:
    """What an eviction left, in device tensors (int32)."""

    lens: object
    """The sequences' new lengths, [seqs]."""
    kept: object
    """The tokens that stayed, ascending: [layers, seqs, heads, budget], -1 past a sequence's."""


class Evictor(PageMover):
    """:class:`everserve_amd.state.pages.PageMover` that also cuts sequences short.

    Caches of any element type, 4-bit caches among them, whose rows are contiguous.

    Raises:
        ValueError: for layers that differ, or that the kernels cannot address.
    """

    def __init__(self, layers, layout=None) -> None:
        super().__init__(layers, layout)
        if self.strides[4] != 1:
            raise ValueError(f"a row's elements must be contiguous: strides {self.strides}")

    def evict(self, block_tables, seq_lens, new_tables, budget: int, mass,
              recent: int = 0) -> Eviction:
        """Cut each sequence to ``budget`` tokens. Of a longer one the ``recent`` last stay, and of
        the others those with the most ``mass``, of equal ones the first.

        ``block_tables`` and ``new_tables`` (int32 [seqs, pages]) name the pages that a sequence has
        and those that it gets; the latter must have room for the budget, be named once, and none
        of them be in ``block_tables``. Shorter sequences move as they are. ``mass`` (f32 [layers,
        num_blocks, heads, block_size], contiguous) moves with the rows. Pages outside the cache hold
        nothing: their tokens go first, and nothing moves from or to them. One of them that stays
        all the same (one of the newest, or where there are no more than the budget) counts in the
        new length, and its new slot holds what it held, for attention to see: evict sequences whose
        pages are all there. Two launches on the current stream; lengths and tables are read on the
        device, so it may be captured.

        Masses of pages that are filled by other means are the caller's to set: :meth:`copy`,
        :meth:`compact` and a restore move rows alone (``mass[:, dst] = mass[:, src]`` with a
        copy's or a plan's pages, 0 for restored ones)."""
        return Eviction(*_kernels().evict(self._ptrs, self.num_blocks, self.num_heads,
                                          self.head_dim, self.block_size, self._strides, self.elem,
                                          block_tables, seq_lens, new_tables, budget, mass, recent))
