"""Pages of a rank's caches moved inside them: copied for sequences that part, and packed.

A page (a block of a block table) is the same id in every layer. Sequences that share a prefix name
the same pages; one that is about to write into a shared page first gets a copy of it
(:meth:`PageMover.copy`). A cache whose used pages lie scattered is packed to its front
(:meth:`PageMover.compact`): the pages past the number in use move into the holes before it, every
block table is rewritten, and the pages from there on are free, for a smaller cache or for another
owner. Nothing waits for the device: the plan's counts stay there and the copy reads them.

The reference leaves pages to its engine and has no counterpart.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Sequence

from everserve_amd.state.paged import CacheLayout, PagedKV, strides_of


@dataclass(frozen=True)
class Compaction:
    """What a compaction did, in device tensors (int32)."""

    tables: object
    """The block tables with the pages' new ids, like those given."""
    src: object
    """The ids that pages had, [num_blocks // 2], -1 past the moves."""
    dst: object
    """The ids that they got."""
    sizes: object
    """[pages in use, pages moved]: pages from ``sizes[0]`` on are free."""


class PageMover:
    """The pages of a rank's caches (one tensor a layer, of one shape, dtype and strides).

    Caches of any element type, 4-bit caches among them, in any of the three layouts. ``layout`` is
    needed only where a shape fits two.

    Raises:
        ValueError: for layers that differ, or that the kernels cannot address.
    """

    def __init__(self, layers: Sequence, layout: CacheLayout | str | None = None) -> None:
        import torch

        if not layers:
            raise ValueError("no layers")
        first = layers[0]
        for t in layers:
            if (t.shape != first.shape or t.stride() != first.stride() or t.dtype != first.dtype
                    or t.device != first.device):
                raise ValueError("every layer's cache must have one shape, strides, dtype and "
                                 "device")
        shape = tuple(int(x) for x in first.shape)
        if layout is None:
            layout = PagedKV.of(first).layout
        self.layout = CacheLayout(layout)
        if self.layout is CacheLayout.COMBINED:
            if len(shape) != 4 or shape[3] % 2:
                raise ValueError(f"no combined cache: shape {shape}")
            self.num_blocks, self.num_heads, self.block_size = shape[:3]
            self.head_dim = shape[3] // 2
        else:
            kv = 0 if self.layout is CacheLayout.KV_FIRST else 1
            if len(shape) != 5 or shape[kv] != 2:
                raise ValueError(f"no {self.layout.value} cache: shape {shape}")
            self.num_blocks, self.block_size, self.num_heads = shape[1 - kv], *shape[2:4]
            self.head_dim = shape[4]
        self.strides = strides_of(self.layout, first.stride(), self.head_dim)
        self.elem = first.element_size()
        if self.elem not in (1, 2, 4):
            raise ValueError(f"elements of {self.elem} bytes: 1, 2 or 4")
        # the copy takes any base; the gathers read such caches in aligned words of 16 bytes
        if all(s * self.elem % 16 == 0 for s in self.strides[:4]) and any(
                t.data_ptr() % 16 for t in layers):
            raise ValueError("caches with strides of whole 16-byte words must start on one")
        self._layers = list(layers)  # the table holds their addresses
        self._strides = (ctypes.c_int64 * 5)(*self.strides)  # converted once for every call
        self._ptrs = torch.tensor([t.data_ptr() for t in layers], dtype=torch.long,
                                  device=first.device)

    def copy(self, src, dst, count=None) -> None:
        """Copy page ``src[i]`` to page ``dst[i]`` (int32, on the device) in every layer. ``count``
        (int32 [1], on the device) cuts the list short. A pair with an id outside the cache moves
        nothing; destinations must be distinct, and none a pair's source. One launch on the
        current stream."""
        _kernels().copy_blocks(self._ptrs, src, dst, self.num_blocks, self.num_heads,
                               self.head_dim, self.block_size, self._strides, self.elem, count)

    def plan(self, block_tables, counts=None) -> Compaction:
        """The moves that pack the pages that ``block_tables`` name (int32 [rows, width], of row r
        the first ``counts[r]`` entries) to the caches' front, without moving them."""
        return Compaction(*_kernels().plan_compaction(block_tables, counts, self.num_blocks))

    def compact(self, block_tables, counts=None) -> Compaction:
        """:meth:`plan`, and the pages moved. The tables given are left as they are; from here on
        the returned ones hold. Every page in use must be in ``block_tables``."""
        plan = self.plan(block_tables, counts)
        if plan.src.numel():
            self.copy(plan.src, plan.dst, plan.sizes[1:])
        return plan


def _kernels():
    """The loaded kernels (raises when they cannot load: no quiet fallback)."""
    from everserve_amd import kernels

    return kernels.load()
