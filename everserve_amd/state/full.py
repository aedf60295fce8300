"""Attention over one layer's paged cache at full width, for batches that share prefixes.

Sequences of a batch often begin alike: samples of one prompt, questions about one document, a system
prompt. Their block tables then name the same pages, and an attention that takes each sequence by
itself reads them once for every sequence. Here a group's prefix is named once
(:class:`SharedPrefix`): its pages are read once for the queries of all its sequences, whose own pages
follow it, and the two parts of each query's softmax are joined.

An attention can also say what it used: with ``mass`` it adds to every token of the cache the weight
that the call's queries gave it, which :class:`everserve_amd.state.evict.Evictor` goes by.

The reference leaves attention to its engine and has no counterpart.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

from everserve_amd.state.paged import CacheLayout, PagedKV, strides_of

MIN_DIM, MAX_DIM = 16, 256


@dataclass(frozen=True)
class SharedPrefix:
    """What groups of a batch's sequences see ahead of their own tokens (int32, on the device)."""

    block_tables: object
    """The prefixes' pages, [groups, pages], a row contiguous."""
    lens: object
    """The prefixes' lengths, [groups]. They need not fill their last page: what follows it there is
    not seen."""
    starts: object
    """[groups + 1], ascending: group g has the sequences ``starts[g]`` to ``starts[g + 1] - 1`` of
    the batch. Sequences of no group have no prefix."""
    max_len: int = 0
    """At least the longest length, if given; as the ``max_len`` of a call."""


class FullCache:
    """A layer's cache of bf16 or f16 rows: the tensor, and its geometry checked and converted once.

    The tensor may be any of the three layouts, or a view with other strides whose rows are
    contiguous and start on 16 bytes. ``layout`` is needed only where a shape fits two (a
    ``blocks_first`` cache of two pages is otherwise taken as ``kv_first``, as everywhere).

    Raises:
        ValueError: for a tensor of another type or shape, or that the kernels cannot address.
    """

    def __init__(self, tensor, layout: CacheLayout | str | None = None) -> None:
        import torch

        if tensor.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"a full-width cache is bf16 or f16, not {tensor.dtype}")
        self.layout = PagedKV.of(tensor).layout if layout is None else CacheLayout(layout)
        shape = tuple(int(x) for x in tensor.shape)
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
        if self.head_dim % 8 or not MIN_DIM <= self.head_dim <= MAX_DIM:
            raise ValueError(f"head size {self.head_dim}: a multiple of 8 from {MIN_DIM} to "
                             f"{MAX_DIM}")
        self.strides = strides_of(self.layout, tensor.stride(), self.head_dim)
        if self.strides[4] != 1 or any(s % 8 for s in self.strides[:4]) or (
                tensor.numel() and tensor.data_ptr() % 16):
            raise ValueError(f"rows must be contiguous and start on 16 bytes: strides "
                             f"{self.strides}")
        self.tensor = tensor
        self._strides = (ctypes.c_int64 * 5)(*self.strides)  # converted once for every call

    def attend(self, q, block_tables, seq_lens, q_starts=None, max_q: int | None = None,
               scale: float | None = None, max_len: int = 0, out=None, return_lse: bool = False,
               prefix: SharedPrefix | None = None, mass=None):
        """Attention of ``q`` ([tokens, q_heads, head_dim] of the cache's type) over the pages of
        ``block_tables``, behind those of ``prefix``: :meth:`everserve_amd.kernels.Kernels.attend`
        with this cache."""
        if q.dim() != 3 or q.shape[2] != self.head_dim:
            raise ValueError(f"attend: queries of shape {tuple(q.shape)}, expected "
                             f"[tokens, heads, {self.head_dim}]")
        return _kernels().attend(q, self.tensor, self.num_blocks, self.block_size, self.num_heads,
                                 self._strides, block_tables, seq_lens, q_starts, max_q, scale,
                                 max_len, out, return_lse, prefix, mass)


def _kernels():
    """The loaded kernels (raises when they cannot load: no quiet fallback)."""
    from everserve_amd import kernels

    return kernels.load()
