"""One layer's paged cache held in 4 bits: rows written and read, and attention over them.

A half-row (the K or V of one slot and head) is ``head_dim / 2`` bytes of E2M1 codes, one
power-of-two scale byte for each 32 elements, and zeros up to a multiple of 4 bytes: the MXFP4 of
the Open Compute microscaling formats, which gfx950's conversions read as it is. 128 elements are 68
bytes instead of 256. The scale that a write chooses is the least power of two that brings the
group's largest magnitude to 7 or below. That text takes the largest's exponent less 2: the same,
but where the largest is between 7 and 8 steps of it, which then is cut to 6.

The cache is a uint8 tensor of any of the three layouts with the half-row's bytes in the place of
the head size, so everything that moves a cache moves it as it stands: the stager, the restore, the
gathers, the scatters and the page copies.

The reference has no counterpart: its caches are its engine's, at 8 bits or more.
"""

from __future__ import annotations

import ctypes

from everserve_amd.state.paged import CacheLayout, PagedKV, strides_of

GROUP = 32
"""Elements that share a scale."""
MIN_DIM, MAX_DIM = 16, 256


def row_bytes(head_dim: int) -> int:
    """Bytes of a half-row of ``head_dim`` elements.

    Raises:
        ValueError: for a head size that is no multiple of 8 from 16 to 256.
    """
    if head_dim % 8 or not MIN_DIM <= head_dim <= MAX_DIM:
        raise ValueError(f"head size {head_dim}: a multiple of 8 from {MIN_DIM} to {MAX_DIM}")
    return (head_dim // 2 + -(-head_dim // GROUP) + 3) // 4 * 4


def cache_shape(layout: CacheLayout | str, num_blocks: int, block_size: int, heads: int,
                head_dim: int) -> tuple[int, ...]:
    """The shape of a 4-bit cache of ``layout``."""
    half = row_bytes(head_dim)
    return {
        CacheLayout.KV_FIRST: (2, num_blocks, block_size, heads, half),
        CacheLayout.BLOCKS_FIRST: (num_blocks, 2, block_size, heads, half),
        CacheLayout.COMBINED: (num_blocks, heads, block_size, 2 * half),
    }[CacheLayout(layout)]


class Fp4Cache:
    """A layer's 4-bit cache: the tensor, and its geometry checked and converted once.

    ``layout`` is needed only where a shape fits two layouts (a ``blocks_first`` cache of two
    pages is otherwise taken as ``kv_first``, as everywhere).

    Raises:
        ValueError: for a tensor that is no uint8 cache of ``head_dim`` elements a half-row, or
            whose strides the kernels cannot address.
    """

    def __init__(self, tensor, head_dim: int, layout: CacheLayout | str | None = None) -> None:
        import torch

        half = row_bytes(head_dim)
        if tensor.dtype != torch.uint8:
            raise ValueError(f"a 4-bit cache is uint8, not {tensor.dtype}")
        if layout is None:
            layout = PagedKV.of(tensor).layout
        self.layout = CacheLayout(layout)
        shape = tuple(int(x) for x in tensor.shape)
        dims = {
            CacheLayout.KV_FIRST: (5, 0, (1, 2, 3)),
            CacheLayout.BLOCKS_FIRST: (5, 1, (0, 2, 3)),
            CacheLayout.COMBINED: (4, None, (0, 2, 1)),
        }
        rank, kv, (b, s, h) = dims[self.layout]
        width = 2 * half if kv is None else half
        if len(shape) != rank or shape[-1] != width or (kv is not None and shape[kv] != 2):
            raise ValueError(f"a {self.layout.value} cache of head size {head_dim} ends in {width} "
                             f"bytes; this one has the shape {shape}")
        self.tensor = tensor
        self.head_dim = head_dim
        self.num_blocks, self.block_size, self.num_heads = shape[b], shape[s], shape[h]
        self.strides = strides_of(self.layout, tensor.stride(), half)
        if self.strides[4] != 1 or any(x % 4 for x in self.strides[:4]):
            raise ValueError(f"a half-row's bytes must be contiguous and start on 4 bytes: strides "
                             f"{self.strides}")
        self._strides = (ctypes.c_int64 * 5)(*self.strides)  # converted once for every call

    @classmethod
    def empty(cls, num_blocks: int, block_size: int, heads: int, head_dim: int,
              layout: CacheLayout | str = CacheLayout.COMBINED, device="cuda") -> "Fp4Cache":
        """A new cache, every row of it zeros. ``combined`` keeps a head's page contiguous; single
        tokens over many heads are read faster where a token's heads lie side by side, as in the
        other two (64 sequences of 1 to 8 Ki tokens, 8 heads of 128: 78 us for 91)."""
        import torch

        shape = cache_shape(layout, num_blocks, block_size, heads, head_dim)
        return cls(torch.zeros(shape, dtype=torch.uint8, device=device), head_dim, layout)

    def write(self, slots, key, value) -> None:
        """Round ``key`` and ``value`` ([n, heads, head_dim]) to 4 bits and write them at ``slots``
        (int64 [n], distinct; a slot outside the cache is padding). One launch on the current
        stream."""
        shape = key.shape
        if len(shape) != 3 or shape[1] != self.num_heads or shape[2] != self.head_dim:
            raise ValueError(f"write: rows of shape {tuple(key.shape)}, expected "
                             f"[n, {self.num_heads}, {self.head_dim}]")
        _kernels().fp4_write_rows(key, value, slots, self.tensor, self.num_blocks, self.block_size,
                                  self._strides)

    def read(self, slots, dtype):
        """``(key, value)`` [n, heads, head_dim] of ``dtype`` at ``slots`` (int64 [n]); zeros for a
        slot outside the cache. One launch on the current stream."""
        return _kernels().fp4_read_rows(self.tensor, self.num_blocks, self.block_size,
                                        self.num_heads, self.head_dim, self._strides, slots, dtype)

    def attend(self, q, block_tables, seq_lens, q_starts=None, max_q: int | None = None,
               scale: float | None = None, max_len: int = 0, out=None, return_lse: bool = False):
        """Attention of ``q`` ([tokens, q_heads, head_dim], bf16 or f16) over the pages of
        ``block_tables``: :meth:`everserve_amd.kernels.Kernels.fp4_attend` with this cache."""
        if q.dim() != 3 or q.shape[2] != self.head_dim:
            raise ValueError(f"attend: queries of shape {tuple(q.shape)}, expected "
                             f"[tokens, heads, {self.head_dim}]")
        return _kernels().fp4_attend(q, self.tensor, self.num_blocks, self.block_size,
                                     self.num_heads, self._strides, block_tables, seq_lens,
                                     q_starts, max_q, scale, max_len, out, return_lse)


def _kernels():
    """The loaded kernels (raises when they cannot load: no quiet fallback)."""
    from everserve_amd import kernels

    return kernels.load()
