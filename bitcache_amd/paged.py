"""A paged compressed KV cache: sequences of their own lengths in one pool of pages."""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from bitcache_amd import _C, _require_extension, functional


class PagedBitCache:
    """Pool of cache pages for one transformer layer of a server.

    BitCache holds one ring per batch row; here sequences of any lengths share a pool
    of ``n_pages`` pages of ``page_size`` slots (a multiple of 64).  The caller assigns
    pages: a token goes to slot ``page * page_size + offset``, and a sequence is a row
    of page numbers and a length.  The encoding is BitCache's.

    Args:
        n_pages, page_size: the pool.
        n_heads, head_dim, device, compensated, n_kv_heads: as BitCache.
    """

    def __init__(self, n_pages: int, page_size: int, n_heads: int, head_dim: int,
                 device: str = "cuda", compensated: bool = True,
                 n_kv_heads: Optional[int] = None) -> None:
        _require_extension()
        assert head_dim % 32 == 0, "head_dim must be a multiple of 32"
        assert head_dim <= 256, "head_dim must be <= 256"
        assert n_pages > 0, "n_pages must be > 0"
        assert page_size > 0 and page_size % 64 == 0, "page_size must be a multiple of 64"
        self.n_pages = n_pages
        self.page_size = page_size
        self.n_heads = n_heads
        self.n_kv_heads = n_heads if n_kv_heads is None else n_kv_heads
        assert self.n_kv_heads > 0 and n_heads % self.n_kv_heads == 0, \
            "n_heads must be a multiple of n_kv_heads"
        self.head_dim = head_dim
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise RuntimeError("PagedBitCache needs a ROCm device (got %s)" % self.device)
        self.compensated = compensated
        n = n_pages * self.n_kv_heads * page_size
        u8 = dict(dtype=torch.uint8, device=self.device)
        self._k_bin = torch.zeros(n * _C.sizeof_binary_vec(), **u8)
        self._v_bin = torch.zeros(n * _C.sizeof_binary_vec(), **u8)
        self._k_res = torch.zeros(n * _C.sizeof_residual_vec(), **u8) if compensated else None
        self._v_res = torch.zeros(n * _C.sizeof_residual_vec(), **u8) if compensated else None

    def slots(self, block_tables: Tensor, positions: Tensor) -> Tensor:
        """Slots [batch] int64 of position positions[b] of the sequence block_tables[b]
        (the token a decode step appends); -1, which goes nowhere, for a position outside
        the table or on a page outside the pool."""
        width = block_tables.shape[1]
        if width == 0:
            return torch.full_like(positions, -1, dtype=torch.int64)
        positions = positions.long()
        entry = torch.div(positions, self.page_size, rounding_mode="floor")
        page = block_tables.gather(1, entry.clamp(0, width - 1)[:, None])[:, 0].long()
        known = (positions >= 0) & (entry < width) & (page >= 0) & (page < self.n_pages)
        return torch.where(known, page * self.page_size + positions % self.page_size, -1)

    def append(self, K: Tensor, V: Tensor, slots: Tensor) -> None:
        """Encode K, V [tokens, n_kv_heads, head_dim] into slots (functional.paged_append)."""
        self._validate(K, self.n_kv_heads, "K")
        self._validate(V, self.n_kv_heads, "V")
        functional.paged_append(K, V, slots, self._k_bin, self._k_res, self._v_bin, self._v_res,
                                self.page_size)

    def append_rotary(self, Q: Tensor, K: Tensor, V: Tensor, positions: Tensor, slots: Tensor,
                      cos: Tensor, sin: Tensor, *, q_weight: Optional[Tensor] = None,
                      k_weight: Optional[Tensor] = None, eps: float = 1e-6,
                      interleaved: bool = False) -> Tensor:
        """Norm and rotate Q and K, encode K and V into slots; returns the rotated Q
        (functional.rotary_append)."""
        self._validate(Q, self.n_heads, "Q")
        self._validate(K, self.n_kv_heads, "K")
        self._validate(V, self.n_kv_heads, "V")
        return functional.rotary_append(Q, K, V, positions, slots, cos, sin, self._k_bin,
                                        self._k_res, self._v_bin, self._v_res, self.page_size,
                                        q_weight=q_weight, k_weight=k_weight, eps=eps,
                                        interleaved=interleaved)

    def attend(self, Q: Tensor, block_tables: Tensor, seq_lens: Tensor, max_seq_len: int,
               shared_len: int = 0) -> Tensor:
        """Attention of Q [batch, n_heads, head_dim] over each sequence's keys
        (functional.paged_attention)."""
        self._validate(Q, self.n_heads, "Q")
        return functional.paged_attention(Q, self._k_bin, self._k_res, self._v_bin, self._v_res,
                                          block_tables, seq_lens, max_seq_len, self.page_size,
                                          n_kv_heads=self.n_kv_heads, shared_len=shared_len)

    def reset(self) -> None:
        """Clear the pool."""
        for b in (self._k_bin, self._v_bin, self._k_res, self._v_res):
            if b is not None:
                b.zero_()

    @property
    def memory_bytes(self) -> int:
        """Bytes allocated for the pool."""
        return sum(b.numel() for b in (self._k_bin, self._v_bin, self._k_res, self._v_res)
                   if b is not None)

    def _validate(self, x: Tensor, heads: int, name: str) -> None:
        assert x.dim() == 3 and x.shape[1:] == (heads, self.head_dim), \
            f"{name} shape {tuple(x.shape)} is not [tokens, {heads}, {self.head_dim}]"

    def __repr__(self) -> str:
        mode = "compensated" if self.compensated else "binary"
        return (f"PagedBitCache(n_pages={self.n_pages}, page_size={self.page_size}, "
                f"n_heads={self.n_heads}, n_kv_heads={self.n_kv_heads}, "
                f"head_dim={self.head_dim}, mode={mode}, mem={self.memory_bytes / 1024:.1f}KB)")
