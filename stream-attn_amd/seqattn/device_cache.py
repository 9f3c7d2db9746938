"""A paged K/V cache in device memory (no counterpart in the reference).

The paged runtime's pages live on the host or on disk and are read in long
scans; these stay in HBM, grow by a token per step and are read by the token
that follows.  The cache owns the pools; which pages a sequence has, and which
are free, is the caller's bookkeeping (``page_table``).
"""

from __future__ import annotations

import torch

from . import _native
from .kernels.decode import paged_decode_attention
from .kernels.rows import MAX_PAGE_TOKENS, append_kv, normalize_rotate_append, read_kv


class DeviceKVCache:
    """K and V pools ``[num_pages, page_tokens, kv_heads, head_dim]``.

    ``storage_dtype="int8"`` holds INT8 values and a float16 scale per row and
    head; by default the pools hold ``dtype``.  In memory a page is head by head
    (the rows of one head follow each other).  The arguments of the methods are
    those of the functions in :mod:`seqattn.kernels` that they call.
    """

    def __init__(
        self,
        num_pages: int,
        page_tokens: int,
        kv_heads: int,
        head_dim: int,
        *,
        dtype: torch.dtype = torch.bfloat16,
        storage_dtype: str | None = None,
        device: torch.device | str = "cuda",
    ) -> None:
        _native.dtype_code(dtype)
        if min(num_pages, page_tokens, kv_heads) < 1:
            raise ValueError("num_pages, page_tokens and kv_heads must be positive")
        if page_tokens > MAX_PAGE_TOKENS or num_pages * page_tokens > 2**31 - 1:
            raise ValueError(f"pages have at most {MAX_PAGE_TOKENS} rows, the cache fewer than 2^31")
        if head_dim % 8 or not 16 <= head_dim <= 256:
            raise ValueError(f"head_dim must be a multiple of 8 in [16, 256], got {head_dim}")
        if storage_dtype not in (None, "int8", str(dtype).removeprefix("torch.")):
            raise ValueError("storage_dtype must be 'int8' or the cache's dtype")
        self.dtype = dtype
        self.page_tokens = page_tokens
        self.int8 = storage_dtype == "int8"

        def pool(shape, pool_dtype):
            return torch.zeros(shape, dtype=pool_dtype, device=device).transpose(1, 2)

        shape = (num_pages, kv_heads, page_tokens, head_dim)
        stored = torch.int8 if self.int8 else dtype
        self.k_pages, self.v_pages = pool(shape, stored), pool(shape, stored)
        self.device = self.k_pages.device
        self.k_scales = pool(shape[:3], torch.float16) if self.int8 else None
        self.v_scales = pool(shape[:3], torch.float16) if self.int8 else None

    @property
    def num_pages(self) -> int:
        return self.k_pages.shape[0]

    @property
    def bytes(self) -> int:
        """Device memory of the pools."""
        pools = (self.k_pages, self.v_pages, self.k_scales, self.v_scales)
        return sum(t.numel() * t.element_size() for t in pools if t is not None)

    def slots(self, page_table: torch.Tensor, sequences: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        """int64 slots of ``positions`` of ``sequences`` (rows of ``page_table``); -1 where the table has no page."""
        rows, columns = page_table.shape
        sequences, positions = sequences.to(torch.int64), positions.to(torch.int64)
        column = torch.div(positions, self.page_tokens, rounding_mode="floor")
        held = (sequences >= 0) & (sequences < rows) & (column >= 0) & (column < columns)
        if not rows or not columns:
            return torch.full_like(positions, -1)
        pages = page_table.to(torch.int64)[sequences.clamp(0, rows - 1), column.clamp(0, columns - 1)]
        return torch.where(held & (pages >= 0), pages * self.page_tokens + positions % self.page_tokens, -1)

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        append_kv(k, v, self.k_pages, self.v_pages, slots, k_scales=self.k_scales, v_scales=self.v_scales)

    def normalize_rotate_append(self, q, k, v, slots, positions=None, frequencies=None, **rotation) -> torch.Tensor:
        return normalize_rotate_append(q, k, v, self.k_pages, self.v_pages, slots, positions, frequencies,
                                       k_scales=self.k_scales, v_scales=self.v_scales, **rotation)

    def read(self, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        return read_kv(self.k_pages, self.v_pages, slots, k_scales=self.k_scales, v_scales=self.v_scales,
                       dtype=self.dtype)

    def attend(self, q: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, **options):
        return paged_decode_attention(q, self.k_pages, self.v_pages, page_table, lengths, k_scales=self.k_scales,
                                      v_scales=self.v_scales, **options)


__all__ = ["DeviceKVCache"]
