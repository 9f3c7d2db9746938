"""A paged K/V cache in device memory (no counterpart in the reference).

The paged runtime's pages live on the host or on disk and are read in long
scans; these stay in HBM, grow by a token per step and are read by the token
that follows.  The cache owns the pools; which pages a sequence has, and which
are free, is the caller's bookkeeping (``page_table``).
"""

from __future__ import annotations

import torch

from . import _native
from .kernels.blocks import append_kv_blocks
from .kernels.decode import paged_decode_attention
from .kernels.prefill import paged_prefill_attention
from .kernels.rows import MAX_PAGE_TOKENS, append_kv, check_sequences, normalize_rotate_append, read_kv


class DeviceKVCache:
    """K and V pools ``[num_pages, page_tokens, kv_heads, head_dim]``.

    ``storage_dtype="int8"`` holds INT8 values and a float16 scale per row and
    head, ``"float8_e4m3fn"`` e4m3 values and a power-of-two scale per
    ``block_tokens`` rows (by default the most of 64, 32 and 16 that divide a page)
    and head; by default the pools hold ``dtype``.  Rows go into a 16-bit or INT8
    cache slot by slot (``append``), into any sequence by sequence (``extend``).  In memory a page is head by head
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
        block_tokens: int | None = None,
        device: torch.device | str = "cuda",
    ) -> None:
        _native.dtype_code(dtype)
        if min(num_pages, page_tokens, kv_heads) < 1:
            raise ValueError("num_pages, page_tokens and kv_heads must be positive")
        if page_tokens > MAX_PAGE_TOKENS or num_pages * page_tokens > 2**31 - 1:
            raise ValueError(f"pages have at most {MAX_PAGE_TOKENS} rows, the cache fewer than 2^31")
        if head_dim % 8 or not 16 <= head_dim <= 256:
            raise ValueError(f"head_dim must be a multiple of 8 in [16, 256], got {head_dim}")
        if storage_dtype not in (None, "int8", "float8_e4m3fn", str(dtype).removeprefix("torch.")):
            raise ValueError("storage_dtype must be 'int8', 'float8_e4m3fn' or the cache's dtype")
        e4m3 = storage_dtype == "float8_e4m3fn"
        if e4m3:
            if block_tokens is None:
                block_tokens = next((n for n in (64, 32) if page_tokens % n == 0), 16)
            if block_tokens < 16 or block_tokens & (block_tokens - 1) or page_tokens % block_tokens:
                raise ValueError("block_tokens must be a power of two from 16 on that divides page_tokens")
        elif block_tokens is not None:
            raise ValueError("only e4m3 pages have blocks")
        self.dtype = dtype
        self.page_tokens = page_tokens
        self.int8 = storage_dtype == "int8"
        self.e4m3 = e4m3
        self.block_tokens = block_tokens

        def pool(shape, pool_dtype):
            return torch.zeros(shape, dtype=pool_dtype, device=device).transpose(1, 2)

        shape = (num_pages, kv_heads, page_tokens, head_dim)
        stored = torch.int8 if self.int8 else torch.float8_e4m3fn if e4m3 else dtype
        self.k_pages, self.v_pages = pool(shape, stored), pool(shape, stored)
        self.device = self.k_pages.device
        self.k_scales = self.v_scales = None
        if self.int8:
            self.k_scales, self.v_scales = pool(shape[:3], torch.float16), pool(shape[:3], torch.float16)
        if e4m3:
            shape = (num_pages, kv_heads, page_tokens // block_tokens)
            self.k_scales, self.v_scales = (pool(shape, torch.uint8).view(torch.float8_e8m0fnu) for _ in range(2))

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

    def _refuse_slots(self) -> None:
        if self.e4m3:
            raise ValueError("an e4m3 cache takes rows sequence by sequence: use extend()")

    def extend(self, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
               cu_tokens: torch.Tensor | None = None) -> None:
        """Append rows ``cu_tokens[s] .. cu_tokens[s + 1] - 1`` (one each without) to every sequence ``s``.

        ``lengths`` hold the new rows already, as for ``attend``; see :func:`seqattn.kernels.append_kv_blocks`.
        """
        if self.e4m3:
            return append_kv_blocks(k, v, self.k_pages, self.v_pages, self.k_scales, self.v_scales, page_table, lengths,
                                    cu_tokens)
        check_sequences(page_table, lengths, cu_tokens, k.shape[0], self.page_tokens, k, "k")
        rows = torch.arange(k.shape[0], device=k.device)
        if cu_tokens is None:
            sequences, positions = rows, lengths.to(torch.int64) - 1
        else:
            # Rows past the last sequence are of none, which has no slots.
            sequences = torch.searchsorted(cu_tokens[1:], rows, right=True)
            ends = torch.cat([lengths.to(torch.int64) - cu_tokens[1:], lengths.new_zeros(1, dtype=torch.int64)])
            positions = ends[sequences] + rows
        # A length past the table's row has no page there either.
        self.append(k, v, self.slots(page_table, sequences, positions))

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        self._refuse_slots()
        append_kv(k, v, self.k_pages, self.v_pages, slots, k_scales=self.k_scales, v_scales=self.v_scales)

    def normalize_rotate_append(self, q, k, v, slots, positions=None, frequencies=None, **rotation) -> torch.Tensor:
        self._refuse_slots()
        return normalize_rotate_append(q, k, v, self.k_pages, self.v_pages, slots, positions, frequencies,
                                       k_scales=self.k_scales, v_scales=self.v_scales, **rotation)

    def read(self, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        return read_kv(self.k_pages, self.v_pages, slots, k_scales=self.k_scales, v_scales=self.v_scales,
                       dtype=self.dtype)

    def attend(self, q: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
               cu_tokens: torch.Tensor | None = None, **options):
        """One token per sequence (:func:`paged_decode_attention`), or with ``cu_tokens`` several."""
        scales = dict(k_scales=self.k_scales, v_scales=self.v_scales)
        if cu_tokens is None:
            return paged_decode_attention(q, self.k_pages, self.v_pages, page_table, lengths, **scales, **options)
        return paged_prefill_attention(q, self.k_pages, self.v_pages, page_table, lengths, cu_tokens, **scales, **options)


__all__ = ["DeviceKVCache"]
