"""K and V rows quantised into e4m3 pages as they are written.

e4m3 pages are ``float8_e4m3fn [num_pages, page_tokens, kv_heads, head_dim]``
tensors, with ``float8_e8m0fnu [num_pages, page_tokens / block_tokens, kv_heads]``
scales: powers of two, one per block of ``block_tokens`` rows (a power of two from
16 on) and K/V head.  A scale belongs to a block's rows together, so rows come
sequence by sequence instead of slot by slot.  No counterpart in the reference.

The launch is asynchronous on torch's current stream of the operands' device and
allocates nothing, so it can be captured into a graph.
"""

from __future__ import annotations

import struct

import torch

from .. import _native
from .rows import check_pools, check_rows, check_sequences, refuse_tangents

# sa_append_blocks_args: 9 pointers, 13 strides and counts, 8 int32.
_APPEND_ARGS = struct.Struct("=9Q13q8i")


def append_kv_blocks(
    k: torch.Tensor,
    v: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    k_scales: torch.Tensor,
    v_scales: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    cu_tokens: torch.Tensor | None = None,
) -> None:
    """Quantise rows ``k, v [tokens, kv_heads, head_dim]`` into e4m3 pages, as the last rows of their sequences.

    Sequence ``s`` has rows ``cu_tokens[s] .. cu_tokens[s + 1] - 1`` (int32
    ``[sequences + 1]``, non-decreasing from 0; without it one row each), which
    become its rows up to ``lengths[s] - 1`` (int32 ``[sequences]``, the new rows
    included): row ``j`` of a sequence is row ``j % page_tokens`` of page
    ``page_table[s, j // page_tokens]`` (int32 ``[sequences, max_pages]``), as the
    attention reads it.  Rows below position 0, past the table's row or in a page
    outside the pool are not written, rows past ``cu_tokens[-1]`` not read.

    A block's scale is the smallest power of two (at least 2^-126) of which 448
    reach the call's largest finite magnitude in the block.  Where the block has
    rows before the first new one it does not fall below the scale it has, and
    where it grows those rows are rounded again.  Values are rounded to
    nearest even in units of the scale; one that is not finite becomes NaN.  A
    page that is written to belongs to one sequence, and K's and V's pages and scales
    share no memory.
    """
    refuse_tangents(k, v, k_pages, v_pages, k_scales, v_scales)
    code = check_rows("k", k)
    check_rows("v", v, k)
    if v.shape != k.shape:
        raise ValueError(f"k and v must have identical shapes, got {k.shape} and {v.shape}")
    if k_pages.dtype != torch.float8_e4m3fn:
        raise ValueError("append_kv_blocks writes float8_e4m3fn pages; append_kv writes others")
    check_pools(k_pages, v_pages, k_scales, v_scales, k, k.dtype, written=True, e4m3=True)
    if k_pages.shape[2:] != k.shape[1:]:
        raise ValueError("the pages' kv_heads and head_dim must be the rows'")
    (num_pages, page_tokens, heads, dim), tokens = k_pages.shape, k.shape[0]
    check_sequences(page_table, lengths, cu_tokens, tokens, page_tokens, k, "k")
    sequences, max_pages = page_table.shape
    if not tokens or not sequences:
        return
    args = _APPEND_ARGS.pack(
        k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(),
        page_table.data_ptr(), lengths.data_ptr(), 0 if cu_tokens is None else cu_tokens.data_ptr(),
        *k.stride()[:2], *v.stride()[:2], *k_pages.stride()[:3], *k_scales.stride(), page_table.stride(0), tokens,
        num_pages, sequences, max_pages, heads, dim, page_tokens, page_tokens // k_scales.shape[1], code, 0)
    device = k.device
    status = _native.lib().sa_append_kv_blocks(args, device.index, _native.current_stream_handle(device))
    if status:
        _native.check(status, "sa_append_kv_blocks")


__all__ = ["append_kv_blocks"]
