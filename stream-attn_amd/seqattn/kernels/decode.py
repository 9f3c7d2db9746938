"""Attention of one new token per sequence over a paged, device-resident K/V cache.

No counterpart in the reference, whose kernels read contiguous K/V.  The
launch is asynchronous on torch's current stream of the operands' device; its
workspace comes from torch's allocator, so calls on several streams, and
captured graphs, each have their own.
"""

from __future__ import annotations

import ctypes
import functools
import struct

import torch

from .. import _native
from .rows import NO_STRIDES, check_place, check_pools, check_rows, new_rows, refuse_tangents

# sa_decode_args: 10 pointers, 14 sizes and strides, the scale, 8 int32.
_DECODE_ARGS = struct.Struct("=10Q14qd8i")


@functools.lru_cache
def _workspace_bytes(device_index: int, q_heads: int, kv_heads: int, head_dim: int, int8: bool) -> int:
    """Workspace of a call, which depends on its head counts, head_dim and kind of pages alone."""
    args = _DECODE_ARGS.pack(*(0,) * 24, 0.0, 1, 0, q_heads, kv_heads, head_dim, 1, 0, int8)
    needed = ctypes.c_int64()
    status = _native.lib().sa_paged_decode_workspace_bytes(args, device_index, ctypes.byref(needed))
    _native.check(status, "sa_paged_decode_workspace_bytes")
    return needed.value


def paged_decode_attention(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    softmax_scale: float | None = None,
    k_scales: torch.Tensor | None = None,
    v_scales: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    return_lse: bool = False,
):
    """``softmax(q k^T * softmax_scale) v`` for one token of every sequence.

    ``q [sequences, q_heads, head_dim]`` attends to keys ``0 .. lengths[s] - 1``
    of its sequence: key ``j`` is row ``j % page_tokens`` of page
    ``page_table[s, j // page_tokens]`` (int32 ``[sequences, max_pages]``;
    entries past a sequence's last page may be anything).  ``lengths`` is int32
    ``[sequences]``, on the device like the rest; a length past the table's row
    stands for the row's keys, one below zero for none.  Query head ``h`` reads
    K/V head ``h // (q_heads // kv_heads)``.  Keys of a page outside the pool are
    not seen, and what rows past a length hold does not matter.  A token that
    sees no key gets zeros, and LSE ``-inf``.

    INT8 pages stand for ``value * scale``.  Logits, softmax and sums are FP32;
    a weight enters the product with V as two 16-bit parts.  A logit of NaN or
    ``+inf`` makes its head NaN, one of ``-inf`` is a key without weight; an element
    of a seen V that is not finite makes its element of ``out`` not finite.
    ``out`` may be ``q``, and shares no memory with the rest.
    Returns ``out`` (like ``q``), and with ``return_lse`` also the natural-log
    LSE ``[q_heads, sequences]``.
    """
    refuse_tangents(q, k_pages, v_pages, k_scales, v_scales, out)
    code = check_rows("q", q)
    int8 = check_pools(k_pages, v_pages, k_scales, v_scales, q, q.dtype)
    sequences, q_heads, dim = q.shape
    num_pages, page_tokens, kv_heads, _ = k_pages.shape
    device = q.device
    if k_pages.shape[3] != dim or q_heads % kv_heads:
        raise ValueError("the pages must have q's head_dim and a divisor of its heads")
    if page_table.dtype != torch.int32 or page_table.ndim != 2 or page_table.device != device:
        raise ValueError("page_table must be an int32 [sequences, max_pages] tensor on q's device")
    if lengths.dtype != torch.int32 or lengths.ndim != 1 or lengths.device != device:
        raise ValueError("lengths must be an int32 [sequences] tensor on q's device")
    max_pages = page_table.shape[1]
    if page_table.shape[0] != sequences or lengths.shape[0] != sequences:
        raise ValueError("page_table and lengths must have one row per sequence")
    if (max_pages > 1 and page_table.stride(1) != 1) or (sequences > 1 and lengths.stride(0) != 1):
        raise ValueError("page_table rows and lengths must be contiguous")
    if max_pages * page_tokens > 2**31 - 1:
        raise ValueError("page_table rows must hold fewer than 2^31 keys")
    if out is None:
        out = new_rows(sequences, q_heads, dim, q.dtype, device)
    else:
        check_rows("out", out, q, output=True)
        if out.shape != q.shape:
            raise ValueError("out must have the shape of q")
        check_place("out", out, q, (k_pages, v_pages))
    lse = None
    if return_lse:
        lse = torch.empty_strided((q_heads, sequences), (sequences, 1), dtype=torch.float32, device=device)
    if sequences:
        index = device.index
        needed = _workspace_bytes(index, q_heads, kv_heads, dim, int8)
        workspace = torch.empty_strided((needed,), (1,), dtype=torch.uint8, device=device)
        args = _DECODE_ARGS.pack(
            q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), k_scales.data_ptr() if int8 else 0,
            v_scales.data_ptr() if int8 else 0, page_table.data_ptr(), lengths.data_ptr(), out.data_ptr(),
            0 if lse is None else lse.data_ptr(), workspace.data_ptr(), needed, *q.stride()[:2], *out.stride()[:2],
            *k_pages.stride()[:3], *(k_scales.stride() if int8 else NO_STRIDES), page_table.stride(0),
            max(sequences, 1), num_pages, dim**-0.5 if softmax_scale is None else float(softmax_scale), sequences, max_pages,
            q_heads, kv_heads, dim, page_tokens, code, int8)
        status = _native.lib().sa_paged_decode(args, index, _native.current_stream_handle(device))
        if status:
            _native.check(status, "sa_paged_decode")
    return (out, lse) if return_lse else out


__all__ = ["paged_decode_attention"]
