"""Attention of several new tokens per sequence over a paged, device-resident K/V cache.

No counterpart in the reference, whose kernels read contiguous K/V.  The launch is
asynchronous on torch's current stream of the operands' device; its workspace
comes from torch's allocator, so calls on several streams, and captured graphs,
each have their own.
"""

from __future__ import annotations

import ctypes
import functools
import struct

import torch

from .. import _native
from .decode import check_window
from .rows import E4M3_PAGES, NO_STRIDES, check_place, check_pools, check_rows, check_sequences, new_rows, refuse_tangents

# sa_prefill_args: 11 pointers, 15 sizes and strides, the scale, 12 int32.
_PREFILL_ARGS = struct.Struct("=11Q15qd12i")


@functools.lru_cache
def _workspace_bytes(device_index: int, tokens: int, sequences: int, max_pages: int, q_heads: int, kv_heads: int,
                     head_dim: int, page_tokens: int, kind: int, window: int, sinks: int) -> int:
    """Workspace of a call, which depends on its sizes alone."""
    args = _PREFILL_ARGS.pack(*(0,) * 24, tokens, 0, 0.0, sequences, max_pages, q_heads, kv_heads, head_dim, page_tokens, 0, kind,
                              window, sinks, 16, 0)
    needed = ctypes.c_int64()
    status = _native.lib().sa_paged_prefill_workspace_bytes(args, device_index, ctypes.byref(needed))
    _native.check(status, "sa_paged_prefill_workspace_bytes")
    return needed.value


def paged_prefill_attention(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    cu_tokens: torch.Tensor,
    *,
    softmax_scale: float | None = None,
    window: int | None = None,
    sinks: int = 0,
    k_scales: torch.Tensor | None = None,
    v_scales: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    return_lse: bool = False,
):
    """``softmax(q k^T * softmax_scale) v`` for the last tokens of every sequence, causal.

    Sequence ``s`` has rows ``cu_tokens[s] .. cu_tokens[s + 1] - 1`` of ``q [tokens,
    q_heads, head_dim]`` (int32 ``[sequences + 1]``, non-decreasing from 0), its last
    tokens: their K and V are in the pages already and counted in ``lengths[s]``,
    so token ``i`` of ``n`` is at position ``p = lengths[s] - n + i``.  It sees the
    keys ``j <= p`` or, with a ``window``, those with ``j > p - window`` and the
    first ``sinks`` keys of its sequence.  Pages, ``page_table``, ``lengths``, scales
    and the heads are those of :func:`paged_decode_attention`, with its answers for
    keys that are not seen: pages outside the pool or with no visible key, rows past
    a length, whatever they hold.  A token that sees no key gets zeros, and LSE
    ``-inf``.  Rows of ``out`` past ``cu_tokens[-1]`` are not written.

    Logits, softmax and sums are FP32.  A weight enters the product with V in ``q``'s
    dtype, with INT8 pages in float16; V's 8-bit values times their scale enter in the
    same, so with INT8 pages and for float16 ``q`` values past float16's largest count as
    that (e4m3 ones are exact in bfloat16).  8-bit pages need a head_dim and strides in
    multiples of 16.  A logit of NaN or ``+inf`` makes its row NaN, one of ``-inf`` is a
    key without weight; an element of a seen V that is not finite makes its element of
    ``out`` not finite.  ``out`` may be ``q``, and shares no memory with the rest.  Returns
    ``out`` (like ``q``), and with ``return_lse`` also the natural-log LSE ``[q_heads,
    tokens]``.
    """
    refuse_tangents(q, k_pages, v_pages, k_scales, v_scales, out)
    code = check_rows("q", q)
    kind = check_pools(k_pages, v_pages, k_scales, v_scales, q, q.dtype, e4m3=True)
    window, sinks = check_window(window, sinks)
    tokens, q_heads, dim = q.shape
    num_pages, page_tokens, kv_heads, _ = k_pages.shape
    device = q.device
    if k_pages.shape[3] != dim or q_heads % kv_heads:
        raise ValueError("the pages must have q's head_dim and a divisor of its heads")
    if kind and (dim % 16 or any(s % 16 for s in k_pages.stride()[:3]) or k_pages.data_ptr() % 16 or v_pages.data_ptr() % 16):
        raise ValueError("8-bit pages must be 16-byte aligned, with head_dim and strides in multiples of 16")
    if cu_tokens is None:
        raise ValueError("cu_tokens is needed: paged_decode_attention takes one token per sequence")
    check_sequences(page_table, lengths, cu_tokens, tokens, page_tokens, q, "q")
    sequences, max_pages = page_table.shape
    if tokens * (q_heads // kv_heads) > 2**31 - 4097:
        raise ValueError("tokens times query heads per K/V head must be below 2^31 - 4096")
    if out is None:
        out = new_rows(tokens, q_heads, dim, q.dtype, device)
    else:
        check_rows("out", out, q, output=True)
        if out.shape != q.shape:
            raise ValueError("out must have the shape of q")
        check_place("out", out, q, (k_pages, v_pages))
    lse = None
    if return_lse:
        lse = torch.empty_strided((q_heads, tokens), (tokens, 1), dtype=torch.float32, device=device)
    if tokens and sequences:
        index = device.index
        needed = _workspace_bytes(index, tokens, sequences, max_pages, q_heads, kv_heads, dim, page_tokens, kind, window, sinks)
        workspace = torch.empty_strided((needed,), (1,), dtype=torch.uint8, device=device)
        args = _PREFILL_ARGS.pack(
            q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), k_scales.data_ptr() if kind else 0,
            v_scales.data_ptr() if kind else 0, page_table.data_ptr(), lengths.data_ptr(), cu_tokens.data_ptr(),
            out.data_ptr(), 0 if lse is None else lse.data_ptr(), workspace.data_ptr(), needed, *q.stride()[:2],
            *out.stride()[:2], *k_pages.stride()[:3], *(k_scales.stride() if kind else NO_STRIDES), page_table.stride(0),
            tokens, tokens, num_pages, dim**-0.5 if softmax_scale is None else float(softmax_scale), sequences, max_pages,
            q_heads, kv_heads, dim, page_tokens, code, kind, window, sinks,
            page_tokens // k_scales.shape[1] if kind == E4M3_PAGES else 0, 0)
        status = _native.lib().sa_paged_prefill(args, index, _native.current_stream_handle(device))
        if status:
            _native.check(status, "sa_paged_prefill")
    return (out, lse) if return_lse else out


__all__ = ["paged_prefill_attention"]
