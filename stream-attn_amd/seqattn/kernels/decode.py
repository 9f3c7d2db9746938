"""Attention of one new token per sequence over a paged, device-resident K/V cache.

No counterpart in the reference, whose kernels read contiguous K/V.  The
launch is asynchronous on torch's current stream of the operands' device; its
workspace comes from torch's allocator, so calls on several streams, and
captured graphs, each have their own.
"""

from __future__ import annotations

import ctypes
import functools
import operator
import struct

import torch

from .. import _native
from .rows import E4M3_PAGES, NO_STRIDES, check_place, check_pools, check_rows, check_sequences, new_rows, refuse_tangents

# sa_decode_args: 10 pointers, 14 sizes and strides, the scale, 8 int32.
_DECODE_ARGS = struct.Struct("=10Q14qd8i")
# What sa_window_decode_args has behind them.
_WINDOW_ARGS = struct.Struct("=4i")


def check_window(window: int | None, sinks: int) -> tuple[int, int]:
    """(window, sinks) as the entry points take them, a window of 0 for none."""
    if window is None:
        if sinks != 0:
            raise ValueError("sinks need a window")
        return 0, 0
    window, sinks = operator.index(window), operator.index(sinks)
    if window < 1 or sinks < 0:
        raise ValueError("window must be positive and sinks must not be negative")
    return min(window, 2**31 - 1), min(sinks, 2**31 - 1)


@functools.lru_cache
def _workspace_bytes(device_index: int, q_heads: int, kv_heads: int, head_dim: int, kind: int) -> int:
    """Workspace of a call, which depends on its head counts, head_dim and kind of pages alone."""
    args = _DECODE_ARGS.pack(*(0,) * 24, 0.0, 1, 0, q_heads, kv_heads, head_dim, 1, 0, kind)
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
    window: int | None = None,
    sinks: int = 0,
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

    With a ``window`` the token, at position ``p = lengths[s] - 1``, sees the last
    ``window`` keys (``j > p - window``) and the first ``sinks`` keys of its
    sequence; pages that hold none of these are not looked up.

    INT8 and e4m3 pages (:mod:`.blocks`) stand for ``value * scale``.  Logits, softmax and sums are FP32;
    a weight enters the product with V as two 16-bit parts.  A logit of NaN or
    ``+inf`` makes its head NaN, one of ``-inf`` is a key without weight; an element
    of a seen V that is not finite makes its element of ``out`` not finite.
    ``out`` may be ``q``, and shares no memory with the rest.
    Returns ``out`` (like ``q``), and with ``return_lse`` also the natural-log
    LSE ``[q_heads, sequences]``.
    """
    refuse_tangents(q, k_pages, v_pages, k_scales, v_scales, out)
    code = check_rows("q", q)
    kind = check_pools(k_pages, v_pages, k_scales, v_scales, q, q.dtype, e4m3=True)
    window, sinks = check_window(window, sinks)
    sequences, q_heads, dim = q.shape
    num_pages, page_tokens, kv_heads, _ = k_pages.shape
    device = q.device
    if k_pages.shape[3] != dim or q_heads % kv_heads:
        raise ValueError("the pages must have q's head_dim and a divisor of its heads")
    check_sequences(page_table, lengths, None, sequences, page_tokens, q, "q")
    max_pages = page_table.shape[1]
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
        needed = _workspace_bytes(index, q_heads, kv_heads, dim, kind)
        workspace = torch.empty_strided((needed,), (1,), dtype=torch.uint8, device=device)
        args = _DECODE_ARGS.pack(
            q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), k_scales.data_ptr() if kind else 0,
            v_scales.data_ptr() if kind else 0, page_table.data_ptr(), lengths.data_ptr(), out.data_ptr(),
            0 if lse is None else lse.data_ptr(), workspace.data_ptr(), needed, *q.stride()[:2], *out.stride()[:2],
            *k_pages.stride()[:3], *(k_scales.stride() if kind else NO_STRIDES), page_table.stride(0),
            max(sequences, 1), num_pages, dim**-0.5 if softmax_scale is None else float(softmax_scale), sequences, max_pages,
            q_heads, kv_heads, dim, page_tokens, code, kind)
        args += _WINDOW_ARGS.pack(window, sinks, page_tokens // k_scales.shape[1] if kind == E4M3_PAGES else 0, 0)
        status = _native.lib().sa_paged_window_decode(args, index, _native.current_stream_handle(device))
        if status:
            _native.check(status, "sa_paged_window_decode")
    return (out, lse) if return_lse else out


__all__ = ["paged_decode_attention"]
