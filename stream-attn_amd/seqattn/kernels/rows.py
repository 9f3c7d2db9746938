"""Rows between a QKV projection and the attention: norms, rotations, cache pages.

``normalize_rotate_qk`` normalizes every head of Q and K and rotates it by its
token's position on one or several axes, in one pass.  ``append_kv`` writes K
and V rows into the pages of a device-resident cache, ``normalize_rotate_append``
does both in one launch (K goes straight from the projection's output to its
page), and ``read_kv`` returns pages as packed rows.  None of them has a
counterpart in the reference.

Pages are ``[num_pages, page_tokens, kv_heads, head_dim]`` tensors of any page,
token and head strides (K's and V's the same), 16-bit, INT8 or e4m3 (:mod:`.blocks`).  INT8 pages hold the storage format of
:mod:`seqattn.quantization` with one token per group: ``[num_pages,
page_tokens, kv_heads]`` float16 scales.  Slot ``page * page_tokens + row``
names a row of them.  :class:`seqattn.DeviceKVCache` keeps such pages.

Every launch is asynchronous on torch's current stream of the operands' device
and allocates nothing but the outputs that are not given, so it can be captured
into a graph.
"""

from __future__ import annotations

import functools
import struct
from collections.abc import Sequence

import torch
from torch.autograd import forward_ad

from .. import _native

MAX_ROTARY_AXES = 4
MAX_PAGE_TOKENS = 2**20
# sa_rows_args: 14 pointers, 20 strides and counts, eps, 16 int32.
_ROWS_ARGS = struct.Struct("=14Q20qd16i")
# sa_read_args: 7 pointers, 8 strides and counts, 6 int32.
_READ_ARGS = struct.Struct("=7Q8q6i")
NO_STRIDES = (0, 0, 0)
# What pages hold (SA_PAGES_*).
ROW_PAGES, INT8_PAGES, E4M3_PAGES = range(3)


def _refuse_gradients() -> None:
    if torch.is_grad_enabled():
        raise ValueError("seqattn is inference-only: call it under torch.no_grad() or with detached tensors")


def refuse_tangents(*operands: torch.Tensor | None) -> None:
    """Forward-mode tangents would be lost (torch.no_grad() does not turn them off)."""
    if getattr(forward_ad, "_current_level", 0) >= 0:  # -1: none can be there
        if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in operands):
            raise ValueError("seqattn is inference-only: call it with detached tensors inside forward_ad.dual_level()")


def _overlap(counts: Sequence[int], strides: Sequence[int], extent: int) -> bool:
    """Whether pieces of ``extent`` elements can lie over each other: a dimension steps past all that shorter steps span."""
    for stride, n in sorted(zip(strides, counts)):
        if n > 1:
            if stride < extent:
                return True
            extent += (n - 1) * stride
    return False


def check_rows(name: str, rows: torch.Tensor, like: torch.Tensor | None = None, *, output: bool = False) -> int:
    """[tokens, heads, head_dim] rows that the kernels can address; their dtype code (0 where ``like`` has it)."""
    if rows.ndim != 3:
        raise ValueError(f"{name} must use packed [tokens, heads, head_dim] layout")
    if not rows.is_cuda:
        raise ValueError("kernel operands must be device tensors")
    st, sh, sd = rows.stride()
    if sd != 1:
        raise ValueError("kernel operands must have a unit stride in the last dimension")
    if st % 8 or sh % 8 or rows.data_ptr() % 16:
        raise ValueError(f"{name} must be 16-byte aligned, with token and head strides in multiples of 8 elements")
    code = 0
    tokens, heads, dim = rows.shape
    if like is None:
        code = _native.dtype_code(rows.dtype)
        if dim % 8 or not 16 <= dim <= 256:
            raise ValueError(f"head_dim must be a multiple of 8 in [16, 256], got {dim}")
    elif rows.device != like.device or rows.dtype != like.dtype:
        raise ValueError(f"{name} must have the device and dtype of the other rows")
    if heads < 1:
        raise ValueError(f"{name} has no heads")
    if output:
        if _overlap((tokens, heads), (st, sh), dim):
            raise ValueError(f"{name} has rows that overlap")
    if rows.requires_grad:
        _refuse_gradients()
    return code


def _meet(offset: int, steps: Sequence[tuple[int, int]], extent: int) -> bool:
    """Whether pieces of two such layouts meet, one ``offset`` behind the other; ``steps``: (stride, count), long ones first."""
    if not steps:
        return offset < extent
    (stride, n), *shorter = steps
    behind, rest = divmod(offset, stride)
    return (behind < n and _meet(rest, shorter, extent)) or (behind + 1 < n and _meet(stride - rest, shorter, extent))


@functools.lru_cache  # the few layouts of a program's pools
def _written_layout(offset: int, counts: Sequence[int], strides: Sequence[int], extent: int) -> tuple[bool, bool]:
    """Whether pieces of a pool overlap, and whether they meet those of the other pool."""
    if _overlap(counts, strides, extent):
        return True, True
    steps = sorted(((s, n) for s, n in zip(strides, counts) if n > 1), reverse=True)
    return False, _meet(offset, steps, extent)


def _check_written(name: str, k: torch.Tensor, v: torch.Tensor, counts, strides, extent: int, rows) -> None:
    offset = abs(v.data_ptr() - k.data_ptr()) // k.element_size()
    overlap, meet = _written_layout(offset, counts, strides, extent)
    if overlap:
        raise ValueError(f"{name} of written pages must not share memory")
    if meet:
        # The same rows may go to one place.
        same = rows is not None and rows[0].data_ptr() == rows[1].data_ptr() and rows[0].stride() == rows[1].stride()
        if offset or not same:
            raise ValueError(f"{name} of K's and V's written pages must not share memory")


def check_pools(
    k_pages, v_pages, k_scales, v_scales, like: torch.Tensor, dtype: torch.dtype, *, written: bool = False,
    rows: tuple[torch.Tensor, torch.Tensor] | None = None, e4m3: bool = False
) -> int:
    """Both pools of a cache, on ``like``'s device; what they hold (ROW_PAGES, INT8_PAGES, E4M3_PAGES).

    ``written``: rows go into them, those of ``rows`` as they are where it is given.  ``e4m3``: they may hold e4m3.
    """
    shape, strides, stored = k_pages.shape, k_pages.stride(), k_pages.dtype
    if len(shape) != 4:
        raise ValueError("k_pages must use [num_pages, page_tokens, kv_heads, head_dim] layout")
    if strides[3] != 1:
        raise ValueError("pages must have a unit stride in head_dim")
    if v_pages.shape != shape or v_pages.dtype != stored or v_pages.stride() != strides:
        raise ValueError("k_pages and v_pages must have the same shape and dtype, and the same strides")
    kind = INT8_PAGES if stored == torch.int8 else E4M3_PAGES if e4m3 and stored == torch.float8_e4m3fn else ROW_PAGES
    align = 8 if kind else 16
    if strides[0] % 8 or strides[1] % 8 or strides[2] % 8 or k_pages.data_ptr() % align or v_pages.data_ptr() % align:
        raise ValueError("pages must be aligned, with their other strides in multiples of 8 elements")
    if k_pages.device != like.device or v_pages.device != like.device:
        raise ValueError("pages must live on the device of the rows")
    if not k_pages.numel():
        raise ValueError("the cache has no pages")
    if shape[1] > MAX_PAGE_TOKENS or shape[0] * shape[1] > 2**31 - 1:
        raise ValueError(f"pages have at most {MAX_PAGE_TOKENS} rows, the cache fewer than 2^31")
    if k_pages.requires_grad or v_pages.requires_grad:
        _refuse_gradients()
    if written:
        _check_written("rows", k_pages, v_pages, shape[:3], strides[:3], shape[3], rows)
    if kind == ROW_PAGES:
        if k_scales is not None or v_scales is not None:
            raise ValueError("only INT8 pages have scales" + (", and e4m3 pages" if e4m3 else ""))
        if stored != dtype:
            raise ValueError(f"pages of {stored} do not match rows of {dtype}")
        return kind
    if k_scales is None or v_scales is None:
        raise ValueError(f"{'INT8' if kind == INT8_PAGES else 'e4m3'} pages need their scales")
    for scales in (k_scales, v_scales):
        if kind == E4M3_PAGES:
            check_block_scales(scales, shape, like.device)
        elif scales.dtype != torch.float16 or scales.shape != shape[:3] or scales.device != like.device:
            raise ValueError("INT8 scales must be float16 [num_pages, page_tokens, kv_heads] on the pages' device")
    if k_scales.stride() != v_scales.stride():
        raise ValueError("k_scales and v_scales must have the same strides")
    if k_scales.requires_grad or v_scales.requires_grad:
        _refuse_gradients()
    if written:
        _check_written("scales", k_scales, v_scales, k_scales.shape, k_scales.stride(), 1, rows)
    return kind


def check_block_scales(scales: torch.Tensor, pages: Sequence[int], device: torch.device) -> None:
    if scales.dtype != torch.float8_e8m0fnu or scales.ndim != 3 or scales.device != device:
        raise ValueError("e4m3 scales must be float8_e8m0fnu [num_pages, page_tokens / block_tokens, kv_heads] "
                         "on the pages' device")
    blocks, page_tokens = scales.shape[1], pages[1]
    if scales.shape[0] != pages[0] or scales.shape[2] != pages[2] or not blocks or page_tokens % blocks:
        raise ValueError("e4m3 scales must have a scale per block of every page and K/V head")
    block_tokens = page_tokens // blocks
    if block_tokens < 16 or block_tokens & (block_tokens - 1):
        raise ValueError(f"blocks must have a power of two of rows from 16 on, got {block_tokens}")


def check_sequences(page_table: torch.Tensor, lengths: torch.Tensor, cu_tokens: torch.Tensor | None, tokens: int,
                    page_tokens: int, rows: torch.Tensor, name: str) -> None:
    """The pages and lengths of sequences, and where each one's rows start among ``tokens`` ones (one each without)."""
    device = rows.device
    if page_table.dtype != torch.int32 or page_table.ndim != 2 or page_table.device != device:
        raise ValueError(f"page_table must be an int32 [sequences, max_pages] tensor on {name}'s device")
    if lengths.dtype != torch.int32 or lengths.ndim != 1 or lengths.device != device:
        raise ValueError(f"lengths must be an int32 [sequences] tensor on {name}'s device")
    sequences, max_pages = page_table.shape
    if lengths.shape[0] != sequences or (cu_tokens is None and tokens != sequences):
        raise ValueError("page_table and lengths must have one row per sequence")
    if (max_pages > 1 and page_table.stride(1) != 1) or (sequences > 1 and lengths.stride(0) != 1):
        raise ValueError("page_table rows and lengths must be contiguous")
    if max_pages * page_tokens > 2**31 - 1:
        raise ValueError("page_table rows must hold fewer than 2^31 keys")
    if cu_tokens is not None:
        if cu_tokens.dtype != torch.int32 or cu_tokens.ndim != 1 or cu_tokens.device != device:
            raise ValueError(f"cu_tokens must be an int32 [sequences + 1] tensor on {name}'s device")
        if cu_tokens.shape[0] != sequences + 1 or (sequences and cu_tokens.stride(0) != 1):
            raise ValueError("cu_tokens must hold one start per sequence and the end, contiguously")


def check_place(name: str, out: torch.Tensor, rows: torch.Tensor, others: Sequence[torch.Tensor | None]) -> None:
    """An output is apart from ``others``; where ``rows`` are, it is ``rows`` itself."""
    where = out.data_ptr()
    if where and any(t is not None and t.data_ptr() == where for t in others):
        raise ValueError(f"{name} must not share memory with another operand")
    if where and rows.data_ptr() == where:
        if any(n > 1 and a != b for n, a, b in zip(out.shape, out.stride(), rows.stride())):
            raise ValueError(f"{name} must not share memory with its input unless it is its input")


def new_rows(tokens: int, heads: int, dim: int, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """Contiguous [tokens, heads, head_dim] memory (the strided form of torch.empty, which takes less host time)."""
    return torch.empty_strided((tokens, heads, dim), (heads * dim, dim, 1), dtype=dtype, device=device)


def _check_slots(slots: torch.Tensor, tokens: int, device: torch.device) -> None:
    if slots.dtype != torch.int64 or slots.ndim != 1 or slots.device != device:
        raise ValueError("slots must be a one-dimensional int64 tensor on the rows' device")
    if slots.shape[0] != tokens or (tokens > 1 and slots.stride(0) != 1):
        raise ValueError("slots must hold one slot per token, contiguously")


def _weight(name: str, weight: torch.Tensor | None, rows: torch.Tensor) -> int:
    if weight is None:
        return 0
    if weight.shape != rows.shape[2:] or weight.device != rows.device or weight.stride(0) != 1:
        raise ValueError(f"{name} must be a contiguous [head_dim] tensor on the rows' device")
    if weight.dtype not in (rows.dtype, torch.float32):
        raise ValueError(f"{name} must have the rows' dtype or float32")
    if weight.data_ptr() % 16:
        raise ValueError(f"{name} must be 16-byte aligned")
    if weight.requires_grad:
        _refuse_gradients()
    return weight.data_ptr()


def _rotation(positions, frequencies, sections, pairing, rows: torch.Tensor):
    """(positions, frequencies) pointers, position strides, pairs, axes, sections, int64 positions."""
    if pairing not in ("halves", "adjacent"):
        raise ValueError("pairing must be 'halves' or 'adjacent'")
    if frequencies is None:
        if positions is not None or sections is not None:
            raise ValueError("a rotation needs both positions and frequencies")
        return 0, 0, 0, 0, 0, 0, (0, 0, 0, 0), 0
    if positions is None:
        raise ValueError("a rotation needs both positions and frequencies")
    tokens, _, dim = rows.shape
    device = rows.device
    if frequencies.dtype != torch.float64 or frequencies.ndim != 1 or frequencies.device != device:
        raise ValueError("frequencies must be a float64 [pairs] tensor on the rows' device")
    if frequencies.requires_grad:
        _refuse_gradients()
    pairs = frequencies.shape[0]
    if not 1 <= pairs <= dim // 2 or (pairs > 1 and frequencies.stride(0) != 1):
        raise ValueError("frequencies must be contiguous, for 1 to head_dim / 2 pairs")
    if positions.dtype not in (torch.int64, torch.int32) or positions.device != device:
        raise ValueError("positions must be an int32 or int64 tensor on the rows' device")
    sections = (pairs,) if sections is None else tuple(sections)
    axes = len(sections)
    if not 1 <= axes <= MAX_ROTARY_AXES or sum(sections) != pairs or min(sections) < 1:
        raise ValueError(f"sections must be 1 to {MAX_ROTARY_AXES} positive counts that add up to the pairs")
    if positions.ndim == 1 and axes == 1:
        axis_stride, token_stride = 0, positions.stride(0)
    elif positions.ndim == 2 and positions.shape[0] == axes:
        axis_stride, token_stride = positions.stride()
    else:
        raise ValueError(f"positions must be [{axes}, tokens]" + (" or [tokens]" if axes == 1 else ""))
    if positions.shape[-1] != tokens:
        raise ValueError("positions must hold one position per token and axis")
    return (positions.data_ptr(), frequencies.data_ptr(), axis_stride, token_stride, pairs, axes,
            (*sections, *(0,) * (MAX_ROTARY_AXES - axes)), positions.dtype == torch.int64)


def _run_rows(q, k, v, q_out, k_out, pools, slots, positions, frequencies, sections, pairing, q_weight, k_weight, eps, code):
    """Launch sa_normalize_rotate_store on checked rows; ``pools`` = (k_pages, v_pages, k_scales, v_scales, int8) or None."""
    tokens, kv_heads, dim = k.shape
    where, freq, axis_stride, token_stride, pairs, axes, counts, wide = _rotation(positions, frequencies, sections, pairing, k)
    eps = float(eps)
    if not 0.0 <= eps < float("inf"):
        raise ValueError("eps must be finite and non-negative")
    weights = _weight("q_weight", q_weight, k), _weight("k_weight", k_weight, k)
    if tokens == 0:
        return
    if pools is None:
        pages, strides, num_pages, page_tokens, int8 = (0, 0, 0, 0), NO_STRIDES * 2, 0, 0, False
    else:
        k_pages, v_pages, k_scales, v_scales, int8 = pools
        num_pages, page_tokens = k_pages.shape[:2]
        if int8:
            pages = k_pages.data_ptr(), v_pages.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr()
            strides = *k_pages.stride()[:3], *k_scales.stride()
        else:
            pages = k_pages.data_ptr(), v_pages.data_ptr(), 0, 0
            strides = *k_pages.stride()[:3], *NO_STRIDES
    none = 0, 0
    args = _ROWS_ARGS.pack(
        0 if q is None else q.data_ptr(), k.data_ptr(), 0 if v is None else v.data_ptr(),
        0 if q_out is None else q_out.data_ptr(), 0 if k_out is None else k_out.data_ptr(),
        *pages, 0 if slots is None else slots.data_ptr(), where, freq, *weights,
        *(none if q is None else q.stride()[:2]), *k.stride()[:2], *(none if v is None else v.stride()[:2]),
        *(none if q_out is None else q_out.stride()[:2]), *(none if k_out is None else k_out.stride()[:2]),
        *strides, axis_stride, token_stride, tokens, num_pages, eps,
        0 if q is None else q.shape[1], kv_heads, dim, page_tokens, pairs, pairing == "adjacent", axes, *counts, wide,
        q_weight is not None and q_weight.dtype == torch.float32,
        k_weight is not None and k_weight.dtype == torch.float32, code, int8)
    device = k.device
    status = _native.lib().sa_normalize_rotate_store(args, device.index, _native.current_stream_handle(device))
    if status:
        _native.check(status, "sa_normalize_rotate_store")


def _check_qk(q: torch.Tensor, k: torch.Tensor) -> int:
    code = check_rows("q", q)
    check_rows("k", k, q)
    if q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError("q and k must have the same tokens and head_dim")
    return code


def _output(name: str, out: torch.Tensor | None, rows: torch.Tensor, others: Sequence[torch.Tensor | None]) -> torch.Tensor:
    """The output of ``rows``, which may be ``rows`` itself but none of ``others``."""
    if out is None:
        return new_rows(*rows.shape, rows.dtype, rows.device)
    check_rows(name, out, rows, output=True)
    if out.shape != rows.shape:
        raise ValueError(f"{name} must have the shape of its input")
    check_place(name, out, rows, others)
    return out


def normalize_rotate_qk(
    q: torch.Tensor,
    k: torch.Tensor,
    positions: torch.Tensor | None = None,
    frequencies: torch.Tensor | None = None,
    *,
    sections: Sequence[int] | None = None,
    pairing: str = "halves",
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    q_out: torch.Tensor | None = None,
    k_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Norm and rotation of every head of ``q [tokens, q_heads, head_dim]`` and ``k [tokens, kv_heads, head_dim]``.

    With ``q_weight`` (``[head_dim]``, the rows' dtype or float32) each head of
    Q becomes ``x * rsqrt(mean(x^2) + eps) * q_weight``; likewise K.  Then pair
    ``i`` of ``frequencies`` (float64 ``[pairs]``, radians per position, at most
    ``head_dim / 2``), elements ``(i, i + pairs)`` with ``pairing="halves"`` or
    ``(2i, 2i + 1)`` with ``"adjacent"``, is rotated by ``frequencies[i] *
    position``; elements past ``2 * pairs`` are not.  ``positions`` is ``[tokens]``, or
    ``[axes, tokens]`` for up to 4 axes of which axis ``a`` turns ``sections[a]``
    consecutive pairs (:func:`seqattn.rotary_frequencies` makes the usual
    frequencies).  Without positions and frequencies nothing is rotated.

    Returns ``(q_out, k_out)``, new tensors unless given.  An output may be
    its input itself, but must not otherwise share memory with an input or the
    other output.
    """
    refuse_tangents(q, k, frequencies, q_weight, k_weight, q_out, k_out)
    code = _check_qk(q, k)
    if positions is None and frequencies is None and q_weight is None and k_weight is None:
        raise ValueError("normalize_rotate_qk needs a weight or a rotation")
    q_out, k_out = _output("q_out", q_out, q, (k, k_out)), _output("k_out", k_out, k, (q,))
    _run_rows(q, k, None, q_out, k_out, None, None, positions, frequencies, sections, pairing, q_weight, k_weight, eps, code)
    return q_out, k_out


def _check_append(k, v, k_pages, v_pages, k_scales, v_scales, slots, rows):
    check_rows("v", v, k)
    if v.shape != k.shape:
        raise ValueError(f"k and v must have identical shapes, got {k.shape} and {v.shape}")
    int8 = check_pools(k_pages, v_pages, k_scales, v_scales, k, k.dtype, written=True, rows=rows)
    if k_pages.shape[2:] != k.shape[1:]:
        raise ValueError("the pages' kv_heads and head_dim must be the rows'")
    _check_slots(slots, k.shape[0], k.device)
    return k_pages, v_pages, k_scales, v_scales, int8


def append_kv(
    k: torch.Tensor,
    v: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    slots: torch.Tensor,
    *,
    k_scales: torch.Tensor | None = None,
    v_scales: torch.Tensor | None = None,
) -> None:
    """Write rows ``k, v [tokens, kv_heads, head_dim]`` to the pages' ``slots`` (int64 ``[tokens]``).

    A row whose slot is negative (padding) or past the pool is not written.
    The slots of a call are distinct: of two rows with one slot either may
    stay, in parts.  K's and V's pages share no memory (one pool may be both
    where ``k`` is ``v``).  INT8 pages: a row that is not finite reads back as NaN.
    """
    refuse_tangents(k, v, k_pages, v_pages, k_scales, v_scales)
    code = check_rows("k", k)
    pools = _check_append(k, v, k_pages, v_pages, k_scales, v_scales, slots, (k, v))
    _run_rows(None, k, v, None, None, pools, slots, None, None, None, "adjacent", None, None, 0.0, code)


def normalize_rotate_append(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    slots: torch.Tensor,
    positions: torch.Tensor | None = None,
    frequencies: torch.Tensor | None = None,
    *,
    sections: Sequence[int] | None = None,
    pairing: str = "halves",
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    k_scales: torch.Tensor | None = None,
    v_scales: torch.Tensor | None = None,
    q_out: torch.Tensor | None = None,
) -> torch.Tensor:
    """:func:`normalize_rotate_qk` and :func:`append_kv` of its K and of V, in one launch.

    Returns the normalized and rotated Q.  INT8 pages take K before it is
    rounded to 16 bits.  Q is written for every token, also where a row's slot
    is negative; ``q_out`` may be ``q``, and shares no memory with the rest.
    """
    refuse_tangents(q, k, v, k_pages, v_pages, frequencies, q_weight, k_weight, k_scales, v_scales, q_out)
    code = _check_qk(q, k)
    pools = _check_append(k, v, k_pages, v_pages, k_scales, v_scales, slots, None)
    q_out = _output("q_out", q_out, q, (k, v))
    _run_rows(q, k, v, q_out, None, pools, slots, positions, frequencies, sections, pairing, q_weight, k_weight, eps, code)
    return q_out


def read_kv(
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    slots: torch.Tensor,
    *,
    k_scales: torch.Tensor | None = None,
    v_scales: torch.Tensor | None = None,
    dtype: torch.dtype | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """The pages' rows at ``slots`` as packed ``(k, v) [tokens, kv_heads, head_dim]``, the runners' layout.

    INT8 and e4m3 rows come as ``value * scale`` in ``dtype`` (default bfloat16),
    others in the pages' own dtype.  A slot outside the pool gives zeros.
    """
    refuse_tangents(k_pages, v_pages, k_scales, v_scales)
    if dtype is None:
        dtype = torch.bfloat16 if k_pages.dtype in (torch.int8, torch.float8_e4m3fn) else k_pages.dtype
    code = _native.dtype_code(dtype)
    if slots.ndim != 1:
        raise ValueError("slots must be a one-dimensional int64 tensor on the rows' device")
    if slots.device.type != "cuda":
        raise ValueError("kernel operands must be device tensors")
    kind = check_pools(k_pages, v_pages, k_scales, v_scales, slots, dtype, e4m3=True)
    tokens, (num_pages, page_tokens, heads, dim) = slots.shape[0], k_pages.shape
    _check_slots(slots, tokens, k_pages.device)
    if dim % 8 or not 16 <= dim <= 256:
        raise ValueError(f"head_dim must be a multiple of 8 in [16, 256], got {dim}")
    k_out, v_out = (new_rows(tokens, heads, dim, dtype, k_pages.device) for _ in range(2))
    if tokens == 0:
        return k_out, v_out
    args = _READ_ARGS.pack(
        k_pages.data_ptr(), v_pages.data_ptr(), k_scales.data_ptr() if kind else 0, v_scales.data_ptr() if kind else 0,
        slots.data_ptr(), k_out.data_ptr(), v_out.data_ptr(), *k_pages.stride()[:3],
        *(k_scales.stride() if kind else NO_STRIDES),
        tokens, num_pages, heads, dim, page_tokens, code, kind,
        page_tokens // k_scales.shape[1] if kind == E4M3_PAGES else 0)
    device = k_pages.device
    status = _native.lib().sa_read_kv(args, device.index, _native.current_stream_handle(device))
    if status:
        _native.check(status, "sa_read_kv")
    return k_out, v_out


__all__ = ["append_kv", "normalize_rotate_append", "normalize_rotate_qk", "read_kv"]
