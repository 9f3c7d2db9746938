"""Kernel boundary (reference src/seqattn_core/kernels/__init__.py).

The reference's Triton launch wrappers are replaced by calls into the gfx950
library through its C ABI; ``triton_is_available`` is kept as an alias of
``hip_is_available`` so capability checks in caller code keep working.
"""

from .blocks import append_kv_blocks
from .decode import paged_decode_attention
from .prefill import paged_prefill_attention
from .rows import append_kv, normalize_rotate_append, normalize_rotate_qk, read_kv
from .streaming import (
    finalize_attention,
    hip_is_available,
    triton_is_available,
    update_attention_state,
    update_attention_state_int8,
)

__all__ = [
    "append_kv",
    "append_kv_blocks",
    "finalize_attention",
    "hip_is_available",
    "normalize_rotate_append",
    "normalize_rotate_qk",
    "paged_decode_attention",
    "paged_prefill_attention",
    "read_kv",
    "triton_is_available",
    "update_attention_state",
    "update_attention_state_int8",
]
