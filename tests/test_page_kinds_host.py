"""CPU test: entry points that write or read pages of rows or INT8 alone refuse e4m3 pages, whose scales lie elsewhere."""

from __future__ import annotations

import pytest

from seqattn import _native
from seqattn.kernels.decode import _DECODE_ARGS
from test_device_cache_host import rows_args

pytestmark = pytest.mark.skipif(not _native.library_is_built(), reason="native library not built")
E4M3 = 2  # SA_PAGES_E4M3


def test_rows_are_not_stored_into_e4m3_pages_as_int8():
    lib = _native.lib()
    paged = dict(k_out=0, v=16, k_pages=16, v_pages=16, k_scales=2, v_scales=2, slots=8, num_pages=2, page_tokens=16, tokens=0)
    assert lib.sa_normalize_rotate_store(rows_args(**paged, int8=1), 0, None) == 0
    assert lib.sa_normalize_rotate_store(rows_args(**paged, int8=E4M3), 0, None) == -1
    assert b"sa_append_kv_blocks" in lib.sa_last_error()
    assert lib.sa_normalize_rotate_store(rows_args(tokens=0, int8=E4M3), 0, None) == 0  # no pages


def test_e4m3_pages_are_not_decoded_as_int8():
    lib = _native.lib()
    # No sequences: 24 pointers, strides and counts, the scale, then the sizes.
    args = lambda kind: _DECODE_ARGS.pack(*(0,) * 24, 0.1, 0, 2, 4, 2, 64, 16, 0, kind)
    assert lib.sa_paged_decode(args(1), 0, None) == 0
    assert lib.sa_paged_decode(args(E4M3), 0, None) == -1
    assert b"sa_paged_window_decode" in lib.sa_last_error()
