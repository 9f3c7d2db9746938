"""Host side of the e4m3 cache and the windowed attention: the reference's rounding, refusals before any GPU call (CPU)."""

from __future__ import annotations

import math

import pytest
import torch

from seqattn import DeviceKVCache, _native
from seqattn.kernels import append_kv_blocks
from seqattn.kernels.blocks import _APPEND_ARGS
from seqattn.kernels.decode import _DECODE_ARGS, _WINDOW_ARGS, check_window
from seqattn.kernels.rows import _READ_ARGS
from blocks_reference import POWERS, VALUES, power_for, rounded

built = pytest.mark.skipif(not _native.library_is_built(), reason="native library not built")


@pytest.fixture(autouse=True)
def no_error_left():
    """A refusal's text stays until the next call of the library."""
    yield
    if _native.library_is_built():
        assert _native.lib().sa_append_kv_blocks(append_args(tokens=0), 0, None) == 0


def test_the_reference_rounds_as_the_format_does():
    table = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(VALUES.nan_to_num(1e3), table.nan_to_num(1e3))
    assert torch.equal(POWERS[:255], torch.arange(255, dtype=torch.uint8).view(torch.float8_e8m0fnu).double())
    finite = VALUES[torch.isfinite(VALUES)].sort().values
    between = (finite[1:] + finite[:-1]) / 2
    x = torch.cat([finite, between, between * (1 + 2.0**-12), between * (1 - 2.0**-12), torch.tensor([math.inf, math.nan])])
    assert torch.equal(rounded(x).nan_to_num(1e3), x.float().to(torch.float8_e4m3fn).double().nan_to_num(1e3))
    for top, power in ((448.0, 1.0), (448.5, 2.0), (0.0, 2.0**-126), (1.0, 2.0**-8), (0.875, 2.0**-9), (math.inf, 2.0**-126)):
        assert power_for(torch.tensor([0.0, top], dtype=torch.float64)) == power


def test_an_e4m3_cache_has_block_scales():
    cache = DeviceKVCache(6, 96, 2, 16, storage_dtype="float8_e4m3fn", device="cpu")
    assert cache.block_tokens == 32 and cache.k_pages.dtype == torch.float8_e4m3fn
    assert cache.k_scales.shape == (6, 3, 2) and cache.k_scales.dtype == torch.float8_e8m0fnu
    assert cache.bytes == 2 * 6 * 2 * (96 * 16 + 3)
    assert DeviceKVCache(6, 64, 2, 16, storage_dtype="float8_e4m3fn", device="cpu").block_tokens == 64
    assert DeviceKVCache(6, 64, 2, 16, storage_dtype="float8_e4m3fn", block_tokens=16, device="cpu").k_scales.shape[1] == 4
    for bad in (dict(block_tokens=8), dict(block_tokens=48), dict(block_tokens=64), dict(page_tokens=24), dict(page_tokens=8),
                dict(block_tokens=32, storage_dtype=None), dict(block_tokens=32, storage_dtype="int8")):
        with pytest.raises(ValueError):
            DeviceKVCache(**{**dict(num_pages=6, page_tokens=96, kv_heads=2, head_dim=16, storage_dtype="float8_e4m3fn",
                                    device="cpu"), **bad})


def test_host_tensors_are_refused():
    k = torch.zeros((2, 2, 16), dtype=torch.bfloat16)
    pages = torch.zeros((2, 16, 2, 16), dtype=torch.float8_e4m3fn)
    scales, n = torch.zeros((2, 1, 2), dtype=torch.float8_e8m0fnu), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="device tensors"):
        append_kv_blocks(k, k, pages, pages, scales, scales, n[:, None], n)


def test_windows():
    assert check_window(None, 0) == (0, 0) and check_window(5, 0) == (5, 0) and check_window(2**40, 2**33) == (2**31 - 1,) * 2
    for window, sinks in ((None, 4), (0, 0), (-1, 0), (5, -1)):
        with pytest.raises(ValueError, match="window"):
            check_window(window, sinks)
    for window, sinks in ((1.5, 0), (5, 0.5), ("5", 0)):
        with pytest.raises(TypeError):
            check_window(window, sinks)


APPEND_FIELDS = ("k v k_pages v_pages k_scales v_scales table lengths cu kt kh vt vh pp pt ph sp sb sh table_stride tokens "
                 "num_pages sequences max_pages kv_heads dim page block dtype _").split()


def append_args(**fields):
    values = dict.fromkeys(APPEND_FIELDS, 0)
    values.update(k=16, v=16, k_pages=8, v_pages=16, k_scales=1, v_scales=2, table=4, lengths=4, cu=4, tokens=3, num_pages=2,
                  sequences=2, max_pages=2, kv_heads=2, dim=64, page=32, block=16)
    values.update(fields)
    return _APPEND_ARGS.pack(*(values[f] for f in APPEND_FIELDS))


@built
def test_append_entry_point_rejects_bad_arguments_without_a_gpu():
    lib = _native.lib()
    for fields, status, word in (
        (dict(dtype=7), -2, b"dtype"), (dict(dim=12), -3, b"head_dim"), (dict(dim=264), -3, b"head_dim"),
        (dict(tokens=-1), -1, b"range"), (dict(tokens=2**31), -1, b"range"), (dict(kv_heads=0), -1, b"range"),
        (dict(kv_heads=2**17), -1, b"range"), (dict(sequences=-1), -1, b"range"), (dict(sequences=2**30 + 1), -1, b"range"),
        (dict(page=0), -1, b"2^20"), (dict(page=2**21), -1, b"2^20"), (dict(num_pages=2**27), -1, b"2^31"),
        (dict(max_pages=2**27), -1, b"2^31"), (dict(max_pages=-1), -1, b"2^31"), (dict(num_pages=-1), -1, b"2^31"),
        (dict(block=8), -1, b"power of two"), (dict(block=0), -1, b"power of two"), (dict(block=-16), -1, b"power of two"),
        (dict(block=64), -1, b"divides"), (dict(page=48, block=48), -1, b"power of two"),
        (dict(cu=0), -1, b"one row per sequence"), (dict(kt=4), -1, b"multiples of 8"), (dict(ph=4), -1, b"multiples of 8"),
        (dict(k=8), -1, b"aligned"), (dict(v=0), -1, b"missing"), (dict(k_pages=4), -1, b"aligned"),
        (dict(v_scales=0), -1, b"missing"), (dict(table=0), -1, b"missing"), (dict(lengths=2), -1, b"aligned"),
        (dict(cu=2), -1, b"aligned"),
    ):
        assert lib.sa_append_kv_blocks(append_args(**fields), 0, None) == status, fields
        assert word in lib.sa_last_error(), (fields, lib.sa_last_error())
    assert lib.sa_append_kv_blocks(None, 0, None) == -1
    for nothing in (dict(tokens=0), dict(sequences=0), dict(max_pages=0), dict(tokens=0, sequences=0, cu=0)):
        assert lib.sa_append_kv_blocks(append_args(**nothing), 0, None) == 0


@built
def test_read_entry_point_checks_blocks():
    lib = _native.lib()
    names = "k v ks vs slots ko vo pp pt ph sp st sh tokens pages heads dim page dtype kind block".split()

    def call(**fields):
        values = dict.fromkeys(names, 0)
        values.update(k=8, v=16, ks=1, vs=3, slots=8, ko=16, vo=16, tokens=0, pages=2, heads=2, dim=64, page=32, kind=2, block=16)
        values.update(fields)
        return lib.sa_read_kv(_READ_ARGS.pack(*(values[n] for n in names)), 0, None)

    assert call() == 0
    for fields in (dict(block=8), dict(block=24), dict(block=64), dict(ks=0), dict(k=4), dict(pt=4)):
        assert call(**fields) == -1, fields


@built
def test_window_decode_entry_point_rejects_bad_arguments_without_a_gpu():
    lib = _native.lib()
    names = ("q k v ks vs table lengths out lse workspace workspace_bytes qt qh ot oh pp pt ph sp st sh "
             "table_stride lse_stride num_pages scale sequences max_pages q_heads kv_heads dim page dtype kind").split()

    def call(window=0, sinks=0, block=0, **fields):
        values = dict.fromkeys(names, 0)
        values.update(q=16, k=16, v=16, table=4, lengths=4, out=16, workspace=16, num_pages=2, scale=0.1, sequences=1,
                      max_pages=2, q_heads=4, kv_heads=2, dim=64, page=32)
        values.update(fields)
        return lib.sa_paged_window_decode(_DECODE_ARGS.pack(*(values[n] for n in names)) +
                                          _WINDOW_ARGS.pack(window, sinks, block, 0), 0, None)

    for fields, word in (
        (dict(kind=3), b"kind"), (dict(kind=-1), b"kind"), (dict(window=-1), b"window"), (dict(window=5, sinks=-1), b"window"),
        (dict(sinks=1), b"window"), (dict(kind=2, ks=1, vs=1, block=24), b"power of two"), (dict(kind=2, block=16), b"missing"),
        (dict(kind=1, ks=1, vs=2), b"aligned"), (dict(), b"workspace"), (dict(kind=2, ks=1, vs=3, k=8, block=16), b"workspace"),
    ):
        assert call(**fields) == -1, fields
        assert word in lib.sa_last_error(), (fields, lib.sa_last_error())
    assert call(dim=12) == -3 and call(dtype=5) == -2
    assert lib.sa_paged_window_decode(None, 0, None) == -1
    assert call(sequences=0, window=5, sinks=2, kind=2, block=32) == 0


@built
def test_prefill_entry_point_rejects_bad_arguments_without_a_gpu():
    import ctypes

    from seqattn.kernels.prefill import _PREFILL_ARGS

    lib = _native.lib()
    names = ("q k v ks vs table lengths cu out lse workspace workspace_bytes qt qh ot oh pp pt ph sp st sh table_stride "
             "lse_stride tokens num_pages scale sequences max_pages q_heads kv_heads dim page dtype kind window sinks block _"
             ).split()

    def args(**fields):
        values = dict.fromkeys(names, 0)
        values.update(q=16, k=16, v=16, table=4, lengths=4, cu=4, out=16, workspace=16, tokens=5, num_pages=2, scale=0.1,
                      sequences=2, max_pages=2, q_heads=4, kv_heads=2, dim=64, page=32)
        values.update(fields)
        return _PREFILL_ARGS.pack(*(values[n] for n in names))

    for fields, status, word in (
        (dict(dtype=7), -2, b"dtype"), (dict(dim=12), -3, b"head_dim"), (dict(dim=264), -3, b"head_dim"),
        (dict(kind=1, dim=72), -3, b"multiple of 16"), (dict(kind=3), -1, b"kind"), (dict(kind=-1), -1, b"kind"),
        (dict(q_heads=5), -1, b"multiple of kv_heads"), (dict(kv_heads=0), -1, b"multiple of kv_heads"),
        (dict(tokens=-1), -1, b"2^31"), (dict(tokens=2**30), -1, b"2^31"), (dict(sequences=2**30 + 1), -1, b"2^30"),
        (dict(page=0), -1, b"2^20"), (dict(num_pages=2**27), -1, b"2^31"), (dict(max_pages=2**27), -1, b"2^31"),
        (dict(window=-1), -1, b"window"), (dict(sinks=2), -1, b"window"), (dict(window=1, sinks=-1), -1, b"window"),
        (dict(kind=2, block=24), -1, b"power of two"), (dict(num_pages=0), -1, b"at least one page"),
        (dict(qt=4), -1, b"multiples of 8"), (dict(pp=4), -1, b"16 bytes"), (dict(kind=1, ph=8), -1, b"16 bytes"),
        (dict(pt=2**26), -1, b"token stride"), (dict(pt=-16), -1, b"token stride"),
        (dict(q=8), -1, b"aligned"), (dict(cu=0), -1, b"missing"), (dict(cu=2), -1, b"aligned"), (dict(table=0), -1, b"missing"),
        (dict(kind=1), -1, b"missing"), (dict(kind=1, ks=1, vs=2), -1, b"aligned"), (dict(kind=2, ks=1, vs=1, k=8, block=16), -1, b"aligned"),
        (dict(workspace=0), -1, b"workspace"), (dict(workspace_bytes=1000), -1, b"workspace"),
    ):
        assert lib.sa_paged_prefill(args(**fields), 0, None) == status, fields
        assert word in lib.sa_last_error(), (fields, lib.sa_last_error())
    assert lib.sa_paged_prefill(None, 0, None) == -1
    for nothing in (dict(tokens=0), dict(sequences=0)):
        assert lib.sa_paged_prefill(args(**nothing), 0, None) == 0
    needed = ctypes.c_int64()
    assert lib.sa_paged_prefill_workspace_bytes(args(), 0, ctypes.byref(needed)) == 0 and needed.value > 0
    assert lib.sa_paged_prefill_workspace_bytes(args(tokens=0), 0, ctypes.byref(needed)) == 0 and needed.value == 0
    assert lib.sa_paged_prefill_workspace_bytes(args(dim=12), 0, ctypes.byref(needed)) == -3
    assert lib.sa_paged_prefill_workspace_bytes(None, 0, ctypes.byref(needed)) == -1
