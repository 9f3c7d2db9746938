"""Host side of the cache operators: refusals before any GPU call, slots, frequencies (CPU)."""

from __future__ import annotations

import ctypes
import itertools
import math

import pytest
import torch
from torch.autograd import forward_ad

from seqattn import DeviceKVCache, _native, rotary_frequencies
from seqattn.kernels import append_kv, normalize_rotate_append, normalize_rotate_qk, paged_decode_attention, read_kv
from seqattn.kernels.decode import _DECODE_ARGS
from seqattn.kernels.rows import _READ_ARGS, _ROWS_ARGS, _overlap, _written_layout

@pytest.fixture(autouse=True)
def no_error_left():
    """A refusal's text stays until the next call of the library."""
    yield
    if _native.library_is_built():
        assert _native.lib().sa_paged_decode(decode_args(sequences=0), 0, None) == 0


built = pytest.mark.skipif(not _native.library_is_built(), reason="native library not built")


def test_frequencies_of_one_and_several_axes():
    f = rotary_frequencies(4, base=16.0, device="cpu")
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1, 0.5, 0.25, 0.125], dtype=torch.float64))
    own = rotary_frequencies((2, 4), base=16.0, device="cpu")
    assert own.tolist() == pytest.approx([1, 0.25, 1, 0.5, 0.25, 0.125])
    shared = rotary_frequencies((2, 2), base=16.0, shared=True, device="cpu")
    assert shared.tolist() == pytest.approx([1, 0.5, 0.25, 0.125])
    for bad in ((), 0, (3, 0), (2.0,)):
        with pytest.raises(ValueError, match="sections"):
            rotary_frequencies(bad, device="cpu")
    for base in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="base"):
            rotary_frequencies(4, base=base, device="cpu")


def test_cache_pools_and_slots():
    cache = DeviceKVCache(6, 4, 2, 16, device="cpu")
    assert cache.k_pages.shape == (6, 4, 2, 16) and cache.k_pages.stride() == (128, 16, 64, 1)
    assert cache.bytes == 2 * 6 * 4 * 2 * 16 * 2
    table = torch.tensor([[5, 2, -1], [0, -1, -1]], dtype=torch.int32)
    sequences = torch.tensor([0, 0, 0, 1, 1, 0, 2, -1, 0])
    positions = torch.tensor([0, 3, 6, 1, 4, 12, 0, 0, -1])
    assert cache.slots(table, sequences, positions).tolist() == [20, 23, 10, 1, -1, -1, -1, -1, -1]
    assert cache.slots(table[:, :0], sequences, positions).tolist() == [-1] * 9
    int8 = DeviceKVCache(6, 4, 2, 16, dtype=torch.float16, storage_dtype="int8", device="cpu")
    assert int8.k_pages.dtype == torch.int8 and int8.k_scales.shape == (6, 4, 2)
    assert int8.bytes == 2 * 6 * 4 * 2 * 18
    for bad in (dict(num_pages=0), dict(page_tokens=0), dict(head_dim=12), dict(head_dim=264), dict(num_pages=2**30),
                dict(num_pages=1, page_tokens=2**20 + 1), dict(storage_dtype="float16"), dict(storage_dtype="fp8")):
        with pytest.raises(ValueError):
            DeviceKVCache(**{**dict(num_pages=6, page_tokens=4, kv_heads=2, head_dim=16, device="cpu"), **bad})
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        DeviceKVCache(6, 4, 2, 16, dtype=torch.float32, device="cpu")


def test_host_tensors_are_refused():
    q, pool = torch.zeros((2, 2, 16), dtype=torch.bfloat16), torch.zeros((2, 4, 2, 16), dtype=torch.bfloat16)
    slots, n = torch.zeros(2, dtype=torch.int64), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: normalize_rotate_qk(q, q, slots, rotary_frequencies(8, device="cpu")),
                 lambda: append_kv(q, q, pool, pool, slots), lambda: read_kv(pool, pool, slots),
                 lambda: paged_decode_attention(q, pool, pool, n[:, None], n)):
        with pytest.raises(ValueError, match="device tensors"):
            call()


ROWS_FIELDS = (
    "q k v q_out k_out k_pages v_pages k_scales v_scales slots positions frequencies q_weight k_weight "
    "qt qh kt kh vt vh qot qoh kot koh pp pt ph sp st sh pos_axis pos_token "
    "tokens num_pages eps q_heads kv_heads head_dim page_tokens pairs adjacent axes s0 s1 s2 s3 pos64 qw32 kw32 "
    "dtype int8").split()


def rows_args(**fields):
    values = dict.fromkeys(ROWS_FIELDS, 0)
    values.update(q=16, k=16, q_out=16, k_out=16, tokens=4, q_heads=4, kv_heads=2, head_dim=64, eps=1e-6)
    values.update(fields)
    return _ROWS_ARGS.pack(*(values[f] for f in ROWS_FIELDS))


@built
def test_rows_entry_point_rejects_bad_arguments_without_a_gpu():
    lib = _native.lib()
    paged = dict(k_out=0, v=16, k_pages=16, v_pages=16, slots=8, num_pages=2, page_tokens=4)
    turned = dict(positions=8, frequencies=8, pos64=1, pairs=32, axes=1, s0=32)
    for fields, status, word in (
        (dict(dtype=7), -2, b"dtype"), (dict(head_dim=12), -3, b"head_dim"), (dict(head_dim=264), -3, b"head_dim"),
        (dict(tokens=-1), -1, b"range"), (dict(kv_heads=0), -1, b"range"), (dict(q_heads=0), -1, b"q_heads"),
        (dict(k=0), -1, b"q with q_out"), (dict(q=0), -1, b"q with q_out"), (dict(k_out=0), -1, b"q with q_out"),
        (dict(paged, v=0), -1, b"q with q_out"), (dict(paged, slots=0), -1, b"q with q_out"),
        (dict(qt=4), -1, b"multiples of 8"), (dict(q=24), -1, b"aligned"), (dict(q_weight=2), -1, b"aligned"),
        (dict(pairs=33), -1, b"pairs"), (dict(pairs=32), -1, b"positions"), (dict(turned, axes=5), -1, b"axes"),
        (dict(turned, s0=31), -1, b"add up"), (dict(turned, s0=33), -1, b"add up"),
        (dict(turned, axes=2), -1, b"add up"),
        (dict(turned, frequencies=4), -1, b"positions"),
        (dict(paged, page_tokens=0), -1, b"2^31"), (dict(paged, num_pages=1, page_tokens=2**20 + 1), -1, b"2^20"),
        (dict(paged, num_pages=2**30), -1, b"2^31"), (dict(paged, int8=1), -1, b"scales"),
        (dict(paged, pp=4), -1, b"aligned"), (dict(paged, slots=4), -1, b"aligned"),
    ):
        assert lib.sa_normalize_rotate_store(rows_args(**fields), 0, None) == status, fields
        assert word in lib.sa_last_error(), (fields, lib.sa_last_error())
    assert lib.sa_normalize_rotate_store(None, 0, None) == -1
    assert lib.sa_normalize_rotate_store(rows_args(tokens=0), 0, None) == 0


@built
def test_read_entry_point_rejects_bad_arguments_without_a_gpu():
    lib = _native.lib()
    names = "k v ks vs slots ko vo pp pt ph sp st sh tokens pages heads dim page dtype int8 _".split()

    def call(**fields):
        values = dict.fromkeys(names, 0)
        values.update(k=16, v=16, slots=8, ko=16, vo=16, tokens=4, pages=2, heads=2, dim=64, page=4)
        values.update(fields)
        return lib.sa_read_kv(_READ_ARGS.pack(*(values[n] for n in names)), 0, None)

    assert call(dtype=3) == -2 and call(dim=20) == -3
    for fields in (dict(k=0), dict(v=8), dict(slots=0), dict(ko=0), dict(vo=8), dict(pt=4), dict(int8=1), dict(page=0),
                   dict(pages=2**30), dict(tokens=2**31), dict(heads=0)):
        assert call(**fields) == -1, fields
        assert b"sa_read_kv" in lib.sa_last_error()
    assert call(tokens=0) == 0 and lib.sa_read_kv(None, 0, None) == -1


@built
def test_decode_entry_point_rejects_bad_arguments_without_a_gpu():
    lib = _native.lib()
    names = ("q k v ks vs table lengths out lse workspace workspace_bytes qt qh ot oh pp pt ph sp st sh "
             "table_stride lse_stride num_pages scale sequences max_pages q_heads kv_heads dim page dtype int8").split()

    def args(**fields):
        values = dict.fromkeys(names, 0)
        values.update(q=16, k=16, v=16, table=4, lengths=4, out=16, num_pages=2, scale=0.1, sequences=1, max_pages=2,
                      q_heads=4, kv_heads=2, dim=64, page=16)
        values.update(fields)
        return _DECODE_ARGS.pack(*(values[n] for n in names))

    for fields, status in ((dict(dtype=2), -2), (dict(dim=12), -3), (dict(dim=264), -3), (dict(q_heads=3), -1),
                           (dict(kv_heads=0), -1), (dict(sequences=-1), -1), (dict(page=0), -1), (dict(num_pages=2**30), -1),
                           (dict(num_pages=1, page=2**20 + 1), -1),
                           (dict(max_pages=2**30), -1), (dict(q=0), -1), (dict(out=8), -1), (dict(qt=4), -1),
                           (dict(pt=4), -1), (dict(int8=1), -1), (dict(table=0), -1), (dict(lengths=2), -1)):
        assert lib.sa_paged_decode(args(**fields), 0, None) == status, fields
        assert b"sa_paged_decode" in lib.sa_last_error()
    assert lib.sa_paged_decode(args(sequences=0), 0, None) == 0
    assert lib.sa_paged_decode(None, 0, None) == -1
    needed = ctypes.c_int64(-1)
    assert lib.sa_paged_decode_workspace_bytes(args(dim=12), 0, ctypes.byref(needed)) == -3
    assert lib.sa_paged_decode_workspace_bytes(args(), 0, None) == -1
    # Its sizes alone decide, and calls of one size need the same.
    assert lib.sa_paged_decode_workspace_bytes(args(q=0, k=0, lengths=0), 0, ctypes.byref(needed)) == 0
    assert needed.value >= 0 and needed.value % 16 == 0


DECODE_FIELDS = (
    "q k v ks vs table lengths out lse workspace workspace_bytes qt qh ot oh pp pt ph sp st sh "
    "table_stride lse_stride num_pages scale sequences max_pages q_heads kv_heads dim page dtype int8").split()


def decode_args(**fields):
    """Arguments of which every refusal but the one asked for is out of the way: the workspace is there and large."""
    values = dict.fromkeys(DECODE_FIELDS, 0)
    values.update(q=16, k=16, v=16, table=4, lengths=4, out=16, workspace=16, workspace_bytes=2**40, num_pages=2,
                  scale=0.1, sequences=1, max_pages=2, q_heads=4, kv_heads=2, dim=64, page=16)
    values.update(fields)
    return _DECODE_ARGS.pack(*(values[n] for n in DECODE_FIELDS))


READ_FIELDS = "k v ks vs slots ko vo pp pt ph sp st sh tokens pages heads dim page dtype int8 _".split()


def read_args(**fields):
    values = dict.fromkeys(READ_FIELDS, 0)
    values.update(k=16, v=16, slots=8, ko=16, vo=16, tokens=4, pages=2, heads=2, dim=64, page=4)
    values.update(fields)
    return _READ_ARGS.pack(*(values[n] for n in READ_FIELDS))


@built
def test_pools_without_pages_are_refused_where_rows_are_read():
    """Pages and slots out of range are replaced by row 0 of page 0, which an empty pool does not have."""
    lib = _native.lib()
    assert lib.sa_paged_decode(decode_args(num_pages=0), 0, None) == -1
    assert b"at least one page" in lib.sa_last_error()
    assert lib.sa_paged_decode(decode_args(num_pages=0, sequences=0), 0, None) == 0
    assert lib.sa_read_kv(read_args(pages=0), 0, None) == -1
    assert b"at least one page" in lib.sa_last_error()
    assert lib.sa_read_kv(read_args(pages=0, tokens=0), 0, None) == 0
    # The workspace's size does not depend on the pool.
    needed = ctypes.c_int64()
    assert lib.sa_paged_decode_workspace_bytes(decode_args(num_pages=0), 0, ctypes.byref(needed)) == 0 < needed.value


@built
def test_decode_refuses_more_sequences_than_its_indexes_hold():
    """A thread's and a workgroup's steps through the sequences would pass 2^31."""
    lib = _native.lib()
    for sequences in (2**30 + 1, 2**31 - 1):
        assert lib.sa_paged_decode(decode_args(sequences=sequences), 0, None) == -1
        assert b"at most 2^30 sequences" in lib.sa_last_error()


@built
def test_decode_refuses_a_misaligned_lse_and_misaligned_scales():
    lib = _native.lib()
    for fields in (dict(lse=2), dict(int8=1, ks=2, vs=3), dict(int8=1, ks=5, vs=2)):
        assert lib.sa_paged_decode(decode_args(**fields), 0, None) == -1
        assert b"missing or not aligned" in lib.sa_last_error()


@built
@pytest.mark.parametrize("fields,status,words", [
    (dict(dtype=2), -2, b"dtype code 2"),
    (dict(dim=12), -3, b"head_dim"), (dict(dim=8), -3, b"head_dim"), (dict(dim=264), -3, b"head_dim"),
    (dict(q_heads=3), -1, b"multiple of kv_heads"), (dict(q_heads=0), -1, b"multiple of kv_heads"),
    (dict(kv_heads=0), -1, b"multiple of kv_heads"), (dict(q_heads=2**17), -1, b"multiple of kv_heads"),
    (dict(sequences=-1), -1, b"below 2^31"), (dict(max_pages=-1), -1, b"below 2^31"), (dict(page=0), -1, b"below 2^31"),
    (dict(num_pages=-1), -1, b"below 2^31"), (dict(num_pages=2**30), -1, b"below 2^31"),
    (dict(max_pages=2**30), -1, b"below 2^31"), (dict(num_pages=1, max_pages=1, page=2**20 + 1), -1, b"2^20"),
    *((dict([(s, 4)]), -1, b"strides must be multiples of 8") for s in ("qt", "qh", "ot", "oh", "pp", "pt", "ph")),
    *((dict([(p, 0)]), -1, b"missing or not aligned") for p in ("q", "k", "v", "out", "lengths", "table")),
    *((dict([(p, 8)]), -1, b"missing or not aligned") for p in ("q", "k", "v", "out")),
    (dict(table=2), -1, b"missing or not aligned"), (dict(lengths=2), -1, b"missing or not aligned"),
    (dict(int8=1), -1, b"missing or not aligned"), (dict(int8=1, ks=2), -1, b"missing or not aligned"),
    (dict(int8=1, ks=2, vs=2, k=4), -1, b"missing or not aligned"),
    (dict(workspace=0), -1, b"workspace"), (dict(workspace=8), -1, b"workspace"),
    (dict(pt=2**26), -1, b"token stride"), (dict(pt=-8), -1, b"token stride"),
])
def test_decode_entry_point_names_what_it_refuses(fields, status, words):
    lib = _native.lib()
    assert lib.sa_paged_decode(decode_args(**fields), 0, None) == status
    assert words in lib.sa_last_error() and b"sa_paged_decode" in lib.sa_last_error()


@built
def test_decode_workspace_size_is_checked():
    lib = _native.lib()
    for sizes in (dict(), dict(q_heads=32, kv_heads=2), dict(dim=256), dict(int8=1, ks=2, vs=2)):
        needed = ctypes.c_int64(-1)
        assert lib.sa_paged_decode_workspace_bytes(decode_args(**sizes), 0, ctypes.byref(needed)) == 0
        assert needed.value > 0 and needed.value % 16 == 0
        assert lib.sa_paged_decode(decode_args(workspace_bytes=needed.value - 1, **sizes), 0, None) == -1
        assert b"workspace" in lib.sa_last_error()


def test_overlapping_layouts_are_told_from_disjoint_ones():
    """The rows of a layout, counted element by element."""
    def shared(counts, strides, extent):
        places = torch.zeros(4000, dtype=torch.int64)
        for index in itertools.product(*(range(n) for n in counts)):
            at = sum(i * s for i, s in zip(index, strides))
            places[at : at + extent] += 1
        return bool((places > 1).any())

    disjoint = [((4, 8), (15 * 16, 32), 16),   # every other one of 15 heads
                ((4, 3), (16, 64), 16), ((4, 3), (48, 16), 16), ((1, 3), (0, 16), 16), ((5, 1), (16, 0), 16),
                ((0, 3), (0, 16), 16), ((3, 4, 2), (256, 16, 64), 16), ((3, 4, 2), (8, 2, 1), 1)]
    over = [((4, 8), (14 * 16, 32), 16), ((4, 3), (0, 16), 16), ((4, 3), (16, 0), 16), ((2, 2), (8, 64), 16),
            ((3, 4, 2), (128, 16, 32), 16), ((3, 4, 2), (192, 16, 48), 16), ((3, 4, 2), (8, 2, 0), 1), ((2, 2, 2), (2, 1, 1), 1)]
    for layout in disjoint:
        assert not _overlap(*layout) and not shared(*layout), layout
    for layout in over:
        assert _overlap(*layout) and shared(*layout), layout


@pytest.mark.parametrize("counts,strides,extent", [
    ((3, 4, 2), (128, 16, 64), 16),   # head by head in a page
    ((3, 4, 2), (256, 64, 16), 16),   # room behind a token's heads
    ((3, 4, 2), (256, 16, 128), 16),  # and between the heads
    ((3, 1, 2), (64, 0, 24), 16),     # pieces with room between them
    ((2, 3, 2), (10, 1, 5), 1),       # scales
])
def test_pools_that_meet_are_told_from_pools_that_do_not(counts, strides, extent):
    def places(at):
        starts = [sum(i * s for i, s in zip(index, strides)) for index in itertools.product(*(range(n) for n in counts))]
        return {at + start + d for start in starts for d in range(extent)}

    first, span = places(0), max(places(0)) + 1
    for offset in range(0, span + 20):
        assert _written_layout(offset, counts, strides, extent) == (False, bool(first & places(offset))), offset


def test_forward_mode_tangents_are_refused():
    """Before any other check, so that host tensors show it."""
    x, w = torch.zeros((2, 2, 16), dtype=torch.bfloat16), torch.zeros(16)
    pool, scales = torch.zeros((2, 4, 2, 16), dtype=torch.bfloat16), torch.zeros((2, 4, 2), dtype=torch.float16)
    i, n, freq = torch.zeros(2, dtype=torch.int64), torch.zeros(2, dtype=torch.int32), rotary_frequencies(8, device="cpu")
    calls = {
        normalize_rotate_qk: dict(q=x, k=x, positions=i, frequencies=freq, q_weight=w, k_weight=w, q_out=x, k_out=x),
        append_kv: dict(k=x, v=x, k_pages=pool, v_pages=pool, slots=i, k_scales=scales, v_scales=scales),
        normalize_rotate_append: dict(q=x, k=x, v=x, k_pages=pool, v_pages=pool, slots=i, positions=i, frequencies=freq,
                                      q_weight=w, k_weight=w, k_scales=scales, v_scales=scales, q_out=x),
        read_kv: dict(k_pages=pool, v_pages=pool, slots=i, k_scales=scales, v_scales=scales),
        paged_decode_attention: dict(q=x, k_pages=pool, v_pages=pool, page_table=n[:, None], lengths=n, k_scales=scales,
                                     v_scales=scales, out=x),
    }
    with forward_ad.dual_level(), torch.no_grad():
        for function, arguments in calls.items():
            with pytest.raises(ValueError, match="device tensors"):
                function(**arguments)
            for name, t in arguments.items():
                if not t.is_floating_point():
                    continue
                dual = forward_ad.make_dual(t, torch.ones_like(t))
                with pytest.raises(ValueError, match="inference-only"):
                    function(**{**arguments, name: dual})
                with pytest.raises(ValueError, match="device tensors"):
                    function(**{**arguments, name: dual.detach()})
