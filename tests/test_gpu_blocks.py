"""GPU tests of the e4m3 pages (``append_kv_blocks``, ``read_kv``) against their definition in 64 bits.

Scales are powers of two and e4m3 rounding is exact in FP32, so what the pages
stand for is compared for equality.  A value read back in 16 bits is rounded once
where it does not fit them (below their normal range), else exact.
"""

from __future__ import annotations

import math

import pytest
import torch

from seqattn import DeviceKVCache
from seqattn.kernels import append_kv_blocks, read_kv
from blocks_reference import POWERS, appended, values

pytestmark = pytest.mark.gpu


def pools(gen, pages, page, heads, dim, block, layout="heads"):
    """Random codes (no NaN) and scales near 1, on the GPU: K's and V's pages and scales."""
    shape = (pages, heads, page, dim) if layout == "heads" else (pages, page, heads, dim)
    scale_shape = (pages, heads, page // block) if layout == "heads" else (pages, page // block, heads)
    view = (lambda t: t.transpose(1, 2)) if layout == "heads" else (lambda t: t)
    out = []
    for _ in range(2):
        codes = torch.randint(0, 255, shape, generator=gen, dtype=torch.uint8)
        codes[codes == 127] = 0
        bytes_ = torch.randint(118, 124, scale_shape, generator=gen, dtype=torch.uint8)
        out.append((view(codes.cuda()).view(torch.float8_e4m3fn), view(bytes_.cuda()).view(torch.float8_e8m0fnu)))
    return out


def host(k_or_v):
    codes, scales = (t.view(torch.uint8).cpu() for t in k_or_v)
    return codes.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu)


def check(k, v, k_pool, v_pool, table, lengths, cu, device_rows=None):
    """Append on the GPU and compare both pools, whole, with the definition."""
    want = []
    for rows, pool in ((k, k_pool), (v, v_pool)):
        codes, scales = host(pool)
        stand, powers = values(codes, scales), POWERS[scales.view(torch.uint8).long()].clone()
        appended(stand, powers, rows, table, lengths, cu)
        want.append((stand, powers))
    dk, dv = device_rows or (k.cuda(), v.cuda())
    append_kv_blocks(dk, dv, k_pool[0], v_pool[0], k_pool[1], v_pool[1], table.cuda(), lengths.cuda(), cu.cuda())
    for pool, (stand, powers) in zip((k_pool, v_pool), want):
        codes, scales = host(pool)
        assert bool((POWERS[scales.view(torch.uint8).long()] == powers).all())
        got = values(codes, scales)
        wrong = ~((got == stand) | (torch.isnan(got) & torch.isnan(stand)))
        assert not bool(wrong.any()), wrong.nonzero()[:5].tolist()


def sequences(gen, new, before, page, pages):
    counts = [-(-(a + b) // page) for a, b in zip(new, before)]
    order = torch.randperm(pages, generator=gen)
    table = torch.full((len(new), max([1, *counts])), -1, dtype=torch.int32)
    at = 0
    for s, c in enumerate(counts):
        table[s, :c] = order[at : at + c].to(torch.int32)
        at += c
    assert at <= pages
    lengths = torch.tensor([a + b for a, b in zip(new, before)], dtype=torch.int32)
    return table, lengths, torch.tensor([0, *new]).cumsum(0).to(torch.int32)


CASES = [
    # new, before, heads, head_dim, page, block, dtype, layout
    ([1], [0], 1, 16, 16, 16, torch.bfloat16, "heads"),
    ([1, 1, 1], [5, 0, 64], 2, 64, 64, 64, torch.bfloat16, "heads"),
    ([17, 0, 1, 40], [3, 9, 15, 0], 3, 128, 32, 16, torch.float16, "tokens"),
    ([130, 64], [0, 65], 2, 128, 64, 64, torch.bfloat16, "heads"),
    ([300], [77], 1, 256, 128, 128, torch.bfloat16, "tokens"),
    ([75, 3], [31, 200], 5, 80, 96, 32, torch.float16, "heads"),
    ([9, 20], [500, 0], 1, 248, 512, 512, torch.bfloat16, "heads"),
    ([600], [0], 2, 24, 256, 256, torch.float16, "heads"),
    ([2] * 300, [0, 14, 15, 16, 30, 7] * 50, 1, 40, 16, 16, torch.bfloat16, "heads"),
]


@pytest.mark.parametrize("new,before,heads,dim,page,block,dtype,layout", CASES)
def test_append_matches_the_definition(new, before, heads, dim, page, block, dtype, layout):
    gen = torch.Generator().manual_seed(sum(new) + dim)
    pages = sum(-(-(a + b) // page) for a, b in zip(new, before)) + 2
    table, lengths, cu = sequences(gen, new, before, page, pages)
    k_pool, v_pool = pools(gen, pages, page, heads, dim, block, layout)
    # Magnitudes far apart: scales that grow, that stay, and codes below e4m3's normal range.
    size = torch.exp2(torch.randint(-12, 6, (sum(new), heads, 1), generator=gen).float())
    k, v = ((torch.randn((sum(new), heads, dim), generator=gen) * size).to(dtype) for _ in range(2))
    check(k, v, k_pool, v_pool, table, lengths, cu)


def test_rows_one_by_one_are_rounded_again_as_the_scale_grows():
    gen = torch.Generator().manual_seed(1)
    table, lengths, _ = sequences(gen, [0, 0], [40, 40], 32, 5)
    k_pool, v_pool = pools(gen, 5, 32, 2, 64, 32)
    cu = torch.arange(3, dtype=torch.int32)
    for t in range(40):
        k, v = ((torch.randn((2, 2, 64), generator=gen) * 1.3**t * 2.0**-6).to(torch.bfloat16) for _ in range(2))
        check(k, v, k_pool, v_pool, table, torch.full_like(lengths, t + 1), cu)


def test_values_next_to_ties_and_extreme_rows():
    gen = torch.Generator().manual_seed(2)
    table, lengths, cu = sequences(gen, [64], [0], 16, 4)
    k_pool, v_pool = pools(gen, 4, 16, 1, 256, 16)
    # 256 consecutive bfloat16 values a row, of every binade; half of them are ties.
    k = (torch.arange(64)[:, None] * 256 + torch.arange(256)).to(torch.int16).view(torch.bfloat16).view(64, 1, 256)
    v = k.flip(0).contiguous()
    check(k, v, k_pool, v_pool, table, lengths, cu)


def test_infinities_nan_zeros_and_largest_values():
    gen = torch.Generator().manual_seed(3)
    table, lengths, cu = sequences(gen, [5, 20], [8, 0], 32, 4)
    k_pool, v_pool = pools(gen, 4, 32, 2, 128, 16)
    k, v = (torch.randn((25, 2, 128), generator=gen).to(torch.float16) for _ in range(2))
    k[0, 0, 5], k[1, 1, 7], v[9, 0, 0] = math.inf, -math.inf, math.nan
    v[6:, 1] = 0
    k[10:, 0] = 65504
    v[2] = math.nan
    check(k, v, k_pool, v_pool, table, lengths, cu)


def test_positions_and_pages_outside_are_not_written():
    gen = torch.Generator().manual_seed(4)
    table, lengths, cu = sequences(gen, [10, 40, 20], [0, 0, 50], 16, 9)
    k_pool, v_pool = pools(gen, 9, 16, 1, 64, 16)
    lengths[0] = 4           # six rows below position 0
    table[1, 1] = -1         # a page outside
    table[2, 4] = 10**6
    table = table[:, :5].contiguous()
    lengths[2] = 85          # the last rows past the table's 80 keys
    k, v = (torch.randn((80, 1, 64), generator=gen).to(torch.bfloat16) for _ in range(2))
    check(k, v, k_pool, v_pool, table, lengths, cu)  # ten rows past cu_tokens' end
    lengths[:] = torch.tensor([-7, 0, 10**9])
    check(k, v, k_pool, v_pool, table, lengths, cu)


def test_disordered_starts_stay_inside():
    """cu_tokens that fall or leave the rows: nothing outside the operands is read or written."""
    gen = torch.Generator().manual_seed(5)
    table, lengths = torch.arange(6, dtype=torch.int32).view(3, 2), torch.full((3,), 30, dtype=torch.int32)
    k_pool, v_pool = pools(gen, 8, 16, 1, 64, 16)
    guard = [host(p)[0][6:].clone() for p in (k_pool, v_pool)]
    k = torch.ones((30, 1, 64), dtype=torch.bfloat16, device="cuda")
    for cu in ([0, 30, 0, 30], [-5, 10**9, 3, 40], [30, 20, 10, 0], [2**31 - 1, -(2**31), 5, 9]):
        append_kv_blocks(k, k.clone(), k_pool[0], v_pool[0], k_pool[1], v_pool[1], table.cuda(), lengths.cuda(),
                         torch.tensor(cu, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    for before, pool in zip(guard, (k_pool, v_pool)):
        assert torch.equal(host(pool)[0][6:].view(torch.uint8), before.view(torch.uint8))


def test_strided_rows_of_a_projection():
    gen = torch.Generator().manual_seed(6)
    table, lengths, cu = sequences(gen, [70], [11], 64, 3)
    k_pool, v_pool = pools(gen, 3, 64, 4, 96, 32)
    fused = torch.randn((70, 16, 96), generator=gen).to(torch.bfloat16)
    device = fused.cuda()
    check(fused[:, 8:12], fused[:, 12:], k_pool, v_pool, table, lengths, cu, (device[:, 8:12], device[:, 12:]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_read_back(dtype):
    gen = torch.Generator().manual_seed(7)
    k_pool, v_pool = pools(gen, 6, 48, 3, 72, 16, "tokens")
    slots = torch.tensor([0, 287, 47, 48, -1, 288, 100, 100, 2**40, -(2**40)])
    k, v = read_kv(k_pool[0], v_pool[0], slots.cuda(), k_scales=k_pool[1], v_scales=v_pool[1], dtype=dtype)
    held = (slots >= 0) & (slots < 288)
    for got, pool in ((k, k_pool), (v, v_pool)):
        stand = values(*host(pool)).flatten(0, 1)[slots.clamp(0, 287)]
        want = torch.where(held[:, None, None], stand, 0.0).to(dtype)
        assert bool((got.cpu() == want).all())


def test_a_cache_of_each_kind_is_extended_alike():
    """extend() and read() of one sequence after another; 16-bit pages hold the rows themselves."""
    gen = torch.Generator().manual_seed(8)
    new, before = [20, 0, 1], [13, 5, 63]
    rows = [torch.randn((24, 2, 64), generator=gen).to(torch.bfloat16).cuda() for _ in range(2)]
    cu = torch.tensor([0, 20, 20, 21], dtype=torch.int32, device="cuda")  # three rows of padding
    lengths = torch.tensor([a + b for a, b in zip(new, before)], dtype=torch.int32, device="cuda")
    table = torch.tensor([[4, 1], [0, 2], [3, 5]], dtype=torch.int32, device="cuda")
    for storage, off in ((None, 0.0), ("int8", 1 / 254 + 2.0**-8 + 2.0**-11), ("float8_e4m3fn", 2.0**-4)):
        cache = DeviceKVCache(6, 64, 2, 64, storage_dtype=storage)
        cache.extend(*rows, table, lengths, cu)
        where = torch.tensor([0] * 20 + [2], device="cuda")
        at = torch.tensor([*range(13, 33), 63], device="cuda")
        back = cache.read(cache.slots(table, where, at))
        for got, want in zip(back, rows):
            # INT8: half a step of the row's, the scale's and the result's rounding.  e4m3: half a step of the value,
            # or half of the smallest step of a scale of at most 2 amax / 448.
            top = want[:21].abs().max().float()
            bound = off * (top if storage == "int8" else want[:21].abs().float()) + top * 2 / 448 * 2.0**-10 * bool(off)
            assert bool(((got.float() - want[:21].float()).abs() <= bound).all())
        untouched = cache.read(cache.slots(table, where[:13] * 0, torch.arange(13, device="cuda")))
        assert all(bool((x == 0).all()) for x in untouched)
        # One token each, no cu_tokens.
        cache.extend(rows[0][:3], rows[1][:3], table, lengths + 1)
        back = cache.read(cache.slots(table, torch.arange(3, device="cuda"), lengths.long()))
        want = rows[0][:3].abs().float()
        bound = off * (want.max() if storage == "int8" else want) + top * 2 / 448 * 2.0**-10 * bool(off)
        assert bool(((back[0].float() - rows[0][:3].float()).abs() <= bound).all())


def test_captured_appends_follow_the_lengths():
    gen = torch.Generator().manual_seed(9)
    table, _, _ = sequences(gen, [0, 0], [64, 64], 32, 6)
    graph_pools, eager_pools = pools(gen, 6, 32, 2, 64, 32), None
    eager_pools = [(c.clone(), s.view(torch.uint8).clone().view(torch.float8_e8m0fnu)) for c, s in graph_pools]
    k, v = (torch.randn((2, 2, 64), generator=gen).to(torch.bfloat16).cuda() for _ in range(2))
    lengths, table = torch.ones(2, dtype=torch.int32, device="cuda"), table.cuda()

    def call(pair):
        (kc, ks), (vc, vs) = pair
        append_kv_blocks(k, v, kc, vc, ks, vs, table, lengths)

    scratch = [(c.clone(), s.view(torch.uint8).clone().view(torch.float8_e8m0fnu)) for c, s in graph_pools]
    call(scratch)  # loads the kernels before the capture
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(graph_pools)
    for t in range(40):
        lengths.fill_(t + 1)
        k.copy_(torch.randn((2, 2, 64), generator=gen) * 1.2**t)
        graph.replay()
        call(eager_pools)
        torch.cuda.synchronize()
        for (a, b), (c, d) in zip(graph_pools, eager_pools):
            assert torch.equal(a.view(torch.uint8), c.view(torch.uint8))
            assert torch.equal(b.view(torch.uint8), d.view(torch.uint8))


def test_refusals():
    k = torch.zeros((3, 2, 64), dtype=torch.bfloat16, device="cuda")
    pages = torch.zeros((4, 32, 2, 64), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scales = torch.zeros((4, 2, 2), dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    more = pages.clone(), scales.view(torch.uint8).clone().view(torch.float8_e8m0fnu)
    table = torch.zeros((3, 2), dtype=torch.int32, device="cuda")
    n, cu = table[:, 0].contiguous(), torch.arange(4, dtype=torch.int32, device="cuda")
    good = dict(k=k, v=k, k_pages=pages, v_pages=more[0], k_scales=scales, v_scales=more[1], page_table=table, lengths=n,
                cu_tokens=cu)
    of = lambda blocks: torch.zeros((4, blocks, 2), dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    for bad, word in (
        (dict(v=k[:2]), "identical shapes"), (dict(v=k.half()), "device and dtype"), (dict(k=k.float()), "float16 or bfloat16"),
        (dict(k=k[..., :8]), "head_dim"), (dict(k_pages=k), "append_kv writes others"),
        (dict(k_pages=pages[..., :32]), "same shape"), (dict(v_pages=pages), "must not share memory"),
        (dict(v_scales=scales), "must not share memory"), (dict(k_scales=None), "need their scales"),
        (dict(k_scales=scales.view(torch.uint8)), "float8_e8m0fnu"), (dict(k_scales=of(3), v_scales=of(3)), "scale per block"),
        (dict(k_scales=of(4), v_scales=of(4)), "power of two"), (dict(k_scales=scales[:2]), "scale per block"),
        (dict(k_scales=scales.cpu()), "pages' device"), (dict(page_table=table.long()), "page_table"),
        (dict(lengths=n.long()), "lengths"), (dict(lengths=n[:2]), "one row per sequence"),
        (dict(cu_tokens=cu.long()), "cu_tokens"), (dict(cu_tokens=cu[:3]), "cu_tokens"),
        (dict(cu_tokens=None, page_table=table[:2], lengths=n[:2]), "one row per sequence"),
        (dict(cu_tokens=torch.arange(8, dtype=torch.int32, device="cuda")[::2]), "contiguously"),
        (dict(page_table=torch.zeros((2, 3), dtype=torch.int32, device="cuda").t()), "contiguous"),
        (dict(k=k[:, :1], v=k[:, :1]), "kv_heads"), (dict(k=k.clone().requires_grad_()), "inference-only"),
    ):
        with pytest.raises(ValueError, match=word):
            append_kv_blocks(**{**good, **bad})
    # Slot by slot only into pages with a scale per row, or none.
    from seqattn.kernels import append_kv

    with pytest.raises(ValueError, match="do not match"):
        append_kv(k, k, pages, more[0], torch.zeros(3, dtype=torch.int64, device="cuda"))
    cache = DeviceKVCache(4, 32, 2, 64, storage_dtype="float8_e4m3fn")
    for call in (lambda: cache.append(k, k, n.long()), lambda: cache.normalize_rotate_append(k, k, k, n.long())):
        with pytest.raises(ValueError, match="extend"):
            call()
    with pytest.raises(ValueError, match="need their scales"):
        read_kv(pages, more[0], n.long())


def test_nothing_to_append():
    cache = DeviceKVCache(2, 16, 1, 32, storage_dtype="float8_e4m3fn")
    none = torch.zeros((0, 1, 32), dtype=torch.bfloat16, device="cuda")
    table = torch.zeros((2, 0), dtype=torch.int32, device="cuda")
    lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
    cache.extend(none, none, table, lengths, torch.zeros(3, dtype=torch.int32, device="cuda"))
    cache.extend(none, none, table[:0], lengths[:0])
    rows = torch.ones((2, 1, 32), dtype=torch.bfloat16, device="cuda")
    cache.extend(rows, rows, table, lengths + 1)  # a table without pages
    assert bool((cache.k_pages.view(torch.uint8) == 0).all()) and bool((cache.k_scales.view(torch.uint8) == 0).all())
