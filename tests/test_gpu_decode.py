"""GPU tests of the paged decoding attention (``paged_decode_attention``) against 64 bits.

Bounds.  Logits are FP32 dot products of at most 256 terms and a scale: off by
at most (head_dim + 4) 2^-24 of the largest sum of |q k| * scale, call it e.
Exponentials, running sums and products are FP32 (2^-20 of a weight covers the
exponent's argument, the exponential and thousands of additions in a tree); a
weight enters the products with V as two 16-bit parts, 2^-16.  So the output is
off by (2 e + 2^-15) times the sum of weight * |v|, plus its rounding, and the
LSE by e + 2^-19 (1 + |lse|).
"""

from __future__ import annotations

import math

import pytest
import torch

from seqattn import DeviceKVCache, rotary_frequencies
from seqattn.kernels import normalize_rotate_qk, paged_decode_attention
from paged_reference import HALF_STEP, attention

pytestmark = pytest.mark.gpu


def make(gen, lengths, q_heads, kv_heads, dim, page, dtype, int8=False, layout="heads", spare=2, outliers=False):
    """CPU q, pools, table, lengths; every row of the pools that no sequence sees holds NaN (INT8: a NaN scale)."""
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + spare
    order = torch.randperm(pages, generator=gen)
    table = torch.full((len(lengths), max([1, *counts]) + 1), -1, dtype=torch.int32)
    seen = torch.zeros((pages, page), dtype=torch.bool)
    at = 0
    for s, (n, c) in enumerate(zip(lengths, counts)):
        table[s, :c] = order[at : at + c].to(torch.int32)
        at += c
        for j in range(n):
            seen[table[s, j // page], j % page] = True
    shape = (pages, page, kv_heads, dim)
    k, v = torch.randn(shape, generator=gen), torch.randn(shape, generator=gen)
    if outliers:
        k[torch.rand(shape[:2], generator=gen) < 0.05] *= 8
    scales = (None, None)
    if int8:
        pools, scales = [], []
        for x in (k, v):
            step = x.abs().amax(-1) / 127
            pools.append(torch.round(x / step[..., None]).to(torch.int8))
            scale = step.half()
            scale[~seen] = math.nan
            scales.append(scale)
        k, v = pools
    else:
        k, v = k.to(dtype), v.to(dtype)
        k[~seen], v[~seen] = math.nan, math.nan
    q = torch.randn((len(lengths), q_heads, dim), generator=gen).to(dtype)
    by_head = (lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)) if layout == "heads" else (lambda t: t)
    pools = [by_head(x.cuda()) for x in (k, v)]
    dev_scales = [None if x is None else by_head(x.cuda()) for x in scales]
    return q, (k, v), tuple(scales), table, torch.tensor(lengths, dtype=torch.int32), pools, dev_scales


def check(q, pools, scales, table, lengths, dev_pools, dev_scales, scale=None):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    out, lse = paged_decode_attention(q.cuda(), *dev_pools, table.cuda(), lengths.cuda(), softmax_scale=scale,
                                      k_scales=dev_scales[0], v_scales=dev_scales[1], return_lse=True)
    ref, ref_lse, size, products = attention(q, *pools, table, lengths, scale, *scales)
    e = (q.shape[2] + 4) * 2.0**-24 * products
    bound = HALF_STEP[q.dtype] * ref.abs() + (1 + HALF_STEP[q.dtype]) * (2 * e + 2.0**-15) * size + 2.0**-25
    error = (out.double().cpu() - ref).abs()
    assert bool((error <= bound).all()), float((error / bound).max())
    seen = torch.isfinite(ref_lse)
    assert torch.equal(torch.isfinite(lse.cpu()), seen) and bool((lse.cpu()[~seen] == -math.inf).all())
    assert bool(((lse.double().cpu() - ref_lse).abs()[seen] <= e + 2.0**-19 * (1 + ref_lse[seen].abs())).all())
    return out, lse


CASES = [
    # lengths, q_heads, kv_heads, head_dim, page, dtype, int8, layout
    ([1], 1, 1, 16, 1, torch.bfloat16, False, "tokens"),
    ([0, 1, 2, 0, 65], 8, 2, 64, 16, torch.bfloat16, False, "heads"),
    ([31, 32, 33, 127, 128, 129], 8, 1, 128, 32, torch.float16, False, "heads"),
    ([700], 32, 8, 128, 64, torch.bfloat16, False, "tokens"),
    ([700, 3], 56, 8, 128, 64, torch.bfloat16, True, "heads"),
    ([257, 255], 12, 4, 96, 256, torch.float16, False, "tokens"),
    ([100, 511], 4, 4, 256, 16, torch.bfloat16, False, "heads"),
    ([100, 41], 3, 3, 256, 48, torch.float16, True, "tokens"),
    ([77], 5, 1, 80, 7, torch.bfloat16, False, "heads"),
    ([90, 17], 17, 1, 40, 5, torch.bfloat16, False, "heads"),
    ([64, 300], 40, 2, 72, 24, torch.bfloat16, True, "heads"),
    ([33], 71, 1, 64, 128, torch.bfloat16, False, "heads"),
    ([50] * 40, 7, 7, 24, 16, torch.float16, False, "heads"),
    ([3] * 300, 2, 1, 32, 4, torch.bfloat16, True, "tokens"),
    ([2500], 8, 2, 248, 33, torch.bfloat16, False, "heads"),
]


@pytest.mark.parametrize("lengths,q_heads,kv_heads,dim,page,dtype,int8,layout", CASES)
def test_matches_64_bits(lengths, q_heads, kv_heads, dim, page, dtype, int8, layout):
    gen = torch.Generator().manual_seed(sum(lengths) + dim)
    check(*make(gen, lengths, q_heads, kv_heads, dim, page, dtype, int8, layout))


@pytest.mark.parametrize("int8", [False, True])
def test_peaked_rows_and_scales(int8):
    gen = torch.Generator().manual_seed(1)
    data = make(gen, [1500, 40], 8, 2, 128, 64, torch.bfloat16, int8, outliers=True)
    for scale in (128**-0.5, 1.0, -0.3, 0.0, 1e-4):
        check(*data, scale=scale)


def test_a_long_sequence_beside_short_ones():
    gen = torch.Generator().manual_seed(2)
    check(*make(gen, [5, 9000, 0, 1, 130], 8, 2, 64, 16, torch.bfloat16))


@pytest.mark.parametrize("q_heads,kv_heads,dim,page,dtype,int8,count", [
    (8, 4, 64, 16, torch.bfloat16, False, 170),   # more items than workgroups, parts found by workgroup
    (8, 4, 64, 24, torch.bfloat16, True, 300),
    (12, 4, 128, 16, torch.float16, False, 150),
    (36, 2, 128, 10, torch.bfloat16, False, 140),  # 18 query heads: two items per K/V head
    (4, 2, 256, 32, torch.bfloat16, True, 150),
    (2, 1, 40, 16, torch.bfloat16, False, 700),    # several sequences per thread of the scan
])
def test_many_sequences_of_very_different_lengths(q_heads, kv_heads, dim, page, dtype, int8, count):
    gen = torch.Generator().manual_seed(count)
    lengths = torch.randint(0, 70, (count,), generator=gen)
    lengths[torch.rand(count, generator=gen) < 0.2] = 0
    lengths[3], lengths[count // 2], lengths[-1] = 3000, 700, 1500
    check(*make(gen, lengths.tolist(), q_heads, kv_heads, dim, page, dtype, int8))


def test_lengths_past_the_table_and_below_zero():
    gen = torch.Generator().manual_seed(3)
    q, pools, scales, table, lengths, dev, dev_scales = make(gen, [64, 32, 48], 4, 2, 64, 16, torch.bfloat16)
    table = table[:, :4].contiguous()
    table[2, 3] = table[0, 0]  # a page of two sequences
    lengths = torch.tensor([10**9, -5, 100], dtype=torch.int32)
    check(q, pools, scales, table, lengths, dev, dev_scales)


def test_pages_outside_the_pool_are_not_seen():
    gen = torch.Generator().manual_seed(4)
    q, pools, scales, table, lengths, dev, dev_scales = make(gen, [200, 60, 33], 8, 2, 64, 16, torch.bfloat16)
    table[0, 0], table[0, 5], table[0, 12] = -1, 10**9, -(2**31)
    table[1, :] = 2**31 - 1  # nothing left
    check(q, pools, scales, table, lengths, dev, dev_scales)


def test_infinite_keys_and_values():
    gen = torch.Generator().manual_seed(5)
    q, pools, scales, table, lengths, dev, dev_scales = make(gen, [100, 70], 4, 2, 64, 16, torch.bfloat16)
    # A key with logit -inf has weight zero; one of minus the type's lowest value too.
    q = q.abs()
    for i, low in ((3, -math.inf), (40, torch.finfo(torch.bfloat16).min)):
        pools[0][table[0, i // 16], i % 16] = low
    dev[0].copy_(pools[0])
    out, lse = paged_decode_attention(q.cuda(), *dev, table.cuda(), lengths.cuda(), return_lse=True)
    keep = [j for j in range(100) if j not in (3, 40)]
    p, r = table[0, torch.tensor(keep) // 16].long(), torch.tensor(keep) % 16
    k, v = pools[0][p, r].double(), pools[1][p, r].double()
    for h in range(4):
        logits = k[:, h // 2] @ q[0, h].double() / 8
        assert abs(float(lse[h, 0]) - float(torch.logsumexp(logits, 0))) < 1e-4
        assert float((out[0, h].double().cpu() - torch.softmax(logits, 0) @ v[:, h // 2]).abs().max()) < 2**-6
    assert bool(torch.isfinite(out).all())
    # Every logit -inf: nothing has weight.
    pools[0][table[1, torch.arange(70) // 16].long(), torch.arange(70) % 16] = -math.inf
    dev[0].copy_(pools[0])
    out, lse = paged_decode_attention(q.cuda(), *dev, table.cuda(), lengths.cuda(), return_lse=True)
    assert bool((out[1] == 0).all()) and bool((lse[:, 1] == -math.inf).all())
    # A value that is not finite shows in its column only.
    pools[1][table[0, 0], 0, 1, 5] = math.nan
    dev[1].copy_(pools[1])
    out = paged_decode_attention(q.cuda(), *dev, table.cuda(), lengths.cuda())
    bad = torch.isnan(out[0]).cpu()
    assert bool(bad[2:, 5].all()) and int(bad.sum()) == 2


def test_strided_q_and_out_and_table():
    gen = torch.Generator().manual_seed(6)
    q, pools, scales, table, lengths, dev, dev_scales = make(gen, [40, 90, 3], 8, 2, 96, 16, torch.bfloat16)
    out, lse = check(q, pools, scales, table, lengths, dev, dev_scales)
    fused = torch.zeros((3, 12, 96), dtype=torch.bfloat16, device="cuda")
    fused[:, :8] = q.cuda()
    wide = torch.full((3, 40), 7, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table.cuda()
    target = torch.full((3, 8, 2, 96), 5.0, dtype=torch.bfloat16, device="cuda")
    got = paged_decode_attention(fused[:, :8], *dev, wide[:, : table.shape[1]], lengths.cuda(), out=target[:, :, 0])
    assert torch.equal(got, out) and bool((target[:, :, 1] == 5).all())
    # Over the query itself.
    paged_decode_attention(fused[:, :8], *dev, wide[:, : table.shape[1]], lengths.cuda(), out=fused[:, :8])
    assert torch.equal(fused[:, :8], out)


def test_no_sequences_and_no_pages():
    pool = torch.zeros((2, 4, 1, 64), dtype=torch.bfloat16, device="cuda")
    q = torch.zeros((0, 2, 64), dtype=torch.bfloat16, device="cuda")
    none = torch.zeros((0, 3), dtype=torch.int32, device="cuda")
    out, lse = paged_decode_attention(q, pool, pool, none, none[:, 0], return_lse=True)
    assert out.shape == (0, 2, 64) and lse.shape == (2, 0)
    q = torch.ones((2, 2, 64), dtype=torch.bfloat16, device="cuda")
    lengths = torch.tensor([5, 0], dtype=torch.int32, device="cuda")
    table = torch.zeros((2, 0), dtype=torch.int32, device="cuda")
    out, lse = paged_decode_attention(q, pool, pool, table, lengths, return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    table = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="no pages"):
        paged_decode_attention(q, pool[:0], pool[:0], table, lengths)


def test_same_bits_every_time_and_on_two_streams():
    gen = torch.Generator().manual_seed(8)
    q, pools, scales, table, lengths, dev, dev_scales = make(gen, [5000, 100, 2000], 32, 8, 128, 64, torch.bfloat16)
    args = (q.cuda(), *dev, table.cuda(), lengths.cuda())
    want, want_lse = paged_decode_attention(*args, return_lse=True)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    results = []
    for _ in range(5):
        for stream in streams:
            with torch.cuda.stream(stream):
                results.append(paged_decode_attention(*args, return_lse=True))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) and torch.equal(l, want_lse) for o, l in results)


def test_two_graphs_replayed_while_the_cache_grows():
    gen = torch.Generator().manual_seed(9)
    lengths = [700, 10, 90]
    q, pools, scales, table, n, dev, dev_scales = make(gen, lengths, 8, 2, 128, 16, torch.bfloat16)
    dq, dtable, dn = q.cuda(), table.cuda(), n.cuda()
    dq2 = torch.randn(q.shape, generator=gen).to(q.dtype).cuda()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        paged_decode_attention(dq, *dev, dtable, dn, return_lse=True)
    torch.cuda.synchronize()
    graphs, results = [], []
    for x in (dq, dq2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            results.append(paged_decode_attention(x, *dev, dtable, dn, return_lse=True))
        graphs.append(graph)
    for shorter in (0, 9, 0, 3):  # the same launch, other lengths
        dn.copy_(n - shorter)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for x, got in zip((dq, dq2), results):
            want = paged_decode_attention(x, *dev, dtable, dn, return_lse=True)
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_pool_past_32_bit_offsets():
    pages, page, heads, dim = 32800, 64, 16, 128
    pool = torch.zeros((pages, heads, page, dim), dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    gen = torch.Generator().manual_seed(10)
    small = torch.randn((3, page, heads, dim), generator=gen).to(torch.bfloat16)
    at = [pages - 1, 3, pages - 2]
    for i, p in enumerate(at):
        pool[p] = small[i].cuda()
    q = torch.randn((1, 32, dim), generator=gen).to(torch.bfloat16)
    lengths = torch.tensor([150], dtype=torch.int32)
    near, far = torch.tensor([[0, 1, 2]], dtype=torch.int32), torch.tensor([at], dtype=torch.int32)
    got = paged_decode_attention(q.cuda(), pool, pool, far.cuda(), lengths.cuda())
    compact = small.cuda()
    want, _ = check(q, (small, small), (None, None), near, lengths, (compact, compact), (None, None))
    assert torch.equal(got, want)
    del pool
    torch.cuda.empty_cache()


@pytest.mark.parametrize("int8", [False, True])
def test_decoding_steps_through_the_cache(int8):
    """Prompts into the cache, then steps that append a token and attend, against 64 bits."""
    gen = torch.Generator().manual_seed(12)
    q_heads, kv_heads, dim, page, prompts = 8, 2, 64, 8, [13, 1, 24]
    cache = DeviceKVCache(32, page, kv_heads, dim, storage_dtype="int8" if int8 else None)
    table = torch.full((3, 6), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(32, generator=gen).tolist()
    freq = rotary_frequencies(32)
    w = (1 + 0.1 * torch.randn(dim, generator=gen)).cuda()
    held = [[], [], []]

    def grow(sequence, rows_, first):
        for j in range(first, first + rows_):
            if j % page == 0:
                table[sequence, j // page] = free.pop()

    def put(sequences, positions):
        n = len(sequences)
        fused = torch.randn((n, q_heads + 2 * kv_heads, dim), generator=gen).to(torch.bfloat16).cuda()
        q, k, v = fused.split([q_heads, kv_heads, kv_heads], dim=1)
        where = torch.tensor(positions, device="cuda")
        slots = cache.slots(table, torch.tensor(sequences, device="cuda"), where)
        assert bool((slots >= 0).all())
        got_q = cache.normalize_rotate_append(q, k, v, slots, where, freq, q_weight=w, k_weight=w)
        assert torch.equal(got_q, normalize_rotate_qk(q, k, where, freq, q_weight=w, k_weight=w)[0])
        k_back, v_back = cache.read(slots)
        if int8:  # the values that the pages stand for
            k_back, v_back = (p[slots // page, slots % page].double() * s[slots // page, slots % page].double()[..., None]
                              for p, s in ((cache.k_pages, cache.k_scales), (cache.v_pages, cache.v_scales)))
        for i, s in enumerate(sequences):
            held[s].append((k_back[i].cpu().double(), v_back[i].cpu().double()))
        return got_q

    for s, n in enumerate(prompts):
        grow(s, n, 0)
        put([s] * n, list(range(n)))
    for step in range(12):
        positions = [len(h) for h in held]
        for s, j in enumerate(positions):
            grow(s, 1, j)
        q = put([0, 1, 2], positions)
        lengths = torch.tensor([len(h) for h in held], dtype=torch.int32, device="cuda")
        out, lse = cache.attend(q, table, lengths, return_lse=True)
        for s in range(3):
            k, v = (torch.stack([row[i] for row in held[s]]) for i in range(2))
            for h in range(q_heads):
                logits = k[:, h // 4] @ q[s, h].double().cpu() / 8
                assert abs(float(lse[h, s]) - float(torch.logsumexp(logits, 0))) < 1e-4
                ref = torch.softmax(logits, 0) @ v[:, h // 4]
                error = (out[s, h].double().cpu() - ref).abs()
                assert bool((error <= 2.0**-8 * ref.abs() + 2.0**-13).all())


def test_refusals():
    gen = torch.Generator().manual_seed(13)
    q, _, _, table, n, (k, v), _ = make(gen, [20, 5], 4, 2, 64, 16, torch.bfloat16)
    q, table, n = q.cuda(), table.cuda(), n.cuda()

    def refused(match, *args, **options):
        with pytest.raises(ValueError, match=match):
            paged_decode_attention(*args, **options)

    refused("layout", q[0], k, v, table, n)
    refused("do not match", q.half(), k, v, table, n)
    refused("divisor of its heads", q[:, :3], k, v, table, n)
    refused("head_dim", q[..., :32], k, v, table, n)
    refused("int32", q, k, v, table.long(), n)
    refused("int32", q, k, v, table, n.long())
    refused("one row per sequence", q, k, v, table[:1], n)
    refused("one row per sequence", q, k, v, table, n[:1])
    refused("contiguous", q, k, v, table.repeat_interleave(2, 1)[:, ::2], n)
    refused("shape of q", q, k, v, table, n, out=q[:1])
    refused("overlap", q, k, v, table, n, out=q[:1].expand(2, 4, 64))
    refused("same shape", q, k, v[:1], table, n)
    refused("need their scales", q, k.to(torch.int8), v.to(torch.int8), table, n)
    refused("device", q, k, v, table.cpu(), n)
    refused("device", q, k, v, table, n.cpu())
    refused("inference-only", q.clone().requires_grad_(), k, v, table, n)
    refused("unit stride", q, k.transpose(2, 3), v, table, n)


# Every form of the kernel: type, kind of pages, padded head_dim (64, 128, 256), 8 or 16 query heads per item, pages
# that do and do not end inside 16 keys.  Sequences that a wave has whole, that are split over a workgroup's waves and
# over workgroups.
@pytest.mark.parametrize("page", [64, 16, 24])
@pytest.mark.parametrize("group", [3, 12, 17])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_form(dtype, int8, dim, group, page):
    gen = torch.Generator().manual_seed(dim + group + page)
    layout = "tokens" if group == 17 else "heads"
    check(*make(gen, [1700, 0, 37, 260], group, 1, dim, page, dtype, int8, layout))


@pytest.mark.parametrize("group,dim,page,dtype,int8", [
    (12, 200, 16, torch.bfloat16, False),
    (16, 248, 40, torch.float16, False),
    (10, 136, 32, torch.float16, True),
    (16, 256, 12, torch.bfloat16, True),
    (12, 96, 16, torch.float16, False),
    (16, 128, 64, torch.bfloat16, True),
    (9, 104, 20, torch.float16, True),
    (16, 56, 16, torch.bfloat16, True),
    (11, 24, 6, torch.float16, False),
])
def test_many_sequences_of_groups_past_eight_heads(group, dim, page, dtype, int8):
    """More items than workgroups, most of them whole in a wave's run of several tiles, some split."""
    gen = torch.Generator().manual_seed(group * dim)
    lengths = torch.randint(0, 90, (700,), generator=gen)
    lengths[torch.rand(700, generator=gen) < 0.2] = 0
    lengths[3], lengths[350], lengths[-1] = 3000, 700, 1500
    check(*make(gen, lengths.tolist(), 2 * group, 2, dim, page, dtype, int8))


def test_an_output_in_the_place_of_other_operands_is_refused():
    gen = torch.Generator().manual_seed(14)
    q, _, _, table, n, (k, v), _ = make(gen, [20, 5, 3, 40], 4, 4, 64, 4, torch.bfloat16, layout="tokens")
    q, table, n = q.cuda(), table.cuda(), n.cuda()
    for out in (k[:4, 0], v[:4, 0], q.transpose(0, 1)):  # [pages, heads, head_dim] rows of the pools
        with pytest.raises(ValueError, match="share memory"):
            paged_decode_attention(q, k, v, table, n, out=out)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("lengths,at", [([100, 40], 70), ([5000, 3], 70), ([5000, 3], 4999), ([33, 1], 32)])
def test_logits_that_are_not_numbers_stay_in_their_head(int8, lengths, at):
    """NaN or +inf: NaN for the head, split over waves and workgroups or not; -inf: a key without weight."""
    gen = torch.Generator().manual_seed(at)
    q, pools, scales, table, n, dev, dev_scales = make(gen, lengths, 8, 2, 64, 16, torch.bfloat16, int8)
    page, row = int(table[0, at // 16]), at % 16
    bad = (0, 1, 2, 3, 5)
    if int8:  # a NaN scale: NaN logits of the K/V head's four query heads
        scales[0][page, row, 0] = math.nan
        dev_scales[0][page, row, 0] = math.nan
    else:
        pools[0][page, row, 0, 7] = math.inf
        dev[0][page, row, 0, 7] = math.inf
        q[0, :4, 7] = torch.tensor([1.0, -1.0, 0.0, 0.25])  # +inf, -inf, NaN, +inf
        bad = (0, 2, 3, 5)
    q[0, 5, 3] = math.nan
    out, lse = paged_decode_attention(q.cuda(), *dev, table.cuda(), n.cuda(), k_scales=dev_scales[0],
                                      v_scales=dev_scales[1], return_lse=True)
    out, lse = out.cpu().double(), lse.cpu().double()
    for h in range(8):
        if h in bad:
            assert bool(torch.isnan(out[0, h]).all()) and math.isnan(lse[h, 0])
    good = [h for h in range(8) if h not in bad]
    ref, ref_lse, size, _ = attention(q, *pools, table, n, 64**-0.5, *scales)
    for s, heads in ((0, good), (1, range(8))):
        for h in heads:
            # Logits of at most 64 products of numbers below 8: e is below 68 * 2^-24 * 2^12 / 8.
            e = 2.0**-9
            bound = 2.0**-8 * ref[s, h].abs() + (1 + 2.0**-8) * (2 * e + 2.0**-15) * size[s, h] + 2.0**-25
            assert bool(((out[s, h] - ref[s, h]).abs() <= bound).all())
            assert abs(float(lse[h, s] - ref_lse[h, s])) <= e + 2.0**-19 * (1 + abs(float(ref_lse[h, s])))


@pytest.mark.parametrize("int8", [False, True])
def test_a_whole_step_captured_with_a_padded_sequence(int8):
    """Slots, norm, rotation, append and attention in one graph, replayed while sequences grow, against the same calls
    made eagerly on another cache; the last sequence is padding (no page, no key)."""
    gen = torch.Generator().manual_seed(15)
    q_heads, kv_heads, dim, page, count = 12, 2, 64, 8, 4
    caches = [DeviceKVCache(24, page, kv_heads, dim, storage_dtype="int8" if int8 else None) for _ in range(2)]
    table = torch.full((count, 6), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(24, generator=gen).tolist()
    lengths = torch.zeros(count, dtype=torch.int32, device="cuda")
    positions, sequences = torch.zeros(count, dtype=torch.int64, device="cuda"), torch.arange(count, device="cuda")
    freq, w = rotary_frequencies(32), torch.ones(dim, device="cuda")
    fused = torch.zeros((count, q_heads + 2 * kv_heads, dim), dtype=torch.bfloat16, device="cuda")
    q, k, v = fused.split([q_heads, kv_heads, kv_heads], dim=1)

    def step(cache):
        slots = cache.slots(table, sequences, positions)
        turned = cache.normalize_rotate_append(q, k, v, slots, positions, freq, q_weight=w, k_weight=w)
        return turned, *cache.attend(turned, table, lengths, return_lse=True)

    stream, spare = torch.cuda.Stream(), DeviceKVCache(1, page, kv_heads, dim, storage_dtype="int8" if int8 else None)
    with torch.cuda.stream(stream):
        step(spare)  # nothing is in the table yet: nothing is written
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = step(caches[0])
    for j in range(20):
        fused.copy_(torch.randn(fused.shape, generator=gen))
        for s in range(count - 1):
            if j % page == 0:
                table[s, j // page] = free.pop()
            positions[s], lengths[s] = j, j + 1
        positions[-1] = j
        graph.replay()
        torch.cuda.synchronize()
        want = step(caches[1])
        assert all(torch.equal(a, b) for a, b in zip(got, want)), j
        assert bool((got[1][-1] == 0).all()) and bool((got[2][:, -1] == -math.inf).all())
        assert bool(torch.isfinite(got[2][:, :-1]).all())
    for a, b in ((caches[0].k_pages, caches[1].k_pages), (caches[0].v_pages, caches[1].v_pages)):
        assert torch.equal(a, b)
