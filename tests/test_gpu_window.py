"""GPU tests of the decoding attention with a sliding window and sinks, and over e4m3 pages, against 64 bits.

Bounds as in test_gpu_decode: logits off by e = (head_dim + 4) 2^-24 of the largest
sum of |q k| * scale, weights by 2^-15 with their two 16-bit parts, FP32 sums, and
the output's rounding.  e4m3 values are exact in 16 bits and their scales enter in
FP32, a rounding more per logit and weight (in the 4 and the 2^-15).
"""

from __future__ import annotations

import math

import pytest
import torch

from seqattn import DeviceKVCache
from seqattn.kernels import paged_decode_attention
from blocks_reference import values
from paged_reference import HALF_STEP

pytestmark = pytest.mark.gpu

KINDS = ["rows", "int8", "e4m3"]


def visible(position, window, sinks):
    """The keys that a token at ``position`` sees."""
    if window is None:
        return torch.arange(position + 1)
    low = max(0, position - window + 1)
    return torch.cat([torch.arange(min(sinks, low)), torch.arange(low, position + 1)])


def hold(gen, kind, shape, dtype, block, seen):
    """Pools of one of K and V on the CPU: (pages, scales, values in 64 bits); rows that nobody sees hold NaN."""
    x = torch.randn(shape, generator=gen)
    if kind == "rows":
        x = x.to(dtype)
        x[~seen] = math.nan
        return x, None, x.double()
    if kind == "int8":
        step = x.abs().amax(-1) / 127
        codes, scale = torch.round(x / step[..., None]).to(torch.int8), step.half()
        scale[~seen] = math.nan
        return codes, scale, codes.double() * scale.double()[..., None]
    codes = torch.randint(0, 255, shape, generator=gen, dtype=torch.uint8)
    codes[codes == 127] = 0
    codes[~seen] = 127  # NaN
    pages, per_page, heads, _ = shape
    power = torch.randint(116, 121, (pages, per_page // block, heads), generator=gen, dtype=torch.uint8)
    power[~seen.view(pages, -1, block).any(-1)] = 255
    codes, power = codes.view(torch.float8_e4m3fn), power.view(torch.float8_e8m0fnu)
    return codes, power, values(codes, power)


def make(gen, lengths, q_heads, kv_heads, dim, page, kind="rows", dtype=torch.bfloat16, window=None, sinks=0, block=16,
         layout="heads"):
    """CPU q, (k, v) values, table, lengths and device pools; what no token sees holds NaN, pages without a visible key
    are not in the table."""
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + 2
    order = torch.randperm(pages, generator=gen)
    table = torch.full((len(lengths), max([1, *counts]) + 1), -1, dtype=torch.int32)
    seen = torch.zeros((pages, page), dtype=torch.bool)
    at = 0
    for s, (n, c) in enumerate(zip(lengths, counts)):
        if n <= 0:
            continue
        keys = visible(n - 1, window, sinks)
        for number in (keys // page).unique().tolist():
            table[s, number] = order[at + number]
        at += c
        seen[table[s, keys // page].long(), keys % page] = True
    shape = (pages, page, kv_heads, dim)
    by_head = (lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)) if layout == "heads" else (lambda t: t)

    def device(t):
        if t is None:
            return None
        raw = t.view(torch.uint8) if t.element_size() == 1 else t
        return by_head(raw.cuda()).view(t.dtype)

    stand, pools, scales = [], [], []
    for _ in range(2):
        codes, scale, value = hold(gen, kind, shape, dtype, block, seen)
        stand.append(value), pools.append(device(codes)), scales.append(device(scale))
    q = torch.randn((len(lengths), q_heads, dim), generator=gen).to(dtype)
    return q, stand, table, torch.tensor(lengths, dtype=torch.int32), pools, scales


def reference(q, stand, table, lengths, page, scale, window, sinks):
    """(out, lse, sum of weight * |v|, largest sum of |q k| * scale) in 64 bits."""
    k_all, v_all = stand
    group = q.shape[1] // k_all.shape[2]
    out, size = (torch.zeros(q.shape, dtype=torch.float64) for _ in range(2))
    lse = torch.full(q.shape[1::-1], -math.inf, dtype=torch.float64)
    products = 0.0
    for s in range(len(q)):
        length = min(int(lengths[s]), table.shape[1] * page)
        if length <= 0:
            continue
        keys = visible(length - 1, window, sinks)
        ids = table[s, keys // page].long()
        held = (ids >= 0) & (ids < k_all.shape[0])
        ids, rows = ids[held], (keys % page)[held]
        if not len(ids):
            continue
        k, v = k_all[ids, rows], v_all[ids, rows]
        for h in range(q.shape[1]):
            x = q[s, h].double()
            logits = k[:, h // group] @ x * scale
            products = max(products, float((k[:, h // group].abs() @ x.abs()).max()) * abs(scale))
            lse[h, s] = torch.logsumexp(logits, 0)
            w = torch.softmax(logits, 0)
            out[s, h], size[s, h] = w @ v[:, h // group], w @ v[:, h // group].abs()
    return out, lse, size, products


def check(data, page, window=None, sinks=0, scale=None):
    q, stand, table, lengths, pools, scales = data
    scale = q.shape[2] ** -0.5 if scale is None else scale
    out, lse = paged_decode_attention(q.cuda(), *pools, table.cuda(), lengths.cuda(), softmax_scale=scale, window=window,
                                      sinks=sinks, k_scales=scales[0], v_scales=scales[1], return_lse=True)
    ref, ref_lse, size, products = reference(q, stand, table, lengths, page, scale, window, sinks)
    e = (q.shape[2] + 4) * 2.0**-24 * products
    half = HALF_STEP[q.dtype]
    bound = half * ref.abs() + (1 + half) * (2 * e + 2.0**-15) * size + 2.0**-25
    error = (out.double().cpu() - ref).abs()
    assert bool((error <= bound).all()), float((error / bound).max())
    some = torch.isfinite(ref_lse)
    assert torch.equal(torch.isfinite(lse.cpu()), some) and bool((lse.cpu()[~some] == -math.inf).all())
    assert bool(((lse.double().cpu() - ref_lse).abs()[some] <= e + 2.0**-19 * (1 + ref_lse[some].abs())).all())
    return out, lse


WINDOWS = [
    # lengths, window, sinks, q_heads, kv_heads, head_dim, page
    ([1, 5, 64, 65, 200], 1, 0, 8, 2, 64, 16),
    ([1, 5, 64, 65, 200], 1, 3, 8, 2, 64, 16),
    ([31, 32, 33, 0, 700], 32, 32, 4, 4, 128, 32),
    ([63, 64, 65, 66, 97, 129], 33, 31, 8, 1, 128, 64),
    ([100, 400, 900], 64, 40, 12, 4, 96, 48),
    ([777, 3], 100, 1, 56, 8, 128, 64),
    ([2000], 512, 4, 17, 1, 256, 256),
    ([500, 600], 250, 300, 4, 2, 80, 16),   # sinks that meet the window
    ([500, 20], 10**6, 5, 4, 2, 40, 16),    # a window past every length
    ([90] * 70, 17, 2, 2, 1, 64, 16),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lengths,window,sinks,q_heads,kv_heads,dim,page", WINDOWS)
def test_window_matches_64_bits(kind, lengths, window, sinks, q_heads, kv_heads, dim, page):
    gen = torch.Generator().manual_seed(sum(lengths) + window % 1000)
    dtype = torch.float16 if sinks % 2 else torch.bfloat16
    layout = "tokens" if page == 48 else "heads"
    check(make(gen, lengths, q_heads, kv_heads, dim, page, kind, dtype, window, sinks, layout=layout), page, window, sinks)


@pytest.mark.parametrize("kind,page", [("rows", 7), ("int8", 5), ("rows", 33)])
def test_windows_over_pages_that_end_anywhere(kind, page):
    gen = torch.Generator().manual_seed(page)
    check(make(gen, [3, 50, 301, 0, 999], 8, 2, 64, page, kind, window=45, sinks=6), page, 45, 6)


@pytest.mark.parametrize("lengths,q_heads,kv_heads,dim,page,block,dtype,layout", [
    ([1], 1, 1, 16, 16, 16, torch.bfloat16, "tokens"),
    ([0, 1, 2, 0, 65], 8, 2, 64, 16, 16, torch.float16, "heads"),
    ([700, 3], 56, 8, 128, 64, 64, torch.bfloat16, "heads"),
    ([257, 255], 12, 4, 96, 256, 32, torch.float16, "tokens"),
    ([100, 511], 4, 4, 256, 64, 32, torch.bfloat16, "heads"),
    ([64, 300], 40, 2, 72, 48, 16, torch.bfloat16, "heads"),
    ([50] * 90, 7, 7, 24, 16, 16, torch.float16, "heads"),
    ([3000, 17], 36, 2, 128, 128, 128, torch.bfloat16, "heads"),
])
def test_e4m3_matches_64_bits(lengths, q_heads, kv_heads, dim, page, block, dtype, layout):
    gen = torch.Generator().manual_seed(sum(lengths) + dim)
    check(make(gen, lengths, q_heads, kv_heads, dim, page, "e4m3", dtype, block=block, layout=layout), page)


def test_e4m3_scales_of_every_size():
    """Scales from 2^-127 to far beyond float16, where K's blocks keep the logits small."""
    gen = torch.Generator().manual_seed(11)
    q, stand, table, lengths, pools, scales = make(gen, [160], 4, 2, 64, 16, "e4m3", torch.float16)
    power = torch.randint(100, 121, scales[0].shape, generator=gen, dtype=torch.uint8)
    power[table[0, 0]], power[table[0, 1]] = 0, 1
    high = torch.randint(0, 160, scales[1].shape, generator=gen, dtype=torch.uint8)
    for i, p in enumerate((power, high)):
        scales[i].view(torch.uint8).copy_(p)
        codes = pools[i].view(torch.uint8).cpu()
        stand[i] = values(codes.view(torch.float8_e4m3fn), p.view(torch.float8_e8m0fnu))
    ref, ref_lse, size, products = reference(q, stand, table, lengths, 16, 0.125, None, 0)
    out, lse = paged_decode_attention(q.bfloat16().cuda(), *pools, table.cuda(), lengths.cuda(), softmax_scale=0.125,
                                      k_scales=scales[0], v_scales=scales[1], return_lse=True)
    ref, ref_lse, size, products = reference(q.bfloat16(), stand, table, lengths, 16, 0.125, None, 0)
    e = 68 * 2.0**-24 * products
    bound = 2.0**-8 * ref.abs() + (1 + 2.0**-8) * (2 * e + 2.0**-15) * size + 2.0**-25
    assert bool(((out.double().cpu() - ref).abs() <= bound).all())
    assert bool(((lse.double().cpu() - ref_lse).abs() <= e + 2.0**-19 * (1 + ref_lse.abs())).all())


def test_pages_outside_the_pool_and_lengths_past_the_table():
    gen = torch.Generator().manual_seed(12)
    for kind in KINDS:
        q, stand, table, lengths, pools, scales = make(gen, [300, 90, 64], 4, 2, 64, 16, kind, window=100, sinks=20)
        table[0, 0], table[0, 15] = -7, 10**9
        table[2, :] = 2**31 - 1  # nothing left
        table[1, 5:] = -1
        table = table[:, :19].contiguous()
        lengths = torch.tensor([10**9, 90, -4], dtype=torch.int32)
        lengths[0] = 300
        check((q, stand, table, lengths, pools, scales), 16, 100, 20)


def test_a_window_over_everything_is_no_window():
    gen = torch.Generator().manual_seed(13)
    for kind in KINDS:
        q, _, table, lengths, pools, scales = make(gen, [900, 33, 257], 8, 2, 128, 64, kind)
        call = lambda **w: paged_decode_attention(q.cuda(), *pools, table.cuda(), lengths.cuda(), k_scales=scales[0],
                                                  v_scales=scales[1], return_lse=True, **w)
        for a, b in zip(call(), call(window=900, sinks=3)):
            assert torch.equal(a, b)


def test_many_windowed_sequences_of_very_different_lengths():
    gen = torch.Generator().manual_seed(14)
    lengths = torch.randint(0, 400, (330,), generator=gen)
    lengths[3], lengths[200], lengths[-1] = 9000, 0, 5000
    for kind in ("rows", "e4m3"):
        check(make(gen, lengths.tolist(), 4, 2, 64, 16, kind, window=150, sinks=5), 16, 150, 5)


def test_a_decoding_run_appends_and_attends():
    """Tokens go into a cache one by one and attend to it through a window, on every kind of pages, in and out of a graph."""
    gen = torch.Generator().manual_seed(15)
    page, window, sinks = 16, 30, 2
    table = torch.randperm(12, generator=gen).to(torch.int32).view(2, 6).cuda()
    for storage in (None, "int8", "float8_e4m3fn"):
        cache = DeviceKVCache(12, page, 2, 64, storage_dtype=storage)
        other = DeviceKVCache(12, page, 2, 64, storage_dtype=storage)
        q = torch.randn((2, 4, 64), generator=gen).to(torch.bfloat16).cuda()
        k, v = (torch.zeros((2, 2, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        lengths = torch.ones(2, dtype=torch.int32, device="cuda")

        def step(c):
            c.extend(k, v, table, lengths)
            return c.attend(q, table, lengths, window=window, sinks=sinks, return_lse=True)

        step(other)  # loads the kernels before the capture
        other.k_pages.view(torch.uint8).zero_(), other.v_pages.view(torch.uint8).zero_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = step(cache)
        for t in range(80):
            lengths.fill_(t + 1)
            k.copy_(torch.randn((2, 2, 64), generator=gen)), v.copy_(torch.randn((2, 2, 64), generator=gen))
            graph.replay()
            eager = step(other)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(captured, eager)), (storage, t)
        # What was attended to is what reads back.
        slots = cache.slots(table, torch.arange(2, device="cuda").repeat_interleave(80), torch.arange(80, device="cuda").repeat(2))
        rows = [x.double().cpu().view(2, 80, 2, 64) for x in cache.read(slots)]
        keys = visible(79, window, sinks)
        for s in range(2):
            for h in range(4):
                logits = rows[0][s, keys, h // 2] @ q[s, h].double().cpu() / 8
                want = torch.softmax(logits, 0) @ rows[1][s, keys, h // 2]
                # The rows that read back are rounded to bfloat16 once (INT8), half a step of values up to 5.
                assert float((captured[0][s, h].double().cpu() - want).abs().max()) <= 5 * 2.0**-8 * 3


def test_refusals():
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16, device="cuda")
    pool = torch.zeros((2, 16, 2, 64), dtype=torch.bfloat16, device="cuda")
    n = torch.ones(2, dtype=torch.int32, device="cuda")
    table = torch.zeros((2, 1), dtype=torch.int32, device="cuda")
    e4m3 = torch.zeros((2, 16, 2, 64), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scales = torch.zeros((2, 1, 2), dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    for more, word in ((dict(window=0), "window"), (dict(window=-3), "window"), (dict(sinks=1), "sinks"),
                       (dict(window=4, sinks=-1), "sinks")):
        with pytest.raises(ValueError, match=word):
            paged_decode_attention(q, pool, pool, table, n, **more)
    with pytest.raises(ValueError, match="e4m3 pages need their scales"):
        paged_decode_attention(q, e4m3, e4m3, table, n)
    with pytest.raises(ValueError, match="float8_e8m0fnu"):
        paged_decode_attention(q, e4m3, e4m3, table, n, k_scales=scales.view(torch.uint8), v_scales=scales.view(torch.uint8))
    with pytest.raises(ValueError, match="have scales"):
        paged_decode_attention(q, pool, pool, table, n, k_scales=scales, v_scales=scales)
