"""GPU tests of a prompt's attention over the paged cache (``paged_prefill_attention``) against 64 bits.

Bounds.  Logits are FP32 dot products of at most 256 terms and a scale: off by at
most e = (head_dim + 4) 2^-24 of the largest sum of |q k| * scale.  A weight enters
the product with V rounded to q's type (h = 2^-8 or 2^-11 of it; in float16, whose
steps end at 2^-24, also by 2^-25 of the row's largest weight), everything else
is FP32 (2^-15 covers the exponential and sums of thousands of keys).  So the
output is off by (2 e + h + 2^-15) times the sum of weight * |v|, with float16 also
keys 2^-25 max |v|, plus its rounding, and the LSE by e + 2^-19 (1 + |lse|).  K's 8-bit
values are exact, their scales a rounding more of the logits (in the 4); V's INT8
values times their scale are rounded to q's type, h more; e4m3 ones are exact but
for float16, whose steps end at 2^-24.
"""

from __future__ import annotations

import math

import pytest
import torch

from seqattn import DeviceKVCache
from seqattn.kernels import paged_decode_attention, paged_prefill_attention
from paged_reference import HALF_STEP
from test_gpu_window import KINDS, hold, visible

pytestmark = pytest.mark.gpu


def make(gen, new, before, q_heads, kv_heads, dim, page, kind="rows", dtype=torch.bfloat16, window=None, sinks=0, block=16,
         layout="heads"):
    """CPU q, (k, v) values, table, lengths, cu and device pools; rows that no token sees hold NaN, pages without a
    visible key are not in the table."""
    lengths = [a + b for a, b in zip(new, before)]
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + 2
    order = torch.randperm(pages, generator=gen)
    table = torch.full((len(lengths), max([1, *counts]) + 1), -1, dtype=torch.int32)
    seen = torch.zeros((pages, page), dtype=torch.bool)
    at = 0
    for s, (n, c) in enumerate(zip(new, counts)):
        if n > 0:
            keys = torch.cat([visible(p, window, sinks) for p in range(lengths[s] - n, lengths[s])]).unique()
            numbers = (keys // page).unique()
            table[s, numbers] = order[at + numbers].to(torch.int32)
            seen[table[s, keys // page].long(), keys % page] = True
        at += c
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
    q = torch.randn((sum(new), q_heads, dim), generator=gen).to(dtype)
    cu = torch.tensor([0, *new]).cumsum(0).to(torch.int32)
    return q, stand, table, torch.tensor(lengths, dtype=torch.int32), cu, pools, scales


def reference(q, stand, table, lengths, cu, page, scale, window, sinks, device="cpu"):
    """(out, lse, sum of weight * |v|, sum of |q k| * scale, keys) in 64 bits, per row; NaN where a row's logits have one."""
    q, table = q.to(device), table.to(device)
    k_all, v_all = (x.to(device) for x in stand)
    tokens, q_heads, dim = q.shape
    kv_heads = k_all.shape[2]
    group = q_heads // kv_heads
    out, size = (torch.zeros(q.shape, dtype=torch.float64, device=device) for _ in range(2))
    lse = torch.full((q_heads, tokens), -math.inf, dtype=torch.float64, device=device)
    products = torch.zeros((q_heads, tokens), dtype=torch.float64, device=device)
    most = 1
    for s in range(len(lengths)):
        start, stop = int(cu[s]), int(cu[s + 1])
        length = max(0, min(int(lengths[s]), table.shape[1] * page))
        keys = torch.arange(length, device=device)
        ids = table[s, keys // page].long()
        held = (ids >= 0) & (ids < k_all.shape[0])
        rows = (keys % page)[held]
        keys, ids = keys[held], ids[held]
        p = torch.arange(start, stop, device=device) + length - stop
        mask = keys[None] <= p[:, None]
        if window is not None:
            mask &= (p[:, None] - keys[None] < window) | (keys[None] < sinks)
        if not mask.any():
            continue
        some = mask.any(0)  # what nobody sees holds anything
        k, v, mask = k_all[ids, rows][some], v_all[ids, rows][some], mask[:, some]
        most = max(most, int(mask.sum(1).max()))
        for h in range(q_heads):
            x = q[start:stop, h].double()
            kh, vh = k[:, h // group], v[:, h // group]
            logits = (x @ kh.t() * scale).masked_fill(~mask, -math.inf)
            products[h, start:stop] = (x.abs() @ kh.abs().t() * abs(scale)).masked_fill(~mask, 0).amax(1)
            lse[h, start:stop] = torch.logsumexp(logits, 1)
            w = torch.softmax(logits, 1).masked_fill(torch.isneginf(logits).all(1, keepdim=True), 0)
            out[start:stop, h], size[start:stop, h] = w @ vh, w @ vh.abs()
    return out.cpu(), lse.cpu(), size.cpu(), products.cpu(), most


def check(data, page, window=None, sinks=0, scale=None, out=None, padding=0, kind="rows", device="cpu"):
    q, stand, table, lengths, cu, pools, scales = data
    scale = q.shape[2] ** -0.5 if scale is None else scale
    dq = torch.cat([q, torch.full((padding, *q.shape[1:]), math.nan, dtype=q.dtype)]).cuda()
    got, lse = paged_prefill_attention(dq, *pools, table.cuda(), lengths.cuda(), cu.cuda(), softmax_scale=scale,
                                       window=window, sinks=sinks, k_scales=scales[0], v_scales=scales[1], out=out,
                                       return_lse=True)
    ref, ref_lse, size, products, most = reference(q, stand, table, lengths, cu, page, scale, window, sinks, device)
    half = HALF_STEP[q.dtype]
    # Weights in q's dtype; with INT8 V in float16, as V's values times their scale are.
    weight, rounded = (2.0**-12, 2.0**-12) if kind == "int8" else (half, 0.0)
    e = (q.shape[2] + 4) * 2.0**-24 * products
    bound = half * ref.abs() + (1 + half) * (2 * e.t()[..., None] + weight + rounded + 2.0**-15) * size + 2.0**-24
    if q.dtype == torch.float16:
        bound += most * 2.0**-25 * float(size.max())
    tokens = len(q)
    error = (got[:tokens].double().cpu() - ref).abs()
    assert bool((error <= bound).all()), (float((error / bound).max()), (error > bound).nonzero()[:5].tolist())
    lse = lse[:, :tokens].cpu()
    some = torch.isfinite(ref_lse)
    assert torch.equal(torch.isfinite(lse), some) and bool((lse[~some] == -math.inf).all())
    assert bool(((lse.double() - ref_lse).abs()[some] <= (e + 2.0**-19 * (1 + ref_lse.abs()))[some]).all())
    return got, lse


CASES = [
    # new, before, q_heads, kv_heads, head_dim, page, window, sinks
    ([1], [0], 1, 1, 16, 16, None, 0),
    ([5, 0, 1, 64], [0, 7, 63, 0], 8, 2, 64, 16, None, 0),
    ([65, 3, 128], [200, 1000, 0], 8, 1, 128, 32, None, 0),
    ([300], [0], 4, 4, 128, 64, None, 0),
    ([40, 200], [1, 333], 12, 4, 96, 48, None, 0),
    ([130, 70], [0, 90], 4, 2, 256, 32, None, 0),
    ([33], [2000], 56, 8, 128, 256, None, 0),
    ([9, 31], [100, 0], 17, 1, 80, 16, None, 0),
    ([300], [0], 4, 4, 128, 64, 1, 0),
    ([300, 20], [50, 0], 8, 2, 64, 16, 33, 0),
    ([300, 20], [50, 0], 8, 2, 64, 16, 33, 5),
    ([150, 7], [500, 300], 8, 1, 128, 64, 64, 64),
    ([260], [400], 6, 2, 256, 16, 100, 3),
    ([257, 255], [3, 129], 5, 5, 128, 128, 127, 200),
    ([90], [10], 40, 2, 80, 32, 10**6, 4),
    ([2] * 70, [30, 64, 1, 500, 0, 9, 80] * 10, 4, 2, 64, 16, 50, 2),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new,before,q_heads,kv_heads,dim,page,window,sinks", CASES)
def test_matches_64_bits(kind, new, before, q_heads, kv_heads, dim, page, window, sinks):
    gen = torch.Generator().manual_seed(sum(new) + dim + sinks)
    dtype = torch.float16 if (sum(new) + dim) % 3 == 0 else torch.bfloat16
    data = make(gen, new, before, q_heads, kv_heads, dim, page, kind, dtype, window, sinks,
                layout="tokens" if page == 48 else "heads")
    check(data, page, window, sinks, kind=kind)


@pytest.mark.parametrize("kind,page", [("rows", 7), ("rows", 33), ("int8", 5), ("int8", 24)])
def test_pages_that_end_anywhere(kind, page):
    gen = torch.Generator().manual_seed(page)
    for window, sinks in ((None, 0), (45, 6)):
        check(make(gen, [80, 3, 140], [100, 0, 31], 8, 2, 64, page, kind, window=window, sinks=sinks), page, window, sinks,
              kind=kind)


@pytest.mark.parametrize("dim,group,dtype,kind", [(128, 1, torch.bfloat16, "rows"), (128, 3, torch.float16, "rows"),
                                                  (64, 2, torch.bfloat16, "rows"), (256, 1, torch.float16, "rows"),
                                                  (128, 2, torch.bfloat16, "int8"), (128, 5, torch.float16, "e4m3"),
                                                  (64, 1, torch.float16, "e4m3"), (256, 2, torch.bfloat16, "e4m3"),
                                                  (256, 1, torch.float16, "int8"), (64, 2, torch.float16, "int8"),
                                                  (96, 2, torch.bfloat16, "rows"), (200, 1, torch.bfloat16, "rows")])
def test_many_rows(dim, group, dtype, kind):
    """The widest workgroups, which many tiles or a table with room for many choose: items split often."""
    gen = torch.Generator().manual_seed(dim + group)
    for new, before in (([1500], [0]), ([1100, 900], [700, 0])):
        q, stand, table, lengths, cu, pools, scales = make(gen, new, before, group, 1, dim, 64, kind, dtype)
        room = torch.full((len(new), 2**17), -1, dtype=torch.int32)
        room[:, : table.shape[1]] = table
        check((q, stand, room, lengths, cu, pools, scales), 64, kind=kind)


@pytest.mark.parametrize("dim,kv_heads,new,before,window,sinks,kind,dtype", [
    (128, 32, [1700, 900], [300, 0], 500, 9, "rows", torch.bfloat16),
    (128, 12, [1800], [0], None, 0, "rows", torch.float16),
    (128, 24, [1700, 900], [300, 0], 500, 9, "e4m3", torch.float16),
    (128, 24, [1700, 900], [300, 0], 500, 70, "int8", torch.bfloat16),
    (256, 44, [1700, 900], [300, 0], 700, 9, "rows", torch.float16),
    (256, 44, [1700, 900], [300, 0], 700, 9, "e4m3", torch.bfloat16),
    (64, 24, [1700, 900], [300, 0], 400, 9, "rows", torch.bfloat16),
    (64, 24, [1700, 900], [300, 0], 400, 9, "int8", torch.float16),
    (80, 24, [1700, 900], [300, 0], 500, 65, "rows", torch.bfloat16),
])
def test_many_items(dim, kv_heads, new, before, window, sinks, kind, dtype):
    """Wide workgroups with windows, more items than workgroups."""
    gen = torch.Generator().manual_seed(dim + kv_heads)
    data = make(gen, new, before, 4 * kv_heads, kv_heads, dim, 64, kind, dtype, window, sinks)
    check(data, 64, window, sinks, kind=kind, device="cuda")


@pytest.mark.parametrize("kind", KINDS)
def test_calls_repeat_bit_for_bit(kind):
    """Split and whole items, many times: what one wave hands to the others is there in time."""
    gen = torch.Generator().manual_seed(8)
    q, _, table, lengths, cu, pools, scales = make(gen, [1800], [0], 48, 12, 128, 64, kind)
    q, table, lengths, cu = q.cuda(), table.cuda(), lengths.cuda(), cu.cuda()
    run = lambda: paged_prefill_attention(q, *pools, table, lengths, cu, k_scales=scales[0], v_scales=scales[1])
    first = run()
    assert sum(int(not torch.equal(run(), first)) for _ in range(300)) == 0


def test_scales_of_every_kind():
    gen = torch.Generator().manual_seed(1)
    data = make(gen, [150, 20], [33, 400], 8, 2, 128, 64)
    for scale in (1.0, -0.3, 0.0, 1e-4):
        check(data, 64, scale=scale)


def test_e4m3_scales_of_every_size():
    gen = torch.Generator().manual_seed(2)
    for dtype in (torch.bfloat16, torch.float16):
        q, stand, table, lengths, cu, pools, scales = make(gen, [90], [70], 4, 2, 64, 16, "e4m3", dtype)
        k_power = torch.randint(100, 121, scales[0].shape, generator=gen, dtype=torch.uint8)
        k_power[table[0, 0]], k_power[table[0, 1]] = 0, 1
        # float16 holds V up to 448 * 2^7.
        v_power = torch.randint(90 if dtype == torch.float16 else 20, 135 if dtype == torch.float16 else 200,
                                scales[1].shape, generator=gen, dtype=torch.uint8)
        from blocks_reference import values

        for i, power in enumerate((k_power, v_power)):
            scales[i].view(torch.uint8).copy_(power)
            codes = pools[i].view(torch.uint8).cpu()
            stand[i] = values(codes.view(torch.float8_e4m3fn), power.view(torch.float8_e8m0fnu))
        check((q, stand, table, lengths, cu, pools, scales), 16)


@pytest.mark.parametrize("head_dim,group", [(64, 1), (64, 4), (128, 3), (256, 2)])
def test_int8_values_past_float16s_largest(head_dim, group):
    """Values times their scale are held in float16, whose largest stands for what is past it; a window hides some."""
    gen = torch.Generator().manual_seed(head_dim)
    data = make(gen, [150, 70], [41, 0], 2 * group, 2, head_dim, 16, "int8", torch.bfloat16)
    q, stand, table, lengths, cu, pools, scales = data
    for key, scale in ((3, 512.0), (40, 511.75), (64, 6e4), (65, -6e4), (130, 2000.0), (131, 65504.0), (180, 515.5)):
        page, row = int(table[0, key // 16]), key % 16
        scales[1][page, row] = scale
        value = pools[1][page, row].cpu().double() * float(scales[1][page, row, 0])
        stand[1][page, row] = value.clamp(-65504, 65504)
    check(data, 16)
    check(data, 16, 50, 4)
    page, row = int(table[0, 4]), 0
    scales[1][page, row, 0] = math.inf
    out = paged_prefill_attention(q.cuda(), *pools, table.cuda(), lengths.cuda(), cu.cuda(), k_scales=scales[0],
                                  v_scales=scales[1])
    assert not bool(torch.isfinite(out[23:150, :group]).any()) and bool(torch.isfinite(out[:23]).all())
    assert bool(torch.isfinite(out[:150, group:]).all()) and bool(torch.isfinite(out[150:]).all())


def test_float16_takes_8_bit_values_up_to_its_largest():
    q = torch.zeros((1, 1, 64), dtype=torch.float16, device="cuda")
    table, n = torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    cu = torch.arange(2, dtype=torch.int32, device="cuda")
    codes = torch.full((1, 16, 1, 64), 0x78, dtype=torch.uint8, device="cuda")  # 256
    codes[0, 0, 0, 5], codes[0, 0, 0, 6], codes[0, 0, 0, 7] = 0xF8, 0x77, 127  # -256, 240, NaN
    power = torch.full((1, 1, 1), 127 + 8, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    pages = codes.view(torch.float8_e4m3fn)
    keys = torch.zeros_like(codes).view(torch.float8_e4m3fn)
    out = paged_prefill_attention(q, keys, pages, table, n, cu, k_scales=power, v_scales=power)[0, 0].cpu()
    assert out[0] == 65504 and out[5] == -65504 and out[6] == 61440 and torch.isnan(out[7])
    pages = torch.full((1, 16, 1, 64), 127, dtype=torch.int8, device="cuda")
    scale = torch.full((1, 16, 1), 516.0, dtype=torch.float16, device="cuda")
    out = paged_prefill_attention(q, torch.zeros_like(pages), pages, table, n, cu, k_scales=scale, v_scales=scale)
    assert bool((out == 65504).all())
    scale[0, 0, 0] = math.nan
    out = paged_prefill_attention(q, torch.zeros_like(pages), pages, table, n, cu, k_scales=scale * 0, v_scales=scale)
    assert bool(torch.isnan(out).all())


def test_pages_outside_the_pool_lengths_past_the_table_and_below_the_new_tokens():
    gen = torch.Generator().manual_seed(3)
    for kind in KINDS:
        q, stand, table, lengths, cu, pools, scales = make(gen, [60, 90, 64, 20], [240, 0, 0, 100], 4, 2, 64, 16, kind)
        table[0, 0], table[0, 17] = -7, 10**9
        table[2, :] = 2**31 - 1  # nothing left
        table = table[:, :19].contiguous()
        lengths = torch.tensor([10**9, 70, 64, -4], dtype=torch.int32)  # 20 tokens before position 0, all of the last
        lengths[0] = 19 * 16 + 5
        # Keys past a shortened table are not what make() filled: seen rows only up to its own lengths.
        lengths[0] = 300
        check((q, stand, table, lengths, cu, pools, scales), 16, kind=kind)
        check((q, stand, table, lengths, cu, pools, scales), 16, 100, 20, kind=kind)


def test_lengths_past_the_table():
    gen = torch.Generator().manual_seed(4)
    q, stand, table, lengths, cu, pools, scales = make(gen, [100], [60], 4, 2, 64, 16)
    table = table[:, :10].contiguous()  # 160 keys, all of them
    got, lse = check((q, stand, table, lengths, cu, pools, scales), 16)
    more, _ = paged_prefill_attention(q.cuda(), *pools, table.cuda(), (lengths + 10**6).cuda(), cu.cuda(), return_lse=True)
    assert torch.equal(got, more)


def test_infinite_keys_and_values():
    """A key of logit -inf has no weight; values that are not finite show where they are seen, and nowhere else."""
    gen = torch.Generator().manual_seed(5)
    for dim, window in ((64, None), (80, None), (128, 40), (256, 70)):
        q, stand, table, lengths, cu, pools, scales = make(gen, [150], [20], 4, 2, dim, 16, window=window, sinks=0)
        q = q.abs()
        at = lambda j: (int(table[0, j // 16]), j % 16)
        for j, low in ((30, -math.inf), (77, torch.finfo(torch.bfloat16).min)):
            pools[0][at(j)] = low
        for j, h, d, x in ((25, 0, 3, math.nan), (90, 1, dim - 1, math.inf), (140, 0, 9, -math.inf)):
            pools[1][(*at(j), h, d)] = x
        out, lse = paged_prefill_attention(q.cuda(), *pools, table.cuda(), lengths.cuda(), cu.cuda(), window=window,
                                           return_lse=True)
        out, lse = out.double().cpu(), lse.double().cpu()
        k, v = (x[table[0, torch.arange(170) // 16].long(), torch.arange(170) % 16].double().cpu() for x in pools)
        for i in range(150):
            keys = visible(20 + i, window, 0)
            weighted = keys[(keys != 30) & (keys != 77)]
            for h in range(4):
                logits = k[weighted, h // 2] @ q[i, h].double() * dim**-0.5
                want = torch.softmax(logits, 0) @ v[weighted, h // 2]
                size = torch.softmax(logits, 0) @ v[weighted, h // 2].abs()
                bad = ~torch.isfinite(v[keys, h // 2]).all(0)
                assert torch.equal(~torch.isfinite(out[i, h]), bad), (dim, i, h)
                assert abs(float(lse[h, i]) - float(torch.logsumexp(logits, 0))) < 1e-4
                error = (out[i, h] - want).abs()[~bad]
                assert bool((error <= 2.0**-8 * want.abs()[~bad] + 2.0**-7 * size[~bad]).all())


def test_nan_and_infinite_logits_stay_in_their_rows():
    gen = torch.Generator().manual_seed(6)
    q, stand, table, lengths, cu, pools, scales = make(gen, [200], [0], 4, 2, 128, 64)
    call = lambda x: paged_prefill_attention(x.cuda(), *pools, table.cuda(), lengths.cuda(), cu.cuda(), return_lse=True)
    want, want_lse = call(q)
    q[17, 1, 5], q[130, 2, 0], q[131, 3, 7] = math.nan, math.inf, -math.inf
    out, lse = call(q)
    bad = torch.zeros((200, 4), dtype=torch.bool)
    bad[17, 1] = bad[130, 2] = bad[131, 3] = True
    out, want = out.cpu(), want.cpu()
    assert bool(torch.isnan(out[bad]).all()) and torch.equal(out[~bad], want[~bad])
    assert bool(torch.isnan(lse.cpu().t()[bad]).all()) and torch.equal(lse.cpu().t()[~bad], want_lse.cpu().t()[~bad])


def test_rows_behind_the_last_sequence_stay():
    gen = torch.Generator().manual_seed(7)
    data = make(gen, [70, 5], [0, 40], 4, 2, 64, 16)
    out = torch.full((80, 4, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    check(data, 16, out=out, padding=5)
    assert bool((out[75:] == 3).all())


def test_strided_and_in_place():
    gen = torch.Generator().manual_seed(8)
    q, stand, table, lengths, cu, pools, scales = make(gen, [140, 9], [60, 200], 8, 2, 96, 32, layout="tokens")
    got, lse = check((q, stand, table, lengths, cu, pools, scales), 32)
    fused = torch.zeros((149, 12, 96), dtype=torch.bfloat16, device="cuda")
    fused[:, :8] = q.cuda()
    wide = torch.full((2, 40), 7, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table.cuda()
    target = torch.full((149, 8, 2, 96), 5.0, dtype=torch.bfloat16, device="cuda")
    args = *pools, wide[:, : table.shape[1]], lengths.cuda(), cu.cuda()
    out = paged_prefill_attention(fused[:, :8], *args, out=target[:, :, 0])
    assert torch.equal(out, got) and bool((target[:, :, 1] == 5).all())
    paged_prefill_attention(fused[:, :8], *args, out=fused[:, :8])
    assert torch.equal(fused[:, :8], got) and bool((fused[:, 8:] == 0).all())


def test_one_token_each_is_decoding():
    gen = torch.Generator().manual_seed(9)
    for kind in KINDS:
        q, stand, table, lengths, cu, pools, scales = make(gen, [1] * 9, [0, 5, 63, 64, 200, 1000, 31, 32, 77], 8, 2, 128, 64,
                                                           kind, window=90, sinks=3)
        check((q, stand, table, lengths, cu, pools, scales), 64, 90, 3, kind=kind)


def test_nothing_to_attend():
    cache = DeviceKVCache(2, 16, 1, 64)
    none = torch.zeros((0, 2, 64), dtype=torch.bfloat16, device="cuda")
    table, n = torch.zeros((2, 0), dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    cu = torch.zeros(3, dtype=torch.int32, device="cuda")
    out, lse = cache.attend(none, table, n, cu, return_lse=True)
    assert out.shape == (0, 2, 64) and lse.shape == (2, 0)
    q = torch.ones((3, 2, 64), dtype=torch.bfloat16, device="cuda")
    target = torch.full_like(q, 4.0)
    cache.attend(q, table, n, cu, out=target)  # no sequence has a token
    assert bool((target == 4).all())
    cu = torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda")
    out, lse = cache.attend(q, table, n + 5, cu, return_lse=True)  # a table without pages
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    cache.attend(q, table[:0], n[:0], cu[:1], out=target)
    assert bool((target == 4).all())


def test_disordered_starts_stay_inside():
    """cu_tokens that fall or leave the rows: nothing outside the operands is read or written."""
    gen = torch.Generator().manual_seed(10)
    q, stand, table, lengths, cu, pools, scales = make(gen, [30, 30, 30], [50, 0, 9], 4, 2, 64, 16)
    store = torch.full((100, 4, 64), 2.0, dtype=torch.bfloat16, device="cuda")
    for bad in ([0, 90, 0, 90], [-5, 10**9, 3, 400], [90, 60, 30, 0], [2**31 - 1, -(2**31), 5, 9]):
        paged_prefill_attention(q.cuda(), *pools, table.cuda(), lengths.cuda(),
                                torch.tensor(bad, dtype=torch.int32, device="cuda"), out=store[5:95])
    torch.cuda.synchronize()
    assert bool((store[:5] == 2).all()) and bool((store[95:] == 2).all())


def test_a_prompt_in_chunks_then_tokens():
    """A cache takes a prompt chunk by chunk and then tokens; every call attends to all that went before."""
    gen = torch.Generator().manual_seed(11)
    page, window, sinks = 16, 60, 4
    table = torch.randperm(24, generator=gen).to(torch.int32).view(2, 12).cuda()
    for storage in (None, "int8", "float8_e4m3fn"):
        cache = DeviceKVCache(24, page, 2, 64, storage_dtype=storage)
        q = torch.randn((2, 190, 4, 64), generator=gen).to(torch.bfloat16)
        k, v = (torch.randn((2, 190, 2, 64), generator=gen).to(torch.bfloat16) for _ in range(2))
        outs, done = [[], []], [0, 0]
        for chunk in ([100, 3], [0, 80], [50, 57], [1, 1], [1, 1], [38, 48]):
            take = lambda x: torch.cat([x[s, done[s] : done[s] + n] for s, n in enumerate(chunk)]).cuda()
            done_after = [a + n for a, n in zip(done, chunk)]
            lengths = torch.tensor(done_after, dtype=torch.int32, device="cuda")
            cu = torch.tensor([0, *chunk]).cumsum(0).to(torch.int32).cuda()
            one = None if chunk == [1, 1] else cu
            cache.extend(take(k), take(v), table, lengths, one)
            out = cache.attend(take(q), table, lengths, one, window=window, sinks=sinks)
            for s in range(2):
                outs[s].append(out[sum(chunk[:s]) : sum(chunk[: s + 1])].cpu())
            done = done_after
        slots = cache.slots(table, torch.arange(2, device="cuda").repeat_interleave(190), torch.arange(190, device="cuda").repeat(2))
        back = [x.double().cpu().view(2, 190, 2, 64) for x in cache.read(slots)]
        # e4m3 rows can be rounded again, in steps of their block's scale, after they were attended to: at most half
        # the smallest step (2^-10) of a scale of at most 2 * 6 / 448.
        off = {None: 0.0, "int8": 6 * 2.0**-8, "float8_e4m3fn": 2.0**-10 * 12 / 448}[storage]
        p = torch.arange(190)
        mask = (p[None] <= p[:, None]) & ((p[:, None] - p[None] < window) | (p[None] < sinks))
        for s in range(2):
            got = torch.cat(outs[s]).double()
            for h in range(4):
                x = q[s, :, h].double()
                logits = (x @ back[0][s, :, h // 2].t() / 8).masked_fill(~mask, -math.inf)
                e = float((x.abs().sum(1) * (off + 2.0**-8 * 6 * (storage == "int8")) / 8).max()) + 1e-5
                w = torch.softmax(logits, 1)
                want, size = w @ back[1][s, :, h // 2], w @ back[1][s, :, h // 2].abs()
                bound = 2.0**-8 * want.abs() + (math.expm1(2 * e) + 2.0**-7) * size + off
                assert bool(((got[:, h] - want).abs() <= bound).all()), (storage, s, h)


def test_captured_calls_follow_lengths_starts_and_pages():
    gen = torch.Generator().manual_seed(12)
    q, stand, table, lengths, cu, pools, scales = make(gen, [90, 40, 0], [400, 20, 33], 8, 2, 128, 32)
    q, table, lengths, cu = q.cuda(), table.cuda(), lengths.cuda(), cu.cuda()
    call = lambda: paged_prefill_attention(q, *pools, table, lengths, cu, window=100, sinks=2, return_lse=True)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = call()
    for new in ([90, 40, 0], [40, 90, 0], [1, 100, 29], [130, 0, 0], [3, 3, 3]):
        cu.copy_(torch.tensor([0, *new]).cumsum(0))
        lengths.copy_(torch.tensor([400 + new[0], 60 if new[1] < 60 else 60 + new[1] - 60, 33]))
        q.copy_(torch.randn(q.shape, generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        kept = [x.clone() for x in captured]
        eager = call()
        torch.cuda.synchronize()
        n = sum(new)
        assert torch.equal(kept[0][:n].nan_to_num(9), eager[0][:n].nan_to_num(9))
        assert torch.equal(kept[1][:, :n].nan_to_num(9), eager[1][:, :n].nan_to_num(9))


def test_two_streams_and_graphs_have_workspaces_of_their_own():
    gen = torch.Generator().manual_seed(13)
    sets = [make(gen, [200], [300], 8, 2, 128, 64), make(gen, [150, 70], [0, 500], 8, 2, 128, 64)]
    calls = []
    for q, _, table, lengths, cu, pools, _ in sets:
        args = q.cuda(), *pools, table.cuda(), lengths.cuda(), cu.cuda()
        calls.append(lambda a=args: paged_prefill_attention(*a, return_lse=True))
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(10):
        got = []
        for stream, c in zip(streams, calls):
            with torch.cuda.stream(stream):
                got.append(c())
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    graphs = []
    for c in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = c()
        graphs.append((graph, out))
    for _ in range(5):
        for stream, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (_, a), b in zip(graphs, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_refusals():
    q = torch.zeros((3, 4, 64), dtype=torch.bfloat16, device="cuda")
    pool = torch.zeros((2, 16, 2, 64), dtype=torch.bfloat16, device="cuda")
    n, table = torch.ones(2, dtype=torch.int32, device="cuda"), torch.zeros((2, 1), dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda")
    good = dict(q=q, k_pages=pool, v_pages=pool, page_table=table, lengths=n, cu_tokens=cu)
    wide = torch.zeros((2, 16, 2, 72), dtype=torch.int8, device="cuda")
    scale = torch.zeros((2, 16, 2), dtype=torch.float16, device="cuda")
    for bad, word in (
        (dict(cu_tokens=None), "paged_decode_attention"), (dict(cu_tokens=cu.long()), "cu_tokens"),
        (dict(cu_tokens=cu[:2]), "cu_tokens"), (dict(cu_tokens=cu.cpu()), "cu_tokens"), (dict(lengths=n[:1]), "one row per sequence"),
        (dict(page_table=table.long()), "page_table"), (dict(q=q[:, :3]), "divisor"), (dict(q=q[..., :32]), "head_dim"),
        (dict(q=q.float()), "float16 or bfloat16"), (dict(q=q.half()), "do not match"), (dict(window=0), "window"),
        (dict(sinks=1), "sinks"), (dict(window=4, sinks=-1), "sinks"), (dict(out=q[:2]), "shape of q"),
        (dict(out=q.half()), "device and dtype"), (dict(k_scales=scale), "have scales"),
        (dict(q=q.clone().requires_grad_()), "inference-only"),
        (dict(q=torch.zeros((3, 4, 72), dtype=torch.bfloat16, device="cuda"), k_pages=wide, v_pages=wide, k_scales=scale,
              v_scales=scale), "multiples of 16"),
        (dict(out=pool.view(-1)[: 3 * 4 * 64].view(3, 4, 64)), "must not share memory"),
    ):
        with pytest.raises(ValueError, match=word):
            paged_prefill_attention(**{**good, **bad})
