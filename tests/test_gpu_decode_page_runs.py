"""GPU tests of decoding where a wave's keys lie in more than 64 pages, whose numbers it looks up 64 at a time.

Query heads in groups that share K/V make the launch's tiles many and the cache small.
A tile of 32 keys can cross into the next page where pages are a multiple of 16 rows
and not of 32.  Sums go tile by tile whatever the pages, so the result over any pages
is bit for bit the one over pages of 64.

Bounds as in test_gpu_window, but for the sums: a lane adds four times per tile, and the
product with V once, each off by at most 2^-24 of a sum that is at most the final one:
8 tiles 2^-24 of the sum of weight * |v|, and of the sum of the weights.
"""

from __future__ import annotations

import pytest
import torch

from seqattn.kernels import paged_decode_attention
from blocks_reference import values
from paged_reference import HALF_STEP
from test_gpu_window import KINDS, visible

pytestmark = pytest.mark.gpu

DIM, Q_HEADS = 16, 1024
WAVE_TILES = 300  # no case has more in a wave's run


def rows_of(gen, kind, keys, dtype):
    """One of K and V of a sequence: stored rows [keys, DIM], scales (by row, or 16 rows), values in 64 bits."""
    if kind == "rows":
        x = torch.randn((keys, DIM), generator=gen).to(dtype)
        return x, None, x.double()
    if kind == "int8":
        x = torch.randint(-127, 128, (keys, DIM), generator=gen, dtype=torch.int8)
        scale = ((2 + 2 * torch.rand(keys, generator=gen)) / 127).half()
        return x, scale, x.double() * scale.double()[:, None]
    codes = torch.randint(0, 255, (keys, DIM), generator=gen, dtype=torch.uint8)
    codes[codes == 127] = 0
    power = torch.randint(116, 121, (-(-keys // 16),), generator=gen, dtype=torch.uint8)
    each = power.repeat_interleave(16)[:keys]
    stand = values(codes.view(keys, 1, 1, DIM).view(torch.float8_e4m3fn), each.view(keys, 1, 1).view(torch.float8_e8m0fnu))
    return codes, power, stand.view(keys, DIM)


def paged(gen, rows, lengths, page, window, sinks):
    """(page_table, pages, scales) on the device of sequences' K or V rows, in a pool in random order."""
    counts = [-(-n // page) for n in lengths]
    pool_pages = sum(counts) + 1
    order = torch.randperm(pool_pages, generator=gen).to(torch.int32)
    table = torch.full((len(lengths), max(counts)), -1, dtype=torch.int32)
    tensors = []
    for tensor in rows:
        stored, scales = tensor[0][0], tensor[0][1]
        pool = torch.zeros((pool_pages, page, 1, DIM), dtype=stored.dtype)
        per_page = 0 if scales is None else page // 16 if scales.dtype == torch.uint8 else page
        pool_scales = torch.zeros((pool_pages, per_page, 1), dtype=None if scales is None else scales.dtype)
        at = 0
        for (x, scale, _), n, count in zip(tensor, lengths, counts):
            ids = order[at : at + count].long()
            padded = torch.zeros((count * page, DIM), dtype=x.dtype)
            padded[:n] = x
            pool[ids, :, 0] = padded.view(count, page, DIM)
            if scale is not None:
                padded = torch.zeros(count * per_page, dtype=scale.dtype)
                padded[: len(scale)] = scale
                pool_scales[ids, :, 0] = padded.view(count, per_page)
            at += count
        tensors.append((pool.cuda(), None if scales is None else pool_scales.cuda()))
    at = 0
    for s, (n, count) in enumerate(zip(lengths, counts)):
        numbers = (visible(n - 1, window, sinks) // page).unique()
        table[s, numbers] = order[at + numbers]
        at += count
    if tensors[0][0].dtype == torch.uint8:
        tensors = [(p.view(torch.float8_e4m3fn), s.view(torch.float8_e8m0fnu)) for p, s in tensors]
    return table.cuda(), *tensors


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lengths,page,window,sinks", [
    ([120000], 48, None, 0),
    ([70000, 60017, 333], 48, None, 0),
    ([130000], 48, 100000, 50),  # the window starts in page 625
    ([200000], 80, None, 0),
    ([280000], 112, None, 0),
    ([66000], 16, None, 0),
])
def test_runs_of_more_than_64_pages(kind, lengths, page, window, sinks):
    gen = torch.Generator().manual_seed(sum(lengths) + page)
    dtype = torch.bfloat16
    rows = [[rows_of(gen, kind, n, dtype) for n in lengths] for _ in range(2)]
    q = (4 * torch.randn((len(lengths), Q_HEADS, DIM), generator=gen)).to(dtype)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")

    def attend(page):
        table, (k, ks), (v, vs) = paged(gen, rows, lengths, page, window, sinks)
        return paged_decode_attention(q.cuda(), k, v, table, n, window=window, sinks=sinks, k_scales=ks, v_scales=vs,
                                      return_lse=True)

    out, lse = attend(page)
    # Against 64 bits: some heads of every item.
    half = HALF_STEP[dtype]
    for s, length in enumerate(lengths):
        keys = visible(length - 1, window, sinks)
        k, v = (rows[i][s][2][keys] for i in range(2))
        for h in range(0, Q_HEADS, 61):
            x = q[s, h].double()
            logits = k @ x * 0.25
            e = (DIM + 4) * 2.0**-24 * float((k.abs() @ x.abs()).max()) * 0.25
            w = torch.softmax(logits, 0)
            ref, size = w @ v, w @ v.abs()
            bound = half * ref.abs() + (1 + half) * (2 * e + 2.0**-15 + 8 * WAVE_TILES * 2.0**-24) * size + 2.0**-25
            error = (out[s, h].double().cpu() - ref).abs()
            assert bool((error <= bound).all()), (s, h, float((error / bound).max()))
            want = float(torch.logsumexp(logits, 0))
            assert abs(float(lse[h, s]) - want) <= e + 2.0**-19 * (1 + abs(want)) + 8 * WAVE_TILES * 2.0**-24
    for a, b in zip((out, lse), attend(64)):
        assert torch.equal(a, b), int((a != b).sum())
