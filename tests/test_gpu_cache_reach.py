"""GPU tests of the paged cache where its operators' ranges end: thousands of sequences, groups of query heads wider than
a workgroup's rows, pages and rows past 2^32 bytes, captured appends of several rows a sequence."""

from __future__ import annotations

import pytest
import torch

from seqattn import DeviceKVCache
from seqattn.kernels import append_kv_blocks, paged_decode_attention, paged_prefill_attention, read_kv
from test_gpu_prefill import check, make
from test_gpu_window import KINDS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("count,kind", [(4096, "rows"), (4097, "rows"), (6000, "e4m3")])
def test_thousands_of_sequences(count, kind):
    gen = torch.Generator().manual_seed(count)
    new, before = torch.randint(0, 4, (count,), generator=gen), torch.randint(0, 40, (count,), generator=gen)
    new[5], new[-3], new[-2], new[-1] = 300, 0, 0, 2
    check(make(gen, new.tolist(), before.tolist(), 4, 2, 64, 16, kind, window=30, sinks=3), 16, 30, 3, kind=kind)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_group_wider_than_a_block(dim):
    gen = torch.Generator().manual_seed(dim)
    check(make(gen, [3, 1, 20], [0, 100, 50], 400, 1, dim, 16), 16)


@pytest.mark.parametrize("kind", KINDS)
def test_pages_past_32_bit_offsets(kind):
    """The last pages of a pool of more than 2^32 elements hold what a pool of eight pages does, and act alike."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    heads, dim, page, pages = 8, 128, 256, 16384 + 40
    first = pages - 8
    stored = {"rows": torch.bfloat16, "int8": torch.int8, "e4m3": torch.uint8}[kind]
    near = [torch.empty((8, page, heads, dim), dtype=stored, device="cuda") for _ in range(2)]
    far = [torch.empty((pages, page, heads, dim), dtype=stored, device="cuda") for _ in range(2)]
    near_scales = far_scales = [None, None]
    if kind == "int8":
        near_scales = [(torch.rand((8, page, heads), generator=gen, device="cuda") / 30).half() for _ in range(2)]
        far_scales = [torch.zeros((pages, page, heads), dtype=torch.float16, device="cuda") for _ in range(2)]
    if kind == "e4m3":
        shape = (page // 64, heads)
        near_scales = [torch.randint(116, 121, (8, *shape), generator=gen, device="cuda", dtype=torch.uint8) for _ in range(2)]
        far_scales = [torch.zeros((pages, *shape), dtype=torch.uint8, device="cuda") for _ in range(2)]
    for a, b, sa, sb in zip(near, far, near_scales, far_scales):
        if kind == "rows":
            a.copy_(torch.randn(a.shape, generator=gen, device="cuda"))
        else:
            a.random_(*((-127, 128) if kind == "int8" else (0, 120)), generator=gen)
        b[first:] = a
        if sa is not None:
            sb[first:] = sa
    if kind == "e4m3":
        near, far = ([x.view(torch.float8_e4m3fn) for x in pools] for pools in (near, far))
        near_scales, far_scales = ([x.view(torch.float8_e8m0fnu) for x in scales] for scales in (near_scales, far_scales))
    q = torch.randn((500, 16, dim), generator=gen, device="cuda").bfloat16()
    table = torch.tensor([[0, 3, 5, 7], [2, 1, 6, 4]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([1000, 777], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 300, 500], dtype=torch.int32, device="cuda")
    for window in (dict(), dict(window=200, sinks=3)):
        outs = []
        for pools, scales, at in ((near, near_scales, 0), (far, far_scales, first)):
            more = dict(window, k_scales=scales[0], v_scales=scales[1], return_lse=True)
            outs.append((*paged_prefill_attention(q, *pools, table + at, lengths, cu, **more),
                         *paged_decode_attention(q[:2], *pools, table + at, lengths, **more)))
        assert all(torch.equal(a, b) for a, b in zip(*outs))
    if kind == "e4m3":
        k, v = (torch.randn((500, heads, dim), generator=gen, device="cuda").bfloat16() for _ in range(2))
        append_kv_blocks(k, v, *near, *near_scales, table, lengths, cu)
        append_kv_blocks(k, v, *far, *far_scales, table + first, lengths, cu)
        for a, b in zip((*near, *near_scales), (*far, *far_scales)):
            assert torch.equal(a.view(torch.uint8), b[first:].view(torch.uint8))
    slots = torch.arange(0, 8 * page, 3, device="cuda")
    read = lambda pools, scales, at: read_kv(*pools, slots + at * page, k_scales=scales[0], v_scales=scales[1])
    assert all(torch.equal(a, b) for a, b in zip(read(near, near_scales, 0), read(far, far_scales, first)))


def test_rows_past_32_bit_offsets():
    """Tokens whose rows of q and out lie past 2^31 elements; half a step of the largest |v| for the weights and the output."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    tokens, q_heads, kv_heads, dim, page = 310_000, 56, 8, 128, 256
    q = torch.empty((tokens, q_heads, dim), dtype=torch.bfloat16, device="cuda")
    for start in range(0, tokens, 10_000):
        q[start : start + 10_000] = torch.randn((10_000, q_heads, dim), generator=gen, device="cuda")
    pages = -(-tokens // page)
    k, v = (torch.randn((pages, kv_heads, page, dim), generator=gen, device="cuda").bfloat16().transpose(1, 2) for _ in range(2))
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    lengths = torch.tensor([tokens], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, tokens], dtype=torch.int32, device="cuda")
    out, lse = paged_prefill_attention(q, k, v, table, lengths, cu, window=64, return_lse=True)
    for i in (0, 100, 200_000, 299_593, 299_594, tokens - 1):
        keys = torch.arange(max(0, i - 63), i + 1, device="cuda")
        rows_k, rows_v = (x[keys // page, keys % page].double() for x in (k, v))
        for h in (0, 7, 55):
            logits = rows_k[:, h // 7] @ q[i, h].double() * dim**-0.5
            want = torch.softmax(logits, 0) @ rows_v[:, h // 7]
            assert float((out[i, h].double() - want).abs().max()) <= 2.0**-7 * float(rows_v.abs().max())
            assert abs(float(lse[h, i]) - float(torch.logsumexp(logits, 0))) < 1e-4


@pytest.mark.parametrize("storage", [None, "int8", "float8_e4m3fn"])
def test_captured_extensions_follow_lengths_and_starts(storage):
    """Every replay writes what an eager call does: rows below position 0, past the table and behind the last sequence."""
    gen = torch.Generator().manual_seed(5)
    cache, other = (DeviceKVCache(12, 16, 2, 64, storage_dtype=storage) for _ in range(2))
    table = torch.randperm(12, generator=gen).to(torch.int32).view(3, 4).cuda()
    k, v = (torch.zeros((40, 2, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    lengths, cu = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (3, 4))
    other.extend(k, v, table, lengths, cu)  # loads the kernels before the capture
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.extend(k, v, table, lengths, cu)
    for new, after in (([10, 20, 3], [10, 20, 3]), ([0, 5, 20], [10, 25, 23]), ([40, 0, 0], [50, 25, 23]),
                       ([1, 1, 1], [51, 26, 24]), ([30, 2, 8], [20, 28, 70])):
        k.copy_(torch.randn(k.shape, generator=gen)), v.copy_(torch.randn(v.shape, generator=gen))
        cu.copy_(torch.tensor([0, *new]).cumsum(0)), lengths.copy_(torch.tensor(after))
        graph.replay()
        torch.cuda.synchronize()
        other.extend(k, v, table, lengths, cu)
        torch.cuda.synchronize()
        for a, b in ((cache.k_pages, other.k_pages), (cache.v_pages, other.v_pages)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), new
    # No sequences, and tables without pages: nothing is written.
    kept = cache.k_pages.clone()
    cache.extend(k, v, table[:0], lengths[:0], cu[:1])
    cache.extend(k, v, table[:, :0], lengths, cu)
    assert torch.equal(kept.view(torch.uint8), cache.k_pages.view(torch.uint8))
