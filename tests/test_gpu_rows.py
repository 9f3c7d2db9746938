"""GPU tests of the norm, rotation and cache rows (``seqattn.kernels.rows``) against 64 bits.

Bounds.  A 16-bit result is rounded once: half a step of its value.  Before
that it is FP32: the norm's sum of at most 256 squares (a tree of FP32
additions), the reciprocal root, two products and the rotation's two come to
under 16 roundings of 2^-24 of the pair's size; the sine and cosine
instructions are within 2^-20 (their input is the FP64 angle's fraction of a
turn, rounded to 2^-26).  So 2^-18 of the pair's size covers both.  INT8 adds
half a step of the row's code, the scale's FP16 rounding (2^-11) and the
rounding of the value read back.
"""

from __future__ import annotations

import pytest
import torch

from seqattn import DeviceKVCache, rotary_frequencies
from seqattn.kernels import append_kv, normalize_rotate_append, normalize_rotate_qk, paged_decode_attention, read_kv
from paged_reference import HALF_STEP, normalized, quantized, rotated

pytestmark = pytest.mark.gpu

FP32 = 2.0**-18


def rows(gen, *shape, dtype):
    return torch.randn(shape, generator=gen).to(dtype)


def close(got, ref, size, dtype):
    error = (got.double().cpu() - ref).abs()
    bound = HALF_STEP[dtype] * (ref.abs() + FP32 * size) + FP32 * size + 2.0**-24
    assert bool((error <= bound).all()), float((error / bound).max())


CASES = [
    # tokens, q_heads, kv_heads, head_dim, sections, pairing, dtype
    (1, 1, 1, 16, (8,), "halves", torch.bfloat16),
    (3, 4, 2, 128, (16, 24, 24), "halves", torch.bfloat16),
    (7, 5, 1, 128, (64,), "adjacent", torch.float16),
    (2, 8, 2, 80, (20,), "halves", torch.float16),       # partial, runs of 4 pairs
    (5, 3, 3, 96, (11, 6), "halves", torch.bfloat16),    # 17 pairs: element by element
    (4, 2, 2, 72, (36,), "halves", torch.bfloat16),      # runs of 4
    (4, 2, 1, 24, (5,), "adjacent", torch.bfloat16),     # partial, an odd number of pairs
    (3, 6, 2, 256, (32, 48, 48), "halves", torch.float16),
    (2, 2, 2, 256, (127,), "halves", torch.bfloat16),    # element by element, 64 lanes
    (9, 40, 8, 64, (8, 8, 8, 8), "adjacent", torch.bfloat16),
    (300, 33, 11, 40, (16,), "halves", torch.bfloat16),
    (2, 3, 1, 248, (62,), "halves", torch.bfloat16),
]


@pytest.mark.parametrize("tokens,q_heads,kv_heads,dim,sections,pairing,dtype", CASES)
@pytest.mark.parametrize("weights", ["both", "q", "none"])
def test_normalize_rotate_matches_64_bits(tokens, q_heads, kv_heads, dim, sections, pairing, dtype, weights):
    gen = torch.Generator().manual_seed(tokens * 1000 + dim)
    # Views of one projection's output.
    fused = rows(gen, tokens, q_heads + 2 * kv_heads, dim, dtype=dtype)
    wq = (1 + 0.2 * torch.randn(dim, generator=gen)).to(dtype) if weights != "none" else None
    wk = 1 + 0.2 * torch.randn(dim, generator=gen) if weights == "both" else None  # float32
    positions = torch.randint(-5000, 2**31 - 1, (len(sections), tokens), generator=gen)
    freq = rotary_frequencies(sections, shared=len(sections) == 2, device="cpu")
    dev = fused.cuda()
    q, k, _ = dev.split([q_heads, kv_heads, kv_heads], dim=1)
    qo, ko = normalize_rotate_qk(q, k, positions.cuda(), freq.cuda(), sections=sections, pairing=pairing,
                                 q_weight=None if wq is None else wq.cuda(), k_weight=None if wk is None else wk.cuda(),
                                 eps=1e-5)
    for got, start, heads, w in ((qo, 0, q_heads, wq), (ko, q_heads, kv_heads, wk)):
        ref, size = rotated(normalized(fused[:, start : start + heads], w, 1e-5), positions, freq, sections, pairing)
        close(got, ref, size, dtype)


def test_far_positions_and_int32_positions():
    gen = torch.Generator().manual_seed(5)
    x = rows(gen, 6, 2, 64, dtype=torch.float16)
    freq = rotary_frequencies(32, device="cpu")
    far = torch.tensor([0, 1, -1, 2**31 - 1, 2**40 + 3, -(2**38) - 7])
    q, _ = normalize_rotate_qk(x.cuda(), x.cuda(), far.cuda(), freq.cuda())
    # The angle in 64 bits is off by 2^-53 of 2^40 radians, 2^-13; both sides
    # have the same products.  Positions below 2^31 hold the tight bound.
    ref, size = rotated(x.double(), far[None], freq, (32,), "halves")
    error = (q.double().cpu() - ref).abs()
    assert bool((error[:4] <= HALF_STEP[x.dtype] * (ref[:4].abs() + FP32 * size[:4]) + FP32 * size[:4]).all())
    assert bool((error[4:] <= HALF_STEP[x.dtype] * ref[4:].abs() + 2.0**-11 * size[4:]).all())
    near = far[:4].to(torch.int32)
    same, _ = normalize_rotate_qk(x[:4].cuda(), x[:4].cuda(), near.cuda(), freq.cuda())
    assert torch.equal(same, q[:4])


def test_in_place_strided_outputs_and_no_tokens():
    gen = torch.Generator().manual_seed(7)
    fused = rows(gen, 10, 8, 96, dtype=torch.bfloat16).cuda()
    freq, pos = rotary_frequencies(48), torch.arange(10, device="cuda")
    w = torch.ones(96, device="cuda")
    q, k = fused[:, :6], fused[:, 6:]
    want = normalize_rotate_qk(q, k, pos, freq, q_weight=w, k_weight=w)
    by_head = torch.zeros((6, 10, 96), dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    got = normalize_rotate_qk(q, k, pos, freq, q_weight=w, k_weight=w, q_out=by_head, k_out=k)
    assert got[0] is by_head and torch.equal(by_head, want[0]) and torch.equal(k, want[1])
    empty = normalize_rotate_qk(fused[:0, :6], fused[:0, 6:], pos[:0], freq)
    assert empty[0].shape == (0, 6, 96)
    # Norm alone.
    q2, k2 = normalize_rotate_qk(want[0], want[1], q_weight=w)
    assert torch.equal(k2, want[1])
    ref = normalized(want[0].cpu(), w.cpu(), 1e-6)
    close(q2, ref, ref.abs(), torch.bfloat16)


def test_zero_rows_and_non_finite_rows_stay_in_their_head():
    x = torch.zeros((4, 2, 64), dtype=torch.bfloat16, device="cuda")
    x[1, 0] = float("inf")
    x[2, 1] = float("nan")
    x[3] = 1.0
    freq, pos = rotary_frequencies(32), torch.arange(4, device="cuda")
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16)
    q, k = normalize_rotate_qk(x, x, pos, freq, q_weight=w, k_weight=w, eps=1e-6)
    assert torch.equal(q.nan_to_num(7.0), k.nan_to_num(7.0))
    assert bool((q[0] == 0).all()) and bool((q[1, 1] == 0).all()) and bool((q[2, 0] == 0).all())
    assert not bool(torch.isfinite(q[1, 0]).any()) and bool(torch.isnan(q[2, 1]).all())
    assert bool(torch.isfinite(q[3]).all())


def pools(pages, page, heads, dim, dtype, layout, int8):
    if layout == "heads":
        make = lambda *s, t: torch.full((s[0], s[2], s[1], *s[3:]), 3, dtype=t, device="cuda").transpose(1, 2)  # noqa: E731
    else:
        make = lambda *s, t: torch.full(s, 3, dtype=t, device="cuda")  # noqa: E731
    stored = torch.int8 if int8 else dtype
    k, v = make(pages, page, heads, dim, t=stored), make(pages, page, heads, dim, t=stored)
    if not int8:
        return k, v, None, None
    return k, v, make(pages, page, heads, t=torch.float16), make(pages, page, heads, t=torch.float16)


def int8_close(got, rows_, size, dtype):
    """Values read back from INT8 pages against the rows that went in."""
    codes, _, step = quantized(rows_)
    error = (got.double().cpu() - rows_).abs()
    row_size = size.amax(-1, keepdim=True)
    bound = (0.5 + 127 * 2.0**-11) * step[..., None] * (1 + 2.0**-7) + 2 * FP32 * row_size + HALF_STEP[dtype] * got.double().cpu().abs() + 2.0**-24
    assert bool((error <= bound).all()), float((error / bound).max())


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
@pytest.mark.parametrize("tokens,heads,dim,page,dtype", [
    (1, 1, 16, 1, torch.bfloat16), (37, 3, 80, 5, torch.float16), (200, 8, 128, 64, torch.bfloat16),
    (11, 2, 256, 16, torch.bfloat16), (19, 5, 24, 7, torch.float16)])
def test_append_and_read(tokens, heads, dim, page, dtype, layout, int8):
    gen = torch.Generator().manual_seed(tokens)
    k, v = rows(gen, tokens, heads, dim, dtype=dtype), rows(gen, tokens, heads, dim, dtype=dtype)
    k[0, 0] = 0  # a row of zeros
    pages = -(-tokens // page) + 2
    kp, vp, ks, vs = pools(pages, page, heads, dim, dtype, layout, int8)
    slots = torch.randperm(pages * page, generator=gen)[:tokens]
    before = [t.clone() for t in (kp, vp)]
    append_kv(k.cuda(), v.cuda(), kp, vp, slots.cuda(), k_scales=ks, v_scales=vs)
    ko, vo = read_kv(kp, vp, slots.cuda(), k_scales=ks, v_scales=vs, dtype=dtype)
    for got, x, pool, scale in ((ko, k, kp, ks), (vo, v, vp, vs)):
        if not int8:
            assert torch.equal(got.cpu(), x)
            assert torch.equal(pool.cpu()[slots // page, slots % page], x)
            continue
        # Rows that are not rotated are quantized from the same floats as the
        # storage format's, with the same operations.
        step = x.float().abs().amax(-1) / 127.0
        step = torch.where(step > 0, step, torch.ones_like(step))
        codes = torch.round(x.float() / step[..., None]).clamp(-127, 127)
        assert torch.equal(pool.cpu()[slots // page, slots % page].float(), codes)
        assert torch.equal(scale.cpu()[slots // page, slots % page], step.half())
        assert torch.equal(got.cpu(), (codes * step.half().float()[..., None]).to(dtype))
    # Rows of no slot of this call keep what they held.
    untouched = torch.ones(pages * page, dtype=torch.bool)
    untouched[slots] = False
    at = untouched.nonzero().squeeze(1)
    for pool, old in zip((kp, vp), before):
        assert torch.equal(pool[at // page, at % page], old[at // page, at % page])


def test_slots_outside_the_pool_are_skipped_and_read_as_zeros():
    k = torch.ones((6, 2, 32), dtype=torch.bfloat16, device="cuda")
    kp, vp, _, _ = pools(2, 4, 2, 32, torch.bfloat16, "heads", False)
    slots = torch.tensor([-1, 8, 5, 2**40, -(2**40), 2**31], device="cuda")
    append_kv(k, k, kp, vp, slots)
    held = torch.zeros((2, 4), dtype=torch.bool)
    held[1, 1] = True
    assert bool((kp.cpu()[held] == 1).all()) and bool((kp.cpu()[~held] == 3).all())
    ko, vo = read_kv(kp, vp, slots)
    assert bool((ko[2] == 1).all()) and bool((vo[2] == 1).all())
    assert bool((ko[[0, 1, 3, 4, 5]] == 0).all())


def test_int8_rows_that_are_not_finite_read_back_as_nan():
    k = torch.ones((3, 2, 32), dtype=torch.bfloat16, device="cuda")
    k[0, 0, 3] = float("inf")
    k[1, 1, 31] = float("nan")
    kp, vp, ks, vs = pools(1, 4, 2, 32, torch.bfloat16, "heads", True)
    slots = torch.arange(3, device="cuda")
    append_kv(k, k, kp, vp, slots, k_scales=ks, v_scales=vs)
    got, _ = read_kv(kp, vp, slots, k_scales=ks, v_scales=vs)
    assert bool(torch.isnan(got[0, 0]).all()) and bool(torch.isnan(got[1, 1]).all())
    assert bool((got[0, 1] - 1).abs().max() < 2**-7) and bool((got[2] - 1).abs().max() < 2**-7)


@pytest.mark.parametrize("tokens,q_heads,kv_heads,dim,sections,pairing,dtype", CASES)
@pytest.mark.parametrize("int8", [False, True])
def test_fused_append_matches_the_parts(tokens, q_heads, kv_heads, dim, sections, pairing, dtype, int8):
    gen = torch.Generator().manual_seed(dim + tokens)
    fused = rows(gen, tokens, q_heads + 2 * kv_heads, dim, dtype=dtype)
    positions = torch.randint(0, 10**6, (len(sections), tokens), generator=gen)
    freq = rotary_frequencies(sections, device="cpu")
    wq, wk = ((1 + 0.2 * torch.randn(dim, generator=gen)).to(dtype) for _ in range(2))
    q, k, v = fused.cuda().split([q_heads, kv_heads, kv_heads], dim=1)
    options = dict(sections=sections, pairing=pairing, q_weight=wq.cuda(), k_weight=wk.cuda())
    q_ref, k_ref = normalize_rotate_qk(q, k, positions.cuda(), freq.cuda(), **options)
    cache = DeviceKVCache(tokens // 4 + 2, 4, kv_heads, dim, dtype=dtype, storage_dtype="int8" if int8 else None)
    slots = torch.randperm(cache.num_pages * 4, generator=gen)[:tokens].cuda()
    q_out = cache.normalize_rotate_append(q, k, v, slots, positions.cuda(), freq.cuda(), **options)
    assert torch.equal(q_out, q_ref)
    ko, vo = cache.read(slots)
    if not int8:
        assert torch.equal(ko, k_ref) and torch.equal(vo, v)
        return
    ref, size = rotated(normalized(fused[:, q_heads : q_heads + kv_heads], wk, 1e-6), positions, freq, sections, pairing)
    int8_close(ko, ref, size, dtype)
    int8_close(vo, fused[:, q_heads + kv_heads :].double(), fused[:, q_heads + kv_heads :].double().abs(), dtype)


def test_pools_past_32_bit_offsets():
    # The last pages of a pool of 2^32 elements and more: one buffer serves as
    # K and, 64 rows of one head further, as V.
    pages, page, heads, dim = 32800, 64, 16, 128
    pool = torch.zeros((pages, heads, page, dim), dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    assert pool.numel() > 2**32
    k = torch.randn((3, heads, dim), device="cuda").to(torch.bfloat16)
    k_pool, v_pool = pool[: pages // 2 + 16385], pool
    slots = torch.tensor([pages * page - 1, pages * page - 64, 5], device="cuda")
    append_kv(k, k, v_pool, v_pool, slots)
    ko, vo = read_kv(v_pool, v_pool, slots)
    assert torch.equal(ko, k) and torch.equal(vo, k)
    assert torch.equal(pool[pages - 1, page - 1], k[0]) and torch.equal(pool[0, 5], k[2])
    assert k_pool.shape[0] < pages
    del pool, k_pool, v_pool
    torch.cuda.empty_cache()


@pytest.mark.parametrize("int8", [False, True])
def test_a_launch_past_the_caches_equals_its_parts(int8):
    """From 256 MB on a launch reads and writes past the caches: the same rows as in small launches."""
    tokens, q_heads, kv_heads, dim = 9001, 48, 8, 128
    gen = torch.Generator(device="cuda").manual_seed(3)
    fused = torch.randn((tokens, q_heads + 2 * kv_heads, dim), generator=gen, device="cuda").to(torch.bfloat16)
    assert fused.numel() * 4 >= 256 << 20
    q, k, v = fused.split([q_heads, kv_heads, kv_heads], dim=1)
    freq, pos = rotary_frequencies((16, 24, 24)), torch.arange(3 * tokens, device="cuda").view(3, tokens)
    options = dict(sections=(16, 24, 24), q_weight=torch.ones(dim, device="cuda"), k_weight=torch.ones(dim, device="cuda"))
    slots = torch.randperm(9024, generator=gen, device="cuda")[:tokens]
    caches = [DeviceKVCache(141, 64, kv_heads, dim, storage_dtype="int8" if int8 else None) for _ in range(2)]
    whole = caches[0].normalize_rotate_append(q, k, v, slots, pos, freq, **options)
    parts = [caches[1].normalize_rotate_append(q[i : i + 1000], k[i : i + 1000], v[i : i + 1000], slots[i : i + 1000],
                                               pos[:, i : i + 1000], freq, **options) for i in range(0, tokens, 1000)]
    assert torch.equal(whole, torch.cat(parts))
    for a, b in zip(caches[0].read(slots), caches[1].read(slots)):
        assert torch.equal(a, b)
    # All of Q and K turned in place.
    want = normalize_rotate_qk(q, k, pos, freq, **options)
    assert torch.equal(want[0], whole)
    normalize_rotate_qk(q, k, pos, freq, q_out=q, k_out=k, **options)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


@pytest.mark.parametrize("heads", [1, 2, 3, 9])
@pytest.mark.parametrize("dim", [16, 64, 72, 128, 256])
def test_appends_of_few_and_many_heads(heads, dim):
    """Both forms of the append, 16-bit rows of every head count next to a wave's."""
    gen = torch.Generator().manual_seed(heads * dim)
    tokens = 133
    k, v = (rows(gen, tokens, heads, dim, dtype=torch.bfloat16).cuda() for _ in range(2))
    cache = DeviceKVCache(20, 8, heads, dim)
    slots = torch.randperm(160, generator=gen)[:tokens].cuda()
    slots[7], slots[132] = -1, 160
    cache.append(k, v, slots)
    ko, vo = cache.read(slots)
    k[[7, 132]], v[[7, 132]] = 0, 0
    assert torch.equal(ko, k) and torch.equal(vo, v)


def test_replayed_graph_and_other_stream():
    gen = torch.Generator().manual_seed(11)
    fused = rows(gen, 5, 8, 64, dtype=torch.bfloat16).cuda()
    q, k, v = fused.split([4, 2, 2], dim=1)
    freq, pos = rotary_frequencies(32), torch.arange(5, device="cuda")
    cache = DeviceKVCache(4, 4, 2, 64)
    slots = torch.arange(5, device="cuda")
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        cache.normalize_rotate_append(q, k, v, slots, pos, freq)
        cache.read(slots)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        q_out = cache.normalize_rotate_append(q, k, v, slots, pos, freq)
        ko, vo = cache.read(slots)
    for step in range(4):
        fused.copy_(rows(gen, 5, 8, 64, dtype=torch.bfloat16))
        pos.add_(17 * step)
        slots.copy_(torch.randperm(16, generator=gen)[:5])
        graph.replay()
        torch.cuda.synchronize()
        want_q, want_k = normalize_rotate_qk(q, k, pos, freq)
        assert torch.equal(q_out, want_q) and torch.equal(ko, want_k) and torch.equal(vo, v)


def test_refusals():
    q = torch.zeros((4, 4, 64), dtype=torch.bfloat16, device="cuda")
    k = torch.zeros((4, 2, 64), dtype=torch.bfloat16, device="cuda")
    freq, pos = rotary_frequencies(32), torch.arange(4, device="cuda")
    w = torch.ones(64, device="cuda")

    def refused(match, *args, **options):
        with pytest.raises(ValueError, match=match):
            normalize_rotate_qk(*args, **options)

    refused("needs a weight or a rotation", q, k)
    refused("both positions and frequencies", q, k, pos)
    refused("both positions and frequencies", q, k, None, freq)
    refused("same tokens and head_dim", q, k[:3], pos, freq)
    refused("device and dtype", q, k.half(), pos, freq)
    refused("no heads", q, k[:, :0], pos, freq)
    refused("no heads", q[:, :0], k, pos, freq)
    refused("float16 or bfloat16", q.float(), k.float(), pos, freq)
    refused("multiple of 8", q[..., :12], k[..., :12], pos, freq[:6])
    refused("unit stride", q.transpose(1, 2), k, pos, freq)
    refused("aligned", torch.zeros(4 * 4 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(4, 4, 64), k, pos, freq)
    refused("float64", q, k, pos, freq.float())
    refused("head_dim / 2 pairs", q, k, pos, rotary_frequencies(33))
    refused("positions must be", q, k, pos, freq, sections=(16, 16))
    refused("add up to the pairs", q, k, pos, freq, sections=(16, 15))
    refused("add up to the pairs", q, k, pos.expand(5, 4), freq, sections=(8, 8, 8, 4, 4))
    refused("one position per token", q, k, pos[:3], freq)
    refused("int32 or int64", q, k, pos.float(), freq)
    refused("pairing", q, k, pos, freq, pairing="pairs")
    refused("q_weight", q, k, pos, freq, q_weight=w[:32])
    refused("dtype or float32", q, k, pos, freq, k_weight=w.half())
    refused("eps", q, k, pos, freq, q_weight=w, eps=-1.0)
    refused("eps", q, k, pos, freq, q_weight=w, eps=float("nan"))
    refused("shape of its input", q, k, pos, freq, q_out=k.clone())
    refused("overlap", q, k, pos, freq, q_out=q[:1].expand(4, 4, 64))
    refused("inference-only", q.clone().requires_grad_(), k, pos, freq)
    with torch.no_grad():
        normalize_rotate_qk(q.clone().requires_grad_(), k, pos, freq)

    kp, vp, _, _ = pools(2, 4, 2, 64, torch.bfloat16, "heads", False)
    k8, v8, s8, t8 = pools(2, 4, 2, 64, torch.bfloat16, "heads", True)
    slots = torch.arange(4, device="cuda")

    def no_append(match, *args, **options):
        with pytest.raises(ValueError, match=match):
            append_kv(*args, **options)

    no_append("identical shapes", k, k[:3], kp, vp, slots)
    no_append("one slot per token", k, k, kp, vp, slots[:3])
    no_append("int64", k, k, kp, vp, slots.int())
    no_append("same shape and dtype", k, k, kp, vp[:1], slots)
    no_append("need their scales", k, k, k8, v8, slots)
    no_append("only INT8", k, k, kp, vp, slots, k_scales=s8)
    no_append("float16", k, k, k8, v8, slots, k_scales=s8.float(), v_scales=t8)
    no_append("do not match", k.half(), k.half(), kp, vp, slots)
    no_append("kv_heads and head_dim", k[:, :1], k[:, :1], kp, vp, slots)
    with pytest.raises(ValueError, match="do not match"):
        read_kv(kp, vp, slots, dtype=torch.float16)
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        read_kv(k8, v8, slots, k_scales=s8, v_scales=t8, dtype=torch.float32)
    with pytest.raises(ValueError, match="needs a weight|both positions"):
        normalize_rotate_append(q, k, k, kp, vp, slots, pos)


def test_gradients_and_shared_memory_are_refused():
    k = torch.zeros((4, 2, 64), dtype=torch.bfloat16, device="cuda")
    freq, slots = rotary_frequencies(32), torch.arange(4, device="cuda")
    kp, vp, _, _ = pools(2, 4, 2, 64, torch.bfloat16, "heads", False)
    k8, v8, s8, t8 = pools(2, 4, 2, 64, torch.bfloat16, "heads", True)
    learned = freq.clone().requires_grad_()
    with pytest.raises(ValueError, match="inference-only"):
        normalize_rotate_qk(k, k, slots, learned)
    with torch.no_grad():
        normalize_rotate_qk(k, k, slots, learned)
    with pytest.raises(ValueError, match="inference-only"):
        append_kv(k, k, kp, vp.clone().requires_grad_(), slots)
    with pytest.raises(ValueError, match="inference-only"):
        read_kv(kp.detach().requires_grad_(), vp, slots)
    with pytest.raises(ValueError, match="inference-only"):
        read_kv(k8, v8, slots, k_scales=s8, v_scales=t8.detach().requires_grad_())
    with pytest.raises(ValueError, match="share memory"):
        append_kv(k, k, kp[:1].expand(2, 4, 2, 64), vp[:1].expand(2, 4, 2, 64), slots)
    with pytest.raises(ValueError, match="share memory"):
        append_kv(k, k, k8, v8, slots, k_scales=s8[..., :1].expand(2, 4, 2), v_scales=t8[..., :1].expand(2, 4, 2))
    read_kv(kp, kp, slots)
    read_kv(kp[:1].expand(2, 4, 2, 64), vp[:1].expand(2, 4, 2, 64), slots)


@pytest.mark.parametrize("dim,sections,pairing,dtype", [
    (128, (32,), "halves", torch.bfloat16),      # 16 elements of a lane
    (80, (20,), "halves", torch.float16),        # 8
    (96, (11, 6), "halves", torch.bfloat16),     # element by element
    (128, (32,), "adjacent", torch.bfloat16),    # 16
    (24, (5,), "adjacent", torch.float16),       # 8, an odd number of pairs: rotated and other pairs on one lane
])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan"), -0.0])
def test_elements_past_the_pairs_stay_as_they_are(dim, sections, pairing, dtype, bad):
    """Without a norm their bits go through, also next to infinities and NaN, into rows and into pages."""
    gen = torch.Generator().manual_seed(dim)
    turned = 2 * sum(sections)
    fused = rows(gen, dim, 6, dim, dtype=dtype)
    for t in range(turned, dim):  # token t has one such element in every head
        fused[t, :, t] = bad
    freq, pos = rotary_frequencies(sections, device="cpu"), torch.arange(len(sections) * dim).view(len(sections), dim)
    clean = torch.where(torch.isfinite(fused), fused, torch.zeros_like(fused))
    q, k, v = fused.cuda().split([3, 2, 1], dim=1)
    qo, ko = normalize_rotate_qk(q, k, pos.cuda(), freq.cuda(), sections=sections, pairing=pairing)
    cache = DeviceKVCache(dim // 8, 8, 2, dim, dtype=dtype)
    slots = torch.arange(dim, device="cuda")
    v2 = torch.cat([v, v], dim=1)
    q2 = cache.normalize_rotate_append(q, k, v2, slots, pos.cuda(), freq.cuda(), sections=sections, pairing=pairing)
    k2, v_back = cache.read(slots)
    for got, x in ((qo, fused[:, :3]), (q2, fused[:, :3]), (ko, fused[:, 3:5]), (k2, fused[:, 3:5])):
        past, want = got.cpu()[..., turned:], x[..., turned:]
        assert torch.equal(torch.isnan(past), torch.isnan(want))
        assert torch.equal(past.contiguous().view(torch.int16)[~torch.isnan(want)],
                           want.contiguous().view(torch.int16)[~torch.isnan(want)])
    for got, start, heads in ((qo, 0, 3), (ko, 3, 2)):
        ref, size = rotated(clean[:, start : start + heads].double(), pos, freq, sections, pairing)
        close(got[..., :turned], ref[..., :turned], size[..., :turned], dtype)
    assert torch.equal(torch.isnan(v_back), torch.isnan(v2))
    assert torch.equal(v_back.nan_to_num(7.0), v2.nan_to_num(7.0))


def test_outputs_that_are_every_other_head_of_an_odd_count():
    """Disjoint rows: the last head of a token ends where the next token starts."""
    gen = torch.Generator().manual_seed(15)
    q, k = rows(gen, 9, 8, 64, dtype=torch.bfloat16).cuda(), rows(gen, 9, 2, 64, dtype=torch.bfloat16).cuda()
    freq, pos = rotary_frequencies(32), torch.arange(9, device="cuda")
    want, _ = normalize_rotate_qk(q, k, pos, freq)
    buffer = torch.full((9, 15, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    normalize_rotate_qk(q, k, pos, freq, q_out=buffer[:, ::2])
    assert torch.equal(buffer[:, ::2], want) and bool((buffer[:, 1::2] == 5).all())
    # One head fewer to a token: its last row is the next token's first.
    shared = torch.empty(9 * 15 * 64, dtype=torch.bfloat16, device="cuda").as_strided((9, 8, 64), (14 * 64, 128, 1))
    with pytest.raises(ValueError, match="overlap"):
        normalize_rotate_qk(q, k, pos, freq, q_out=shared)


def test_written_pages_of_overlapping_strides_are_refused():
    k = torch.zeros((4, 2, 64), dtype=torch.bfloat16, device="cuda")
    slots = torch.arange(4, device="cuda")
    memory = torch.zeros((2, 4096), dtype=torch.bfloat16, device="cuda")
    for strides in ((256, 128, 64, 1), (512, 64, 64, 1), (512, 128, 32, 1)):
        kp, vp = (m.as_strided((2, 4, 2, 64), strides) for m in memory)
        with pytest.raises(ValueError, match="share memory"):
            append_kv(k, k, kp, vp, slots)
        read_kv(kp, vp, slots)
    k8, v8, _, _ = pools(2, 4, 2, 64, torch.bfloat16, "heads", True)
    ks, vs = (m.half().as_strided((2, 4, 2), (8, 1, 3)) for m in memory)
    with pytest.raises(ValueError, match="share memory"):
        append_kv(k, k, k8, v8, slots, k_scales=ks, v_scales=vs)
    # Heads of a buffer that others have the rest of.
    for strides in ((1024, 256, 128, 1), (1024, 64, 256, 1)):
        kp, vp = (m.as_strided((2, 4, 2, 64), strides) for m in memory)
        append_kv(k + 1, k + 2, kp, vp, slots)
        ko, vo = read_kv(kp, vp, slots)
        assert bool((ko == 1).all()) and bool((vo == 2).all())


def test_one_pool_as_k_and_v_is_refused_for_different_rows():
    k, v = (torch.full((4, 2, 64), x, dtype=torch.bfloat16, device="cuda") for x in (1.0, 2.0))
    freq, slots = rotary_frequencies(32), torch.arange(4, device="cuda")
    kp, vp, _, _ = pools(2, 4, 2, 64, torch.bfloat16, "heads", False)
    k8, v8, ks, vs = pools(2, 4, 2, 64, torch.bfloat16, "heads", True)
    both, wide = pools(3, 4, 2, 64, torch.bfloat16, "heads", False)[0], pools(2, 4, 4, 64, torch.bfloat16, "heads", False)[0]
    for call in (lambda: append_kv(k, v, kp, kp, slots), lambda: append_kv(k, v, both[:2], both[1:], slots),
                 lambda: append_kv(k, k, both[:2], both[1:], slots),
                 lambda: append_kv(k, v, k8, v8, slots, k_scales=ks, v_scales=ks),
                 lambda: append_kv(k, v, k8, k8, slots, k_scales=ks, v_scales=vs),
                 lambda: normalize_rotate_append(k, k, k, kp, kp, slots, slots, freq)):
        with pytest.raises(ValueError, match="share memory"):
            call()
    assert bool((both == 3).all()) and bool((kp == 3).all())
    # The same rows, and pools that are each other's neighbours.
    append_kv(k, k, kp, kp, slots)
    assert bool((kp[0] == 1).all()) and bool((kp[1] == 3).all())
    append_kv(k, v, wide[:, :, :2], wide[:, :, 2:], slots)
    assert bool((wide[0, :, :2] == 1).all()) and bool((wide[0, :, 2:] == 2).all()) and bool((wide[1] == 3).all())


def test_outputs_in_the_place_of_other_operands_are_refused():
    gen = torch.Generator().manual_seed(16)
    q, k, v = (rows(gen, 4, 4, 64, dtype=torch.bfloat16).cuda() for _ in range(3))
    freq, pos = rotary_frequencies(32), torch.arange(4, device="cuda")
    spare, held = torch.empty_like(q), q.clone()
    kp, vp, _, _ = pools(1, 4, 4, 64, torch.bfloat16, "heads", False)
    for outs in (dict(q_out=k), dict(k_out=q), dict(q_out=k, k_out=q), dict(q_out=spare, k_out=spare),
                 dict(q_out=q.transpose(0, 1))):
        with pytest.raises(ValueError, match="share memory"):
            normalize_rotate_qk(q, k, pos, freq, **outs)
    for out in (k, v):
        with pytest.raises(ValueError, match="share memory"):
            normalize_rotate_append(q, k, v, kp, vp, pos, pos, freq, q_out=out)
    assert torch.equal(q, held)
    want = normalize_rotate_qk(q, k, pos, freq)
    normalize_rotate_append(q, k, v, kp, vp, pos, pos, freq, q_out=spare)
    assert torch.equal(spare, want[0])
    normalize_rotate_qk(q, k, pos, freq, q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    # Nothing lies anywhere without tokens.
    normalize_rotate_qk(q[:0], k[:0], pos[:0], freq, q_out=q[:0], k_out=q[:0])


def test_outputs_that_require_gradients_are_refused():
    q = torch.ones((4, 4, 64), dtype=torch.bfloat16, device="cuda")
    freq, pos = rotary_frequencies(32), torch.arange(4, device="cuda")
    learned = torch.zeros_like(q).requires_grad_()
    kp, vp, _, _ = pools(1, 4, 4, 64, torch.bfloat16, "heads", False)
    table, n = torch.zeros((4, 1), dtype=torch.int32, device="cuda"), torch.ones(4, dtype=torch.int32, device="cuda")
    calls = (lambda: normalize_rotate_qk(q, q, pos, freq, q_out=learned),
             lambda: normalize_rotate_qk(q, q, pos, freq, k_out=learned),
             lambda: normalize_rotate_append(q, q, q, kp, vp, pos, pos, freq, q_out=learned),
             lambda: paged_decode_attention(q, kp, vp, table, n, out=learned))
    for call in calls:
        with pytest.raises(ValueError, match="inference-only"):
            call()
        assert bool((learned == 0).all())
        with torch.no_grad():
            call()
            assert not bool((learned == 0).all())
            learned.zero_()


@pytest.mark.parametrize("int8", [False, True])
def test_pools_past_32_bit_offsets_hold_k_and_v_apart(int8):
    """K in the first, V in the last heads of one buffer of more than 2^32 elements: rows written, read and attended."""
    pages, page, heads, dim = 32800, 64, 8, 128
    both, _, scales, _ = pools(pages, page, 2 * heads, dim, torch.bfloat16, "heads", int8)
    assert both.numel() > 2**32
    kp, vp = both[:, :, :heads], both[:, :, heads:]
    options = dict(k_scales=scales[:, :, :heads], v_scales=scales[:, :, heads:]) if int8 else {}
    gen = torch.Generator().manual_seed(17)
    k, v = (rows(gen, 130, heads, dim, dtype=torch.bfloat16) for _ in range(2))
    table = torch.tensor([[pages - 1, 2, pages - 2]], dtype=torch.int32)
    at = torch.arange(130)
    slots = (table[0, at // page].long() * page + at % page).cuda()
    append_kv(k.cuda(), v.cuda(), kp, vp, slots, **options)
    ko, vo = read_kv(kp, vp, slots, **options)
    near = DeviceKVCache(3, page, heads, dim, storage_dtype="int8" if int8 else None)
    near.append(k.cuda(), v.cuda(), at.cuda())
    want_k, want_v = near.read(at.cuda())
    assert torch.equal(ko, want_k) and torch.equal(vo, want_v)
    if not int8:
        assert torch.equal(ko.cpu(), k) and torch.equal(vo.cpu(), v)
    page_of, row = slots // page, slots % page
    assert torch.equal(both[page_of, row], torch.cat([near.k_pages, near.v_pages], dim=2)[at // page, at % page])
    # The rows around them hold what they held.
    assert bool((both[pages - 2, 2:] == 3).all()) and bool((both[1] == 3).all()) and bool((both[pages - 3] == 3).all())
    q = rows(gen, 1, 4 * heads, dim, dtype=torch.bfloat16).cuda()
    lengths = torch.tensor([130], dtype=torch.int32, device="cuda")
    got = paged_decode_attention(q, kp, vp, table.cuda(), lengths, **options)
    assert torch.equal(got, near.attend(q, torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda"), lengths))
    del both, kp, vp, scales, options
    torch.cuda.empty_cache()


def test_launches_of_more_than_2_to_the_23_tokens_go_in_parts():
    tokens, dim, page = 2**23 + 5, 16, 64
    gen = torch.Generator(device="cuda").manual_seed(18)
    q, k, v = (torch.randn((tokens, 1, dim), generator=gen, device="cuda").to(torch.bfloat16) for _ in range(3))
    freq, pos = rotary_frequencies(8), torch.arange(tokens, device="cuda")
    half = tokens // 2
    parts = [normalize_rotate_qk(q[i], k[i], pos[i], freq) for i in (slice(0, half), slice(half, tokens))]
    want_q, want_k = (torch.cat(x) for x in zip(*parts))
    del parts
    cache = DeviceKVCache(tokens // page + 1, page, 1, dim)
    got_q = cache.normalize_rotate_append(q, k, v, pos, pos, freq)
    assert torch.equal(got_q, want_q)
    ko, vo = cache.read(pos)
    assert torch.equal(ko, want_k) and torch.equal(vo, v)
    got_q, got_k = normalize_rotate_qk(q, k, pos, freq)
    assert torch.equal(got_q, want_q) and torch.equal(got_k, want_k)
    cache.append(v, k, pos)
    ko, vo = cache.read(pos)
    assert torch.equal(ko, v) and torch.equal(vo, k)
    last = cache.read(torch.arange(tokens, cache.num_pages * page, device="cuda"))
    assert all(bool((x == 0).all()) for x in last)
    del q, k, v, pos, want_q, want_k, cache, got_q, got_k, ko, vo
    torch.cuda.empty_cache()
