"""The operators around a device-resident K/V cache, as measurable cases.

The kinds of case, each with the framework's entry points (``own``) and in
plain torch operations:

* ``rotate``: the norm of every head of Q and K and the rotation by their
  positions, on the output of a QKV projection
  (``kernels.normalize_rotate_qk``).
* ``append``: the same with K and V written to the pages of a cache, a prefill
  (``kernels.normalize_rotate_append``).
* ``append_read``: K and V rows written to the pages and read back as packed
  rows (``kernels.append_kv``, ``kernels.read_kv``): a prompt that goes into
  the cache and from there to a runner that continues it.
* ``decode``: the attention of one new token per sequence over the pages
  (``kernels.paged_decode_attention``).
* ``step``: an attention layer's share of a decoding step, norm, rotation and
  append, then the attention that reads what was appended.

Q, K, V are N(0, 1) and the norms' weights near 1, as in the repository's tests
and benchmark; pages lie in the pool in random order.
"""

from __future__ import annotations

import itertools
import math
import random
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6
BASE = 10000.0


def _case(kind, sequences, tokens, q_heads, kv_heads, head_dim, *, name=None, dtype="bf16", keys=0, ragged=False,
          page=64, int8=False, axes=1, pairing="halves", partial=False, layout="heads"):
    """``tokens`` rows of Q (and of new K, V); ``keys`` tokens in the cache over all sequences."""
    case = dict(kind=kind, sequences=sequences, tokens=tokens, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim,
                dtype=dtype, keys=keys, ragged=ragged, page=page, int8=int8, axes=axes, pairing=pairing,
                partial=partial, layout=layout)
    if name is not None:
        case["name"] = name
    return case


def listed():
    return [
        # A token of each of 48 sequences: latency.
        _case("rotate", 48, 48, 32, 8, 128, name="rotate_decode48_gqa"),
        # The projected pipeline's tokens and heads, a video's three axes.
        _case("rotate", 1, 61312, 56, 56, 128, name="rotate_61312x56_3axes", axes=3),
        # Adjacent pairs over half of an odd head size.
        _case("rotate", 1, 8190, 16, 16, 80, name="rotate_8190x16_d80_adjacent_fp16", dtype="fp16",
              pairing="adjacent", partial=True),
        # A packed ragged prefill into the cache.
        _case("append", 11, 20011, 32, 8, 128, name="append_ragged11_20011_gqa", ragged=True),
        # A prompt into INT8 pages and back.
        _case("append_read", 1, 16384, 56, 8, 128, name="append_read_int8_16384x8", int8=True, page=256),
        # An attention layer's decoding step of 24 sequences, 8,000 keys on
        # average.
        _case("step", 24, 24, 32, 8, 128, name="step24_gqa", keys=192007, ragged=True),
        # One short sequence, 8 heads of 64: the smallest attention, latency.
        _case("decode", 1, 1, 8, 8, 64, name="decode1_4096x8_d64", keys=4096, page=16),
        # One long sequence, the headline's 56 query heads: all of the split
        # is over its length.
        _case("decode", 1, 1, 56, 8, 128, name="decode1_524288_gqa", keys=524288, page=256),
        # A serving batch over INT8 pages.
        _case("decode", 96, 96, 40, 8, 128, name="decode96_int8_gqa", keys=1048576, ragged=True, int8=True),
        # Wide heads, one query head per K/V head, pages laid out token by
        # token.
        _case("decode", 7, 7, 16, 16, 256, name="decode7_mha_d256_fp16", dtype="fp16", keys=57330, ragged=True,
              page=32, layout="tokens"),
        # Few heads, short and long sequences.
        _case("decode", 200, 200, 12, 4, 96, name="decode200_short_d96", keys=60013, ragged=True, page=16),
        # The largest batch.
        _case("decode", 64, 64, 32, 8, 128, name="decode64_1m_gqa", keys=1048576),
    ]


def _size(rng, low, high):
    """A size spread over the logarithm of [low, high], mostly odd ones."""
    n = int(round(low * (high / low) ** rng.random()))
    return max(low, n // 64 * 64) if rng.random() < 0.3 else n


def draw(rng: random.Random):
    """One more case of the listed kinds, with at most the largest listed one's work."""
    kind = rng.choice(["rotate", "append", "append_read", "step", "decode", "decode", "decode"])
    q_heads, kv_heads = rng.choice([(8, 8), (16, 16), (32, 32), (32, 8), (40, 8), (12, 4), (8, 2), (56, 8), (28, 4),
                                    (8, 1)])
    more = dict(dtype=rng.choice(["bf16", "bf16", "fp16"]), page=rng.choice([16, 32, 64, 128, 256]),
                int8=rng.random() < 0.3 and kind in ("append_read", "step", "decode"), axes=rng.choice([1, 1, 2, 3]),
                pairing=rng.choice(["halves", "halves", "adjacent"]), partial=rng.random() < 0.25,
                layout=rng.choice(["heads", "heads", "tokens"]), ragged=rng.random() < 0.7)
    head_dim = rng.choice([64, 128, 128, 128, 80, 96, 256])
    if kind in ("rotate", "append", "append_read"):
        sequences = rng.randint(1, 16)
        tokens = max(sequences, _size(rng, 1, 32_000))
        return _case(kind, sequences, tokens, q_heads, kv_heads, head_dim, **more)
    sequences = _size(rng, 1, 256)
    keys = max(sequences, _size(rng, sequences * 16, min(sequences * 32_000, 8_000_000 // (kv_heads * head_dim // 128 + 1))))
    if kind == "step":
        # The appended pages come back whole, INT8 ones as their values: 16-bit
        # pages here.
        more["int8"] = False
    return _case(kind, sequences, sequences, q_heads, kv_heads, head_dim, keys=keys, **more)


def _split(total, parts, ragged):
    """Lengths of `parts` sequences that add up to `total`; ragged ones are the same for every seed."""
    if not ragged:
        return [total // parts + (1 if i < total % parts else 0) for i in range(parts)]
    rng = random.Random(parts)
    weights = [rng.uniform(0.2, 1.8) for _ in range(parts)]
    lengths = [max(1, int(total * w / sum(weights))) for w in weights]
    while sum(lengths) > total:
        lengths[lengths.index(max(lengths))] -= 1
    lengths[-1] += total - sum(lengths)
    return lengths


def _pairs(case):
    """Rotated pairs of a head."""
    return case["head_dim"] // (4 if case["partial"] else 2)


def _sections(case):
    pairs = _pairs(case)
    if case["axes"] == 1:
        return (pairs,)
    if case["axes"] == 2:
        return (pairs // 2, pairs - pairs // 2)
    side = 3 * pairs // 8
    return (pairs - 2 * side, side, side)


def _normal(gen, shape, dtype):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    rows = max(1, (1 << 27) // max(1, math.prod(shape[1:])))
    for start in range(0, shape[0], rows):  # in pieces: few temporaries
        piece = out[start : start + rows]
        piece.copy_(torch.randn(piece.shape, generator=gen, device="cuda"))
    return out


def _pools(case, gen, pages):
    """K and V pages [pages, page, kv_heads, head_dim] (memory head by head in each page, or token by token) and
    their INT8 scales [pages, page, kv_heads]."""
    heads, page, dim = case["kv_heads"], case["page"], case["head_dim"]
    by_head = case["layout"] == "heads"
    shape = (pages, heads, page, dim) if by_head else (pages, page, heads, dim)
    view = (lambda t: t.transpose(1, 2)) if by_head else (lambda t: t)
    pools = {}
    for name in ("k", "v"):
        if case["int8"]:
            pools[name + "_pages"] = view(torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda", generator=gen))
            steps = (2.0 + 2.0 * torch.rand(shape[:3], generator=gen, device="cuda")) / 127.0
            pools[name + "_scales"] = view(steps.to(torch.float16))
        else:
            pools[name + "_pages"] = view(_normal(gen, shape, DTYPES[case["dtype"]]))
            pools[name + "_scales"] = None
    return pools


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    kind, heads, dim, page = case["kind"], case["kv_heads"], case["head_dim"], case["page"]
    tokens, sequences = case["tokens"], case["sequences"]
    state = dict(kind=kind, dtype=dtype, page=page, q_heads=case["q_heads"], kv_heads=heads, head_dim=dim,
                 scale=dim**-0.5)
    if kind == "decode":
        state["q"] = _normal(gen, (tokens, case["q_heads"], dim), dtype)
    else:
        # Q, K and V of a token are one row of the projection's output.
        fused = _normal(gen, (tokens, case["q_heads"] + 2 * heads, dim), dtype)
        state["q"], state["k"], state["v"] = fused.split([case["q_heads"], heads, heads], dim=1)
    if kind in ("rotate", "append", "step"):
        sections = _sections(case)
        state["sections"], state["pairing"] = sections, case["pairing"]
        # Every axis has the frequencies of its own pairs.
        state["frequencies"] = torch.cat([
            BASE ** (-torch.arange(n, dtype=torch.float64, device="cuda") / n) for n in sections])
        state["axis"] = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], device="cuda")
        state["q_weight"] = (1 + 0.1 * torch.randn(dim, generator=gen, device="cuda")).to(dtype)
        state["k_weight"] = (1 + 0.1 * torch.randn(dim, generator=gen, device="cuda")).to(dtype)
    if kind in ("decode", "step"):
        lengths = _split(case["keys"], sequences, case["ragged"])
    elif kind in ("append", "append_read"):
        lengths = _split(tokens, sequences, case["ragged"])
    if kind == "step":
        positions = torch.tensor([n - 1 for n in lengths], device="cuda")
    elif kind == "append":
        positions = torch.cat([torch.arange(n, device="cuda") for n in lengths])
    else:
        # A stretch of a long sequence.
        positions = torch.arange(tokens, device="cuda") + int(torch.randint(0, 1_000_000, (1,), generator=gen, device="cuda"))
    if kind in ("rotate", "append", "step"):
        if case["axes"] == 1:
            state["positions"] = positions
        else:  # frames of rows of 40 patches, 24 rows each
            grid = [positions // 960, positions // 40 % 24, positions % 40]
            state["positions"] = torch.stack(grid if case["axes"] == 3 else grid[1:])
    if kind != "rotate":
        counts = [-(-n // page) for n in lengths]
        total = sum(counts)
        state.update(_pools(case, gen, total + total // 10 + 1))
        order = torch.randperm(state["k_pages"].shape[0], generator=gen, device="cuda")[:total].to(torch.int32)
        table = torch.full((sequences, max(counts)), -1, dtype=torch.int32, device="cuda")
        for s, (first, n) in enumerate(zip(itertools.accumulate([0, *counts]), counts)):
            table[s, :n] = order[first : first + n]
        state["page_table"] = table
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        if kind == "step":
            where, at = torch.arange(sequences, device="cuda"), positions
        else:
            where = torch.repeat_interleave(torch.arange(sequences, device="cuda"), state["lengths"])
            at = torch.cat([torch.arange(n, device="cuda") for n in lengths])
        state["slots"] = table[where, at // page].long() * page + at % page
    return state


# ---- the framework's entry points -------------------------------------------


def _kernels():
    package = str(Path(__file__).resolve().parents[1] / "stream-attn_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import seqattn.kernels

    return seqattn.kernels


def _run_own(s):
    kernels = _kernels()
    rotation = {name: s[name] for name in ("sections", "pairing", "q_weight", "k_weight") if name in s}
    if s["kind"] == "rotate":
        return kernels.normalize_rotate_qk(s["q"], s["k"], s["positions"], s["frequencies"], eps=EPS, **rotation)
    pools = s["k_pages"], s["v_pages"]
    scales = dict(k_scales=s["k_scales"], v_scales=s["v_scales"])
    if s["kind"] == "append_read":
        kernels.append_kv(s["k"], s["v"], *pools, s["slots"], **scales)
        return kernels.read_kv(*pools, s["slots"], dtype=s["dtype"], **scales)
    q, results = s["q"], ()
    if s["kind"] in ("append", "step"):
        q = kernels.normalize_rotate_append(q, s["k"], s["v"], *pools, s["slots"], s["positions"], s["frequencies"],
                                            eps=EPS, **scales, **rotation)
        results = (q, *pools)
    if s["kind"] in ("decode", "step"):
        results = (*kernels.paged_decode_attention(q, *pools, s["page_table"], s["lengths"], softmax_scale=s["scale"],
                                                   return_lse=True, **scales), *results)
    return results


# ---- the plain forms ----------------------------------------------------------


def _plain_rotate(x, weight, s):
    """[tokens, heads, head_dim] in float32: normalized, weighted and rotated."""
    y = x.float()
    y = y * torch.rsqrt(y.square().mean(dim=-1, keepdim=True) + EPS) * weight.float()
    positions = s["positions"].view(-1, x.shape[0])
    angles = positions[s["axis"]].t().double() * s["frequencies"]  # [tokens, pairs]
    cos, sin = angles.cos().float()[:, None, :], angles.sin().float()[:, None, :]
    pairs = angles.shape[1]
    if s["pairing"] == "halves":
        a, b = y[..., :pairs], y[..., pairs : 2 * pairs]
    else:
        a, b = y[..., 0 : 2 * pairs : 2], y[..., 1 : 2 * pairs : 2]
    turned = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat(turned, dim=-1) if s["pairing"] == "halves" else torch.stack(turned, dim=-1).flatten(-2)
    return torch.cat([turned, y[..., 2 * pairs :]], dim=-1)


def _plain_store(rows, pages, scales, slots):
    """float32 rows [tokens, heads, head_dim] into the pages."""
    page, offset = slots // pages.shape[1], slots % pages.shape[1]
    if scales is None:
        pages[page, offset] = rows.to(pages.dtype)
        return
    step = rows.abs().amax(dim=-1) / 127.0
    step = torch.where(step > 0, step, torch.ones_like(step))
    pages[page, offset] = torch.round(rows / step[..., None]).clamp_(-127, 127).to(torch.int8)
    scales[page, offset] = step.to(torch.float16)


def _plain_values(pages, scales, index):
    """The float32 values that the pages hold at an index."""
    values = pages[index].float()
    return values if scales is None else values * scales[index].float()[..., None]


def _plain_attention(q, s):
    sequences, q_heads, dim = q.shape
    kv_heads, group = s["kv_heads"], q_heads // s["kv_heads"]
    table = s["page_table"].long().clamp(min=0)
    keys = table.shape[1] * s["page"]
    seen = torch.arange(keys, device=q.device) < s["lengths"][:, None]  # [sequences, keys]

    def rows(name):  # [sequences, kv_heads, keys, head_dim]
        x = _plain_values(s[name + "_pages"], s[name + "_scales"], table)
        return x.permute(0, 3, 1, 2, 4).reshape(sequences, kv_heads, keys, dim)

    logits = torch.matmul(q.float().view(sequences, kv_heads, group, dim) * s["scale"], rows("k").transpose(2, 3))
    logits = torch.where(seen[:, None, None, :], logits, -math.inf)
    top = logits.amax(dim=-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    weights = torch.exp(logits - top)
    total = weights.sum(dim=-1, keepdim=True)
    v = torch.where(seen[:, None, :, None], rows("v"), 0.0)
    out = torch.matmul(weights, v) / torch.where(total > 0, total, 1.0)
    lse = (top + torch.log(total)).view(sequences, q_heads).t().contiguous()
    return out.view(sequences, q_heads, dim).to(q.dtype), lse


def run(s):
    if own:
        return _run_own(s)
    if s["kind"] == "rotate":
        return tuple(_plain_rotate(s[x], s[x + "_weight"], s).to(s["dtype"]) for x in ("q", "k"))
    if s["kind"] == "append_read":
        _plain_store(s["k"].float(), s["k_pages"], s["k_scales"], s["slots"])
        _plain_store(s["v"].float(), s["v_pages"], s["v_scales"], s["slots"])
        index = s["slots"] // s["page"], s["slots"] % s["page"]
        return tuple(_plain_values(s[x + "_pages"], s[x + "_scales"], index).to(s["dtype"]) for x in ("k", "v"))
    q, results = s["q"], ()
    if s["kind"] in ("append", "step"):
        q = _plain_rotate(q, s["q_weight"], s).to(s["dtype"])
        _plain_store(_plain_rotate(s["k"], s["k_weight"], s), s["k_pages"], s["k_scales"], s["slots"])
        _plain_store(s["v"].float(), s["v_pages"], s["v_scales"], s["slots"])
        results = (q, s["k_pages"], s["v_pages"])
    if s["kind"] in ("decode", "step"):
        results = (*_plain_attention(q, s), *results)
    return results


def work(case):
    tokens, dim, page = case["tokens"], case["head_dim"], case["page"]
    q_row, kv_row = 2 * case["q_heads"] * dim, 2 * case["kv_heads"] * dim  # bytes of 16-bit rows
    stored = case["kv_heads"] * (dim + 2) if case["int8"] else kv_row  # a row of K or V in its page
    nbytes = flops = 0
    if case["kind"] in ("rotate", "append", "step"):
        # Q and K in and Q out; K to its own tensor or its page; the positions.
        nbytes += tokens * (2 * q_row + kv_row + 8 * case["axes"])
        nbytes += tokens * (kv_row if case["kind"] == "rotate" else stored)
        flops += tokens * (case["q_heads"] + case["kv_heads"]) * 8 * dim
    if case["kind"] in ("append", "step"):
        nbytes += tokens * (kv_row + stored + 8)
    if case["kind"] == "append_read":
        nbytes += tokens * (2 * kv_row + 4 * stored + 2 * kv_row + 16)
        flops += tokens * case["kv_heads"] * dim * 8
    if case["kind"] in ("decode", "step"):
        # Every key's K and V, Q in and out, the LSE, the lengths and pages.
        nbytes += case["keys"] * 2 * stored + tokens * (2 * q_row + 4 * case["q_heads"] + 4) + case["keys"] // page * 4
        flops += 4 * case["keys"] * case["q_heads"] * dim
    return {"bytes": nbytes, "flops": flops}


# ---- from the definitions, in 64 bits ------------------------------------------


def _exact_rotate(case, x, weight, positions):
    y = x.double()
    y = weight.double() * y / torch.sqrt((y * y).sum(-1, keepdim=True) / y.shape[-1] + EPS)
    out = y.clone()
    positions = positions.double().reshape(case["axes"], -1)
    pair = 0
    for axis, count in enumerate(_sections(case)):
        for j in range(count):
            angle = positions[axis] * BASE ** (-j / count)
            lo, hi = (pair, pair + _pairs(case)) if case["pairing"] == "halves" else (2 * pair, 2 * pair + 1)
            # One complex number per head, turned by the angle.
            z = torch.complex(y[..., lo], y[..., hi]) * torch.polar(torch.ones_like(angle), angle)[:, None]
            out[..., lo], out[..., hi] = z.real, z.imag
            pair += 1
    return out


def _exact_int8(rows):
    step = rows.abs().amax(-1, keepdim=True) / 127
    step[step == 0] = 1
    return torch.clamp(torch.round(rows / step), -127, 127) * step.half().double()


def _exact_attention(case, s, q, pages):
    """``pages(x, s)``: the values [keys, kv_heads, head_dim] of one sequence, in 64 bits."""
    outs, lses = [], []
    group = case["q_heads"] // case["kv_heads"]
    for index, length in enumerate(s["lengths"].tolist()):
        k, v = (pages(name, index)[:length] for name in ("k", "v"))
        heads = []
        for h in range(case["kv_heads"]):
            logits = q[index, h * group : (h + 1) * group] @ k[:, h].t() * case["head_dim"] ** -0.5
            heads.append((torch.softmax(logits, -1) @ v[:, h], torch.logsumexp(logits, -1)))
        outs.append(torch.cat([o for o, _ in heads]))
        lses.append(torch.cat([l for _, l in heads]))
    return torch.stack(outs), torch.stack(lses, dim=1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append_read":
        return tuple(_exact_int8(s[x].double()) if case["int8"] else s[x].double() for x in ("k", "v"))
    q, results, stored = s["q"].double(), (), {}
    if case["kind"] != "decode":
        q, k = (_exact_rotate(case, s[x], s[x + "_weight"], s["positions"]) for x in ("q", "k"))
        if case["kind"] == "rotate":
            return q, k
        whole = []
        for name, rows in (("k", k), ("v", s["v"].double())):
            pool = s[name + "_pages"].double()
            flat = pool.reshape(-1, *pool.shape[2:])
            flat[s["slots"]] = rows
            whole.append(flat.reshape(pool.shape))
            s[name + "_pages"] = whole[-1].to(s["dtype"])  # what the attention then finds there
        results = (q, *whole)
        q = q.to(s["dtype"]).double()
    if case["kind"] in ("decode", "step"):
        def pages(name, index):
            found = s["page_table"][index]
            found = found[found >= 0].long()
            x = s[name + "_pages"][found].double()
            if case["int8"]:
                x = x * s[name + "_scales"][found].double()[..., None]
            return x.flatten(0, 1)

        results = (*_exact_attention(case, s, q, pages), *results)
    return results
