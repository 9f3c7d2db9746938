"""Windowed attention over a paged K/V cache and a cache in 8 bits with block scales, as measurable cases.

The kinds of case, each with the framework's entry points (``own``) and in
plain torch operations:

* ``prompt``: the attention of several new tokens per sequence over the pages
  of a cache that holds them already (``kernels.paged_prefill_attention``),
  causal, with or without a sliding window and first tokens that stay visible
  (sinks).
* ``token``: the same for one new token per sequence
  (``kernels.paged_decode_attention``).
* ``append_read``: K and V rows quantised into e4m3 pages with one
  power-of-two scale per block of tokens and K/V head, and read back
  (``kernels.append_kv_blocks``, ``kernels.read_kv``).
* ``step``: a decoding step's share of the cache: one token per sequence
  appended to e4m3 pages, its block read back, and the attention over them.

Pages hold the rows' type, INT8 values with a scale per row, or e4m3 values with
a scale per block.  Q, K, V are N(0, 1), as in the repository's tests and
benchmark; pages lie in the pool in random order.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
MOST_FLOPS = 7.0e12
MOST_BYTES = 2.2e9


def _case(kind, sequences, tokens, q_heads, kv_heads, head_dim, *, name=None, dtype="bf16", keys=0, ragged=False,
          page=64, block=64, stored="rows", window=0, sinks=0, layout="heads"):
    """``tokens`` new tokens and ``keys`` cached ones (the new ones among them) over all sequences; window 0: none."""
    case = dict(kind=kind, sequences=sequences, tokens=tokens, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim,
                dtype=dtype, keys=keys or tokens, ragged=ragged, page=page, block=min(block, page), stored=stored,
                window=window, sinks=sinks, layout=layout)
    if name is not None:
        case["name"] = name
    return case


def listed():
    return [
        # Five drafted tokens each of four sequences, checked in one pass: latency.
        _case("prompt", 4, 20, 32, 8, 128, name="prompt4x5_window1024", keys=8200, window=1024, sinks=4, ragged=True),
        # A packed ragged batch of prompts into an empty cache.
        _case("prompt", 7, 20011, 32, 8, 128, name="prompt_ragged7_20011_window4096", ragged=True, window=4096, sinks=4),
        # One long prompt at the projected pipeline's tokens, the headline's query heads.
        _case("prompt", 1, 61312, 56, 8, 128, name="prompt_61312x56_window4096", window=4096, sinks=16, page=256),
        # A prompt's chunk behind a long cached one, e4m3 pages, every key seen.
        _case("prompt", 1, 2000, 40, 8, 128, name="prompt2000_over_131072_e4m3", keys=131072, stored="e4m3"),
        # Wide heads, one query head per K/V head, pages laid out token by token, an odd window without sinks.
        _case("prompt", 3, 6007, 16, 16, 256, name="prompt3_6007_d256_fp16_window1000", dtype="fp16", ragged=True,
              page=32, window=1000, layout="tokens"),
        # Chunks of nine prompts behind INT8 pages.
        _case("prompt", 9, 2700, 12, 4, 64, name="prompt9x300_d64_int8_window2048", keys=36000, ragged=True,
              stored="int8", page=16, window=2048, sinks=1),
        # A serving batch whose tokens see a quarter of their sequences.
        _case("token", 64, 64, 32, 8, 128, name="token64_window4096", keys=1048576, window=4096, sinks=4),
        # Few short windows: latency.
        _case("token", 3, 3, 8, 8, 64, name="token3_d64_window512", keys=12000, page=16, window=512, sinks=4,
              ragged=True),
        # A serving batch over e4m3 pages.
        _case("token", 96, 96, 40, 8, 128, name="token96_1m_e4m3", keys=1048576, ragged=True, stored="e4m3"),
        # One long sequence over e4m3 pages, the headline's query heads.
        _case("token", 1, 1, 56, 8, 128, name="token1_524288_e4m3", keys=524288, stored="e4m3", page=256),
        # A packed ragged prefill into e4m3 pages and back.
        _case("append_read", 11, 20011, 8, 8, 128, name="append_read_e4m3_ragged11_20011x8", ragged=True, stored="e4m3"),
        # An attention layer's decoding step of 24 sequences.
        _case("step", 24, 24, 32, 8, 128, name="step24_e4m3_window4096", keys=192007, ragged=True, stored="e4m3",
              window=4096, sinks=4),
    ]


def _size(rng, low, high):
    """A size spread over the logarithm of [low, high], mostly odd ones."""
    n = int(round(low * (high / low) ** rng.random()))
    return max(low, n // 64 * 64) if rng.random() < 0.3 else n


def draw(rng: random.Random):
    """One more case of the listed kinds, with at most the largest listed one's work."""
    while True:
        kind = rng.choice(["prompt", "prompt", "prompt", "token", "token", "append_read", "step"])
        q_heads, kv_heads = rng.choice([(8, 8), (16, 16), (32, 8), (40, 8), (12, 4), (8, 2), (56, 8), (28, 4), (8, 1)])
        page = rng.choice([16, 32, 64, 128, 256])
        more = dict(dtype=rng.choice(["bf16", "bf16", "fp16"]), page=page, block=rng.choice([16, 32, 64, 64]),
                    layout=rng.choice(["heads", "heads", "tokens"]), ragged=rng.random() < 0.7,
                    stored="e4m3" if kind in ("append_read", "step") else rng.choice(["rows", "rows", "int8", "e4m3"]))
        if kind != "append_read" and rng.random() < 0.7:
            more.update(window=_size(rng, 16, 8192), sinks=rng.choice([0, 1, 4, 16, 64]))
        head_dim = rng.choice([64, 128, 128, 128, 80, 96, 256])
        sequences = _size(rng, 1, 16 if kind in ("prompt", "append_read") else 256)
        if kind in ("prompt", "append_read"):
            tokens = max(sequences, _size(rng, 1, 48_000))
            keys = tokens + (0 if rng.random() < 0.5 else _size(rng, sequences, sequences * 16_000))
        else:
            tokens = sequences
            keys = _size(rng, sequences * 16, sequences * 32_000)
        case = _case(kind, sequences, tokens, q_heads, kv_heads, head_dim, keys=keys, **more)
        cost = work(case)
        pool = case["keys"] * 4 * kv_heads * head_dim
        if cost["flops"] <= MOST_FLOPS and cost["bytes"] <= MOST_BYTES and pool <= 4 * MOST_BYTES:
            return case


def _split(total, parts, ragged):
    """Lengths of `parts` sequences that add up to `total`; ragged ones are the same for every seed."""
    if total < parts:
        return [1] * total + [0] * (parts - total)
    if not ragged:
        return [total // parts + (1 if i < total % parts else 0) for i in range(parts)]
    rng = random.Random(parts)
    weights = [rng.uniform(0.2, 1.8) for _ in range(parts)]
    lengths = [max(1, int(total * w / sum(weights))) for w in weights]
    while sum(lengths) > total:
        lengths[lengths.index(max(lengths))] -= 1
    lengths[-1] += total - sum(lengths)
    return lengths


def _sequences(case):
    """New tokens and keys of every sequence."""
    if case["kind"] in ("token", "step"):
        return [1] * case["sequences"], _split(case["keys"], case["sequences"], case["ragged"])
    new = _split(case["tokens"], case["sequences"], case["ragged"])
    before = _split(case["keys"] - case["tokens"], case["sequences"], case["ragged"])
    return new, [a + b for a, b in zip(new, before)]


def _normal(gen, shape, dtype):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    rows = max(1, (1 << 27) // max(1, math.prod(shape[1:])))
    for start in range(0, shape[0], rows):  # in pieces: few temporaries
        piece = out[start : start + rows]
        piece.copy_(torch.randn(piece.shape, generator=gen, device="cuda"))
    return out


def _pools(case, gen, pages):
    """K and V pages [pages, page, kv_heads, head_dim] (memory head by head in each page, or token by token) and their
    scales: INT8 float16 [pages, page, kv_heads], e4m3 E8M0 [pages, page / block, kv_heads]."""
    heads, page, dim = case["kv_heads"], case["page"], case["head_dim"]
    by_head = case["layout"] == "heads"
    shape = (pages, heads, page, dim) if by_head else (pages, page, heads, dim)
    view = (lambda t: t.transpose(1, 2)) if by_head else (lambda t: t)
    pools = {}
    for name in ("k", "v"):
        scales = None
        if case["stored"] == "int8":
            values = torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda", generator=gen)
            steps = (2.0 + 2.0 * torch.rand(shape[:3], generator=gen, device="cuda")) / 127.0
            scales = view(steps.to(torch.float16))
        elif case["stored"] == "e4m3":
            # Blocks of N(0, 1) have their largest magnitudes near 4, and scales
            # of 2^-6 (2^-7 where they end below 3.5).
            values = torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda")
            rows = max(1, (1 << 27) // math.prod(shape[1:]))
            for start in range(0, pages, rows):
                piece = values[start : start + rows]
                x = torch.randn(piece.shape, generator=gen, device="cuda").mul_(100.0).clamp_(-448.0, 448.0)
                piece.copy_(x.to(torch.float8_e4m3fn))
            scale_shape = (pages, heads, page // case["block"]) if by_head else (pages, page // case["block"], heads)
            exponents = torch.randint(120, 122, scale_shape, dtype=torch.uint8, device="cuda", generator=gen)
            scales = view(exponents).view(torch.float8_e8m0fnu)
        else:
            values = _normal(gen, shape, DTYPES[case["dtype"]])
        pools[name + "_pages"], pools[name + "_scales"] = view(values), scales
    return pools


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, page, block = DTYPES[case["dtype"]], case["page"], case["block"]
    kind, sequences, heads, dim = case["kind"], case["sequences"], case["kv_heads"], case["head_dim"]
    new, lengths = _sequences(case)
    state = dict(kind=kind, dtype=dtype, page=page, block=block, q_heads=case["q_heads"], kv_heads=heads, head_dim=dim,
                 scale=dim**-0.5, window=case["window"] or None, sinks=case["sinks"], new=new, keys=lengths)
    if kind != "append_read":
        state["q"] = _normal(gen, (case["tokens"], case["q_heads"], dim), dtype)
    if kind in ("append_read", "step"):
        # K and V of a token are next to each other, as a projection leaves them.
        fused = _normal(gen, (case["tokens"], 2 * heads, dim), dtype)
        state["k"], state["v"] = fused.split([heads, heads], dim=1)
    counts = [-(-n // page) for n in lengths]
    total = sum(counts)
    state.update(_pools(case, gen, total + total // 10 + 1))
    order = torch.randperm(state["k_pages"].shape[0], generator=gen, device="cuda")[:total].to(torch.int32)
    table = torch.full((sequences, max(counts)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(counts):
        table[s, :n] = order[at : at + n]
        at += n
    state["page_table"] = table
    state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, *new]).cumsum(0)
    state["cu_tokens"] = cu.to(torch.int32).cuda()
    if kind in ("append_read", "step"):
        where = torch.repeat_interleave(torch.arange(sequences), torch.tensor(new)).cuda()
        at = torch.cat([torch.arange(n - m, n) for m, n in zip(new, lengths)]).cuda()
        state["new_slots"] = state["slots"] = table[where, at // page].long() * page + at % page
        if kind == "step":
            # The rows of the new token's block up to it, -1 behind it.
            rows = torch.arange(block, device="cuda")[None] + (at // block * block)[:, None]
            page_of = torch.gather(table, 1, rows // page).long()
            state["slots"] = torch.where(rows <= at[:, None], page_of * page + rows % page, -1).flatten()
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
    pools = s["k_pages"], s["v_pages"]
    scales = dict(k_scales=s["k_scales"], v_scales=s["v_scales"])
    visible = dict(softmax_scale=s["scale"], window=s["window"], sinks=s["sinks"], return_lse=True)
    if s["kind"] == "prompt":
        return kernels.paged_prefill_attention(s["q"], *pools, s["page_table"], s["lengths"], s["cu_tokens"], **scales,
                                               **visible)
    results = ()
    if s["kind"] in ("append_read", "step"):
        one_each = s["kind"] == "step"
        kernels.append_kv_blocks(s["k"], s["v"], *pools, s["k_scales"], s["v_scales"], s["page_table"], s["lengths"],
                                 None if one_each else s["cu_tokens"])
        results = kernels.read_kv(*pools, s["slots"], dtype=s["dtype"], **scales)
    if s["kind"] in ("token", "step"):
        results = (*kernels.paged_decode_attention(s["q"], *pools, s["page_table"], s["lengths"], **scales, **visible),
                   *results)
    return results


# ---- the plain forms ----------------------------------------------------------


def _plain_power(e):
    """2^e in float64, by its bits: a power that is off by its last bit moves values off their ties."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _plain_rows(s, name, slots):
    """The float32 values of the pages' rows at ``slots``, [..., kv_heads, head_dim]."""
    pages, scales = s[name + "_pages"], s[name + "_scales"]
    page, row = slots // s["page"], slots % s["page"]
    if scales is None:
        return pages[page, row].float()
    if pages.dtype == torch.int8:
        return pages[page, row].float() * scales[page, row].float()[..., None]
    values = pages.view(torch.uint8)[page, row].view(torch.float8_e4m3fn).float()
    exponents = scales.view(torch.uint8)[page, row // s["block"]].to(torch.int32) - 127
    return values * _plain_power(exponents).float()[..., None]


def _plain_softmax(logits, visible, v):
    """Weights of the visible logits times v, and the LSE."""
    logits = torch.where(visible, logits, -math.inf)
    top = logits.amax(dim=-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    weights = torch.exp(logits - top)
    total = weights.sum(dim=-1, keepdim=True)
    return torch.matmul(weights, v) / torch.where(total > 0, total, 1.0), (top + torch.log(total))[..., 0]


def _plain_prompt(s):
    q_heads, kv_heads, dim = s["q_heads"], s["kv_heads"], s["head_dim"]
    group = q_heads // kv_heads
    out = torch.empty_like(s["q"])
    lse = torch.empty((q_heads, len(s["q"])), dtype=torch.float32, device=out.device)
    done = 0
    for index, (new, length) in enumerate(zip(s["new"], s["keys"])):
        positions = torch.arange(length, device=out.device)
        slots = s["page_table"][index].long()[positions // s["page"]] * s["page"] + positions % s["page"]
        span = length if s["window"] is None else min(length, s["window"] + s["sinks"])
        step = max(1, min(new, 512, (1 << 28) // (q_heads * span)))
        k, v = (_plain_rows(s, name, slots).transpose(0, 1).contiguous() for name in ("k", "v"))
        for start in range(0, new, step):
            stop = min(new, start + step)
            first, last = length - new + start, length - new + stop - 1  # positions
            at = positions[: last + 1]
            if s["window"] is not None:
                low = max(0, first - s["window"] + 1)
                at = torch.cat([positions[: min(s["sinks"], low)], positions[low : last + 1]])
            p = torch.arange(first, last + 1, device=out.device)[:, None]
            visible = at <= p
            if s["window"] is not None:
                visible &= (at > p - s["window"]) | (at < s["sinks"])
            rows = s["q"][done + start : done + stop].float() * s["scale"]
            rows = rows.view(-1, kv_heads, group, dim).permute(1, 2, 0, 3).reshape(kv_heads, -1, dim)
            logits = torch.matmul(rows, k[:, at].transpose(1, 2)).view(kv_heads, group, stop - start, -1)
            o, l = _plain_softmax(logits, visible, v[:, at][:, None])
            out[done + start : done + stop] = o.permute(2, 0, 1, 3).reshape(-1, q_heads, dim).to(out.dtype)
            lse[:, done + start : done + stop] = l.reshape(q_heads, -1)
        done += new
    return out, lse


def _plain_token(s):
    q, lengths = s["q"], s["lengths"].long()[:, None]
    sequences, q_heads, dim = q.shape
    kv_heads, group = s["kv_heads"], q_heads // s["kv_heads"]
    longest = max(s["keys"])
    if s["window"] is None:
        at = torch.arange(longest, device=q.device)[None].expand(sequences, -1)
        visible = at < lengths
    else:
        first = torch.arange(min(s["sinks"], longest), device=q.device)[None].expand(sequences, -1)
        low = (lengths - s["window"]).clamp(min=0)
        recent = low + torch.arange(min(s["window"], longest), device=q.device)
        at = torch.cat([first, recent], dim=1)
        visible = torch.cat([first < low, recent < lengths], dim=1)  # every key once
    held = torch.where(visible, at, 0)
    slots = torch.gather(s["page_table"].long(), 1, held // s["page"]) * s["page"] + held % s["page"]
    out = torch.empty_like(q)
    lse = torch.empty((q_heads, sequences), dtype=torch.float32, device=q.device)
    step = max(1, (1 << 30) // (at.shape[1] * kv_heads * dim))
    for i in range(0, sequences, step):
        k, v = (_plain_rows(s, name, slots[i : i + step]).permute(0, 2, 1, 3) for name in ("k", "v"))
        rows = q[i : i + step].float().view(-1, kv_heads, group, dim) * s["scale"]
        o, l = _plain_softmax(torch.matmul(rows, k.transpose(2, 3)), visible[i : i + step, None, None], v)
        out[i : i + step] = o.reshape(-1, q_heads, dim).to(q.dtype)
        lse[:, i : i + step] = l.reshape(-1, q_heads).t()
    return out, lse


def _plain_exponents(amax):
    """E8M0 bytes of the smallest power of two, at least 2^-126, of which 448 reach amax."""
    mantissa, e = torch.frexp(amax)  # amax = mantissa 2^e, 0.5 <= mantissa < 1, and 448 = 0.875 * 2^9
    e = torch.where(mantissa > 0.875, e - 8, e - 9)
    return torch.where(amax > 0, e, -126).clamp(-126, 127) + 127


def _plain_append(s, name):
    rows, block, per_page = s[name].float(), s["block"], s["page"] // s["block"]
    pages, scales = s[name + "_pages"].view(torch.uint8), s[name + "_scales"].view(torch.uint8)
    slots = s["new_slots"]
    page, row = slots // s["page"], slots % s["page"]
    blocks = page * per_page + row // block
    touched, which = torch.unique(blocks, return_inverse=True)
    need = torch.zeros((len(touched), s["kv_heads"]), dtype=torch.int32, device=rows.device)
    need.scatter_reduce_(0, which[:, None].expand(-1, s["kv_heads"]), _plain_exponents(rows.abs().amax(-1)), "amax")
    first = torch.full_like(touched, block).scatter_reduce_(0, which, row % block, "amin")
    t_page, t_block = touched // per_page, touched % per_page
    old = scales[t_page, t_block].to(torch.int32)
    e = torch.where((first > 0)[:, None], torch.maximum(old, need), need)
    # The rows before the new ones, in the new scale.
    at = t_block[:, None] * block + torch.arange(block, device=rows.device)
    kept = pages[t_page[:, None], at].view(torch.float8_e4m3fn).float()
    again = (kept * _plain_power(old - e)[:, None, :, None]).float().to(torch.float8_e4m3fn).view(torch.uint8)
    before = (torch.arange(block, device=rows.device) < first[:, None])[..., None, None]
    pages[t_page[:, None], at] = torch.where(before, again, pages[t_page[:, None], at])
    codes = (rows * _plain_power(127 - e[which])[..., None]).float().to(torch.float8_e4m3fn)
    pages[page, row] = codes.view(torch.uint8)
    scales[t_page, t_block] = e.to(torch.uint8)


def run(s):
    if own:
        return _run_own(s)
    if s["kind"] == "prompt":
        return _plain_prompt(s)
    results = ()
    if s["kind"] in ("append_read", "step"):
        _plain_append(s, "k")
        _plain_append(s, "v")
        slots = s["slots"]
        held = (slots >= 0)[:, None, None]
        results = tuple(torch.where(held, _plain_rows(s, name, slots.clamp(min=0)), 0.0).to(s["dtype"])
                        for name in ("k", "v"))
    if s["kind"] in ("token", "step"):
        results = (*_plain_token(s), *results)
    return results


def work(case):
    new, lengths = _sequences(case)
    window, sinks = case["window"], case["sinks"]
    pairs = seen = 0
    for n, length in zip(new, lengths):
        for last in (length, length - n):  # keys seen by the tokens at positions below `last`, added and taken off
            sign = 1 if last == length else -1
            if window and last > window:
                far = last - window  # positions from `window` on: the window, and sinks that have left it
                some = window * (window + 1) // 2 + far * window
                some += sinks * far - sinks * (sinks - 1) // 2 if far >= sinks else far * (far + 1) // 2
            else:
                some = last * (last + 1) // 2
            pairs += sign * some
        low = max(0, length - n - window + 1) if window else 0
        seen += length - low + min(sinks, low)
    heads, dim = case["kv_heads"], case["head_dim"]
    q_row, kv_row = 2 * case["q_heads"] * dim, 2 * heads * dim  # bytes of 16-bit rows
    stored = {"rows": kv_row, "int8": heads * (dim + 2), "e4m3": heads * (dim + 1 / case["block"])}[case["stored"]]
    nbytes = flops = 0
    if case["kind"] in ("append_read", "step"):
        back = case["tokens"] if case["kind"] == "append_read" else sum((n - 1) % case["block"] + 1 for n in lengths)
        nbytes += case["tokens"] * 2 * (kv_row + stored) + back * 2 * (stored + kv_row)
        flops += (case["tokens"] + back) * 4 * heads * dim
    if case["kind"] != "append_read":
        nbytes += seen * 2 * stored + case["tokens"] * (2 * q_row + 4 * case["q_heads"]) + seen // case["page"] * 4
        flops += 4 * pairs * case["q_heads"] * dim
    return {"bytes": int(nbytes), "flops": flops}


# ---- from the definitions, in 64 bits ------------------------------------------


def _exact_powers(device):
    """The values of the 255 E8M0 scales."""
    return torch.tensor([2.0 ** (n - 127) for n in range(255)], dtype=torch.float64, device=device)


def _exact_values(case, s, name, index):
    """All of one sequence's rows in the pages, [keys, kv_heads, head_dim] in 64 bits."""
    length = s["keys"][index]
    found = s["page_table"][index, : -(-length // case["page"])].long()
    x = s[name + "_pages"]
    if case["stored"] == "e4m3":
        x = x.view(torch.uint8)[found].view(torch.float8_e4m3fn).double()
        power = _exact_powers(x.device)[s[name + "_scales"].view(torch.uint8)[found].long()]
        x = x * power.repeat_interleave(case["block"], 1)[..., None]
    elif case["stored"] == "int8":
        x = x[found].double() * s[name + "_scales"][found].double()[..., None]
    else:
        x = x[found].double()
    return x.flatten(0, 1)[:length]


def _exact_attention(case, s, values):
    """``values(name, index)``: one sequence's rows in 64 bits."""
    group, window, sinks = case["q_heads"] // case["kv_heads"], case["window"], case["sinks"]
    outs, lses, done = [], [], 0
    for index, (n, length) in enumerate(zip(s["new"], s["keys"])):
        k, v = values("k", index), values("v", index)
        for start in range(0, n, 1024):
            count = min(1024, n - start)
            position = torch.arange(count, device=k.device) + (length - n + start)
            key = torch.arange(int(length - n + start) + count, device=k.device)
            if window:
                key = key[(key < sinks) | (key > length - n + start - window)]
            mask = key[None] <= position[:, None]
            if window:
                mask = mask & ((key[None] < sinks) | (position[:, None] - key[None] < window))
            q = s["q"][done + start : done + start + count].double()
            heads, sums = [], []
            for h in range(case["q_heads"]):
                logits = (q[:, h] @ k[key, h // group].t()) / math.sqrt(case["head_dim"])
                logits = logits.masked_fill(~mask, -math.inf)
                heads.append(torch.softmax(logits, -1) @ v[key, h // group])
                sums.append(torch.logsumexp(logits, -1))
            outs.append(torch.stack(heads, 1))
            lses.append(torch.stack(sums))
        done += n
    return torch.cat(outs), torch.cat(lses, 1)


def _exact_e4m3(x):
    """To the nearest e4m3 value, ties to even: 3 bits behind the first one, steps of 2^-9 below 2^-6."""
    binade = torch.frexp(x.abs()).exponent.clamp(min=-5).long()  # |x| in [2^(binade - 1), 2^binade)
    step = torch.tensor([2.0 ** (n - 9) for n in range(300)], dtype=torch.float64, device=x.device)[binade + 5]
    return torch.round(x / step) * step


def _exact_append(case, s, name):
    """Every sequence's rows after the append, in 64 bits."""
    whole, done = [], 0
    for index, (n, length) in enumerate(zip(s["new"], s["keys"])):
        rows = _exact_values(case, s, name, index)
        fresh, start = s[name][done : done + n].double(), length - n
        done += n
        for low in range(start // case["block"] * case["block"], length, case["block"]):
            high = min(length, low + case["block"])
            begin = max(low, start)
            top = fresh[begin - start : high - start].abs().amax((0, 2))  # [kv_heads]
            power = torch.exp2(torch.ceil(torch.log2((top / 448).clamp(min=2.0**-126))))
            if begin > low:
                at = s["page_table"][index, low // case["page"]].long()
                held = s[name + "_scales"].view(torch.uint8)[at, low % case["page"] // case["block"]].long()
                power = torch.maximum(power, _exact_powers(at.device)[held])
                rows[low:begin] = _exact_e4m3(rows[low:begin] / power[:, None]) * power[:, None]
            rows[begin:high] = _exact_e4m3(fresh[begin - start : high - start] / power[:, None]) * power[:, None]
        whole.append(rows)
    return whole


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("prompt", "token"):
        return _exact_attention(case, s, lambda name, index: _exact_values(case, s, name, index))
    stored = {name: _exact_append(case, s, name) for name in ("k", "v")}
    back = []
    for name in ("k", "v"):
        if case["kind"] == "append_read":
            back.append(torch.cat([rows[length - n :] for rows, n, length in zip(stored[name], s["new"], s["keys"])]))
        else:
            last = torch.zeros((case["sequences"], case["block"], case["kv_heads"], case["head_dim"]),
                               dtype=torch.float64, device="cuda")
            for index, length in enumerate(s["keys"]):
                low = (length - 1) // case["block"] * case["block"]
                last[index, : length - low] = stored[name][index][low:]
            back.append(last.flatten(0, 1))
    if case["kind"] == "append_read":
        return tuple(back)
    return (*_exact_attention(case, s, lambda name, index: stored[name][index]), *back)
