"""The row and decoding operators in 64 bits, on the CPU, from their definitions."""

from __future__ import annotations

import math

import torch

HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def normalized(x, weight, eps):
    x = x.double()
    if weight is None:
        return x
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()


def pair_indices(pairs, pairing):
    i = torch.arange(pairs)
    return (i, i + pairs) if pairing == "halves" else (2 * i, 2 * i + 1)


def rotated(y, positions, frequencies, sections, pairing):
    """(rows, size of each element's pair): ``positions`` [axes, tokens] ints, exact angles in turns by integers."""
    size = y.abs().clone()
    if frequencies is None:
        return y, size
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections))
    angles = positions[axis].t().double() * frequencies  # [tokens, pairs]
    lo, hi = pair_indices(len(frequencies), pairing)
    a, b = y[..., lo], y[..., hi]
    cos, sin = angles.cos()[:, None], angles.sin()[:, None]
    out = y.clone()
    out[..., lo], out[..., hi] = a * cos - b * sin, b * cos + a * sin
    size[..., lo] = size[..., hi] = torch.sqrt(a * a + b * b)
    return out, size


def quantized(rows):
    """(codes, float16 scales, steps) of the INT8 storage format with one token per group."""
    step = rows.abs().amax(-1) / 127
    step = torch.where(step > 0, step, torch.ones_like(step))
    return torch.round(rows / step[..., None]).clamp(-127, 127), step.half(), step


def attention(q, k_pages, v_pages, table, lengths, scale, k_scales=None, v_scales=None):
    """(out, lse, sum of weight * |v|, largest sum of |q k| * scale): pools as held, all on the CPU."""
    sequences, q_heads, dim = q.shape
    pages, page_tokens, kv_heads, _ = k_pages.shape
    group = q_heads // kv_heads
    out = torch.zeros(q.shape, dtype=torch.float64)
    size = torch.zeros_like(out)
    lse = torch.full((q_heads, sequences), -math.inf, dtype=torch.float64)
    products = 0.0
    for s in range(sequences):
        length = max(0, min(int(lengths[s]), table.shape[1] * page_tokens))
        keys = [(int(table[s, j // page_tokens]), j % page_tokens) for j in range(length)]
        keys = [(p, r) for p, r in keys if 0 <= p < pages]
        if not keys:
            continue
        p, r = (torch.tensor(x) for x in zip(*keys))
        k, v = k_pages[p, r].double(), v_pages[p, r].double()
        if k_scales is not None:
            k, v = k * k_scales[p, r].double()[..., None], v * v_scales[p, r].double()[..., None]
        for h in range(q_heads):
            x = q[s, h].double()
            logits = k[:, h // group] @ x * scale
            products = max(products, float((k[:, h // group].abs() @ x.abs()).max()) * abs(scale))
            if torch.isneginf(logits).all():
                continue
            lse[h, s] = torch.logsumexp(logits, 0)
            w = torch.softmax(logits, 0)
            out[s, h] = w @ v[:, h // group]
            size[s, h] = w @ v[:, h // group].abs()
    return out, lse, size, products
