"""e4m3 pages with power-of-two block scales, from their definition, on the CPU in 64 bits."""

from __future__ import annotations

import math

import torch

# Every e4m3 value of a byte, from the format: sign, 4 bits of exponent (bias 7), 3 of mantissa, all ones NaN.
VALUES = torch.tensor([
    (-1.0) ** (b >> 7) * (math.nan if b & 127 == 127 else
                          (b & 7) * 2.0**-9 if b & 120 == 0 else (8 + (b & 7)) * 2.0 ** ((b >> 3 & 15) - 10))
    for b in range(256)], dtype=torch.float64)
POWERS = torch.tensor([2.0 ** (b - 127) for b in range(255)] + [math.nan], dtype=torch.float64)


def rounded(x):
    """To the nearest e4m3 value, ties to even (|x| <= 448); what is not finite to NaN."""
    step = torch.full_like(x, 2.0**-9)
    for n in range(-6, 9):
        step[x.abs() >= 2.0**n] = 2.0 ** (n - 3)
    return torch.where(torch.isfinite(x), torch.round(x / step) * step, math.nan)


def power_for(x):
    """The smallest 2^e, e >= -126, of which 448 reach every finite |x|."""
    x = x[torch.isfinite(x)].abs()
    top = float(x.max()) if x.numel() else 0.0
    e = -126
    while 448 * 2.0**e < top:
        e += 1
    return 2.0**e


def values(pages, scales):
    """What e4m3 pages and their scales (CPU) stand for, in 64 bits."""
    block = pages.shape[1] // scales.shape[1]
    power = POWERS[scales.view(torch.uint8).long()].repeat_interleave(block, 1)
    return VALUES[pages.view(torch.uint8).long()] * power[..., None]


def appended(pages, scales, rows, table, lengths, cu):
    """``values`` and the scales' powers after an append, from those before: 64-bit tensors, changed in place."""
    per_page = pages.shape[1]
    block = per_page // scales.shape[1]
    room = table.shape[1] * per_page
    for s in range(table.shape[0]):
        start, stop = int(cu[s]), int(cu[s + 1])
        by_block = {}
        for t in range(start, stop):
            position = int(lengths[s]) - (stop - t)
            if 0 <= position < room:
                by_block.setdefault(position // block, []).append((position, t))
        for index, members in by_block.items():
            page = int(table[s, index * block // per_page])
            if not 0 <= page < pages.shape[0]:
                continue
            low, at = index * block % per_page, index * block % per_page // block
            before = members[0][0] - index * block
            for h in range(pages.shape[2]):
                new = rows[[t for _, t in members], h].double()
                power = power_for(new)
                if before:
                    power = max(power, float(scales[page, at, h]))
                    kept = slice(low, low + before)
                    pages[page, kept, h] = rounded(pages[page, kept, h] / power) * power
                first = members[0][0] % per_page
                pages[page, first : first + len(members), h] = rounded(new / power) * power
                # Rows behind the new ones are no sequence's: their codes stay, whatever they stand for now.
                pages[page, first + len(members) : low + block, h] *= power / scales[page, at, h]
                scales[page, at, h] = power
