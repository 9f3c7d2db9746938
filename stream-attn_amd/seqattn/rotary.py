"""Frequencies of rotary positions (no counterpart in the reference)."""

from __future__ import annotations

import math
from collections.abc import Sequence

import torch


def rotary_frequencies(
    sections: int | Sequence[int],
    *,
    base: float = 10000.0,
    shared: bool = False,
    device: torch.device | str = "cuda",
) -> torch.Tensor:
    """Radians per position of each rotated pair, float64 ``[sum(sections)]``.

    ``sections`` counts the pairs of each position axis (an int: one axis, of
    ``head_dim // 2`` pairs where the whole head is rotated).  By default every
    axis has its own ladder, ``base ** (-j / n)`` for pair ``j`` of its ``n``;
    with ``shared`` the axes divide one ladder over all pairs among them.
    """
    counts = (sections,) if isinstance(sections, int) else tuple(sections)
    if not counts or any(not isinstance(n, int) or n < 1 for n in counts):
        raise ValueError("sections must be positive pair counts")
    if not (math.isfinite(base) and base > 0):
        raise ValueError("base must be finite and positive")
    ladders = (sum(counts),) if shared else counts
    steps = torch.cat([torch.arange(n, dtype=torch.float64) / n for n in ladders])
    return torch.pow(torch.tensor(base, dtype=torch.float64), -steps).to(device)


__all__ = ["rotary_frequencies"]
