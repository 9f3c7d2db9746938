"""Callback types of the projected pipeline (reference
src/seqattn_core/projection/types.py:1-12).

``QKVProjector(hidden_tile, start, stop) -> (q, k, v)``: maps a device tile
``[tokens, hidden_features]`` of rows ``start:stop`` to device tensors
``[tokens, q_heads, head_dim]`` and ``[tokens, kv_heads, head_dim]`` (x2).

``OutputProjector(attention_tile, start, stop) -> projected``: maps a
finalized attention tile ``[tokens, q_heads * head_dim]`` in HBM to the
device rows written into ``out[start:stop]``.
"""

from __future__ import annotations

from collections.abc import Callable, Sequence
from dataclasses import dataclass

import torch

from ..kernels.rows import normalize_rotate_qk

QKVProjector = Callable[[torch.Tensor, int, int], tuple[torch.Tensor, torch.Tensor, torch.Tensor]]
OutputProjector = Callable[[torch.Tensor, int, int], torch.Tensor]


@dataclass(frozen=True, eq=False)  # by identity: tensors have no truth value of their equality
class QKRotation:
    """Norm and rotation of the projected Q and K (no counterpart in the reference).

    The fields are the arguments of :func:`seqattn.kernels.normalize_rotate_qk`,
    for all tokens of the call: ``positions`` is ``[tokens]`` or ``[axes, tokens]``
    on the planned device.  The pipeline applies it to each projected tile; with
    Q/K/V resident in HBM in the pass that moves the tile to its place.
    """

    positions: torch.Tensor | None = None
    frequencies: torch.Tensor | None = None
    sections: Sequence[int] | None = None
    pairing: str = "halves"
    q_weight: torch.Tensor | None = None
    k_weight: torch.Tensor | None = None
    eps: float = 1e-6

    def validate(self, tokens: int) -> None:
        if self.positions is not None and (self.positions.ndim not in (1, 2) or self.positions.shape[-1] != tokens):
            raise ValueError("qk_rotation positions must be [tokens] or [axes, tokens] of the whole call")

    def apply(self, q, k, start: int, stop: int, *, q_out=None, k_out=None) -> tuple[torch.Tensor, torch.Tensor]:
        """Rows ``start:stop`` of the call."""
        positions = None if self.positions is None else self.positions[..., start:stop]
        return normalize_rotate_qk(
            q, k, positions, self.frequencies, sections=self.sections, pairing=self.pairing,
            q_weight=self.q_weight, k_weight=self.k_weight, eps=self.eps, q_out=q_out, k_out=k_out,
        )


__all__ = ["OutputProjector", "QKRotation", "QKVProjector"]
