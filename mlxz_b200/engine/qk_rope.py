"""What a layer does to its queries and keys before the cache: the norm of each
head and the rotation by position, with the layer's weights.

The steps of this package take one ``QKNormRope`` for all layers or one per
layer and run it ahead of the attention (``ops.qk_norm_rope``), in the prefill
step together with the append (``ops.qk_norm_rope_append``): the model's q_norm,
k_norm and rope calls and the cache update behind them, which the reference runs
inside the model (src/mlxz/engine/continuous.py:625-633).
"""
from __future__ import annotations

from collections.abc import Sequence
from dataclasses import dataclass

import torch

from .. import ops


@dataclass(slots=True)
class QKNormRope:
    """Arguments of ``ops.qk_norm_rope`` that belong to a layer."""

    inv_freq: torch.Tensor
    q_weight: torch.Tensor | None = None
    k_weight: torch.Tensor | None = None
    eps: float | None = None
    weight_offset: float = 0.0
    interleaved: bool = False
    freq_axes: torch.Tensor | None = None

    def _args(self, positions: torch.Tensor) -> dict:
        return dict(q_weight=self.q_weight, k_weight=self.k_weight, eps=self.eps,
                    weight_offset=self.weight_offset, interleaved=self.interleaved,
                    # text alone has one position, the same on every axis
                    freq_axes=None if positions.dim() == 1 else self.freq_axes)

    def apply(self, q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor
              ) -> tuple[torch.Tensor, torch.Tensor]:
        return ops.qk_norm_rope(q, k, positions, self.inv_freq, **self._args(positions))

    def apply_append(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                     positions: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                     slots: torch.Tensor) -> torch.Tensor:
        return ops.qk_norm_rope_append(q, k, v, positions, self.inv_freq, k_pool, v_pool, slots,
                                       **self._args(positions))


def per_layer(rope: "QKNormRope | Sequence[QKNormRope] | None", n_layers: int
              ) -> "list[QKNormRope | None]":
    """One entry per layer."""
    if rope is None or isinstance(rope, QKNormRope):
        return [rope] * n_layers
    rope = list(rope)
    if len(rope) != n_layers:
        raise ValueError(f"rope must be one QKNormRope or one per layer ({n_layers})")
    return rope
