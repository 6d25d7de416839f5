"""Rotary positions of queries and keys with their gradient, and the frequencies of checkpoints made for long contexts.

``apply_rotary`` is one kernel for queries and keys of any lengths, layouts and positions; ``rotary_plan`` gives the table of
frequencies and the scale that a configuration's ``rope_parameters`` call for.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import ops

LAYOUTS = {"half": 0, "pairs": 1}


class _Rotary(torch.autograd.Function):
    """The gradient of a turn is the turn back, with the same scale; its gradient in turn is the turn itself."""

    @staticmethod
    def forward(ctx, q, k, positions, freq, layout, inverse, scale):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions, freq)
        ctx.how = layout, inverse, scale
        return ops.rotary(q, k, positions, freq, layout, inverse, scale)

    @staticmethod
    def backward(ctx, dq, dk):
        if dq is None and dk is None:
            return (None,) * 7
        positions, freq = ctx.saved_tensors
        layout, inverse, scale = ctx.how
        turn = _Rotary.apply if torch.is_grad_enabled() else ops.rotary
        dq, dk = turn(dq, dk, positions, freq, layout, not inverse, scale)
        return dq, dk, None, None, None, None, None


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, freq: torch.Tensor, *, layout: str = "half",
                 scale: float = 1.0) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``q [B, Hq, S, D]`` and ``k [B, Hkv, S, D]`` (or None) turned by their positions, as new tensors of the same type.

    ``positions``: int32 or int64, ``[B, S]``, ``[1, S]`` or ``[S]``.  ``freq``: fp32 ``[pairs, 2]``, every frequency (radians per
    position) as a high and a low part; the first ``2 * pairs`` elements of a head turn and are multiplied by ``scale``, the others are
    copied.  ``layout``: ``"half"`` turns element i with ``pairs + i``, ``"pairs"`` element 2i with 2i + 1.  Angles are exact to fp32 at
    any position, and a result is rounded once.  Any strides; the results are stored token by token (``[B, S, H, D]`` in memory).
    Differentiable in q and k."""
    how = LAYOUTS.get(layout)
    if how is None:
        raise ValueError(f"layout {layout!r}: one of {sorted(LAYOUTS)}")
    shape = q.shape
    if len(shape) != 4 or (k is not None and (k.dim() != 4 or k.shape[0] != shape[0] or k.shape[2:] != shape[2:])):
        raise ValueError(f"queries {tuple(shape)} and keys {None if k is None else tuple(k.shape)}: want [B, H, S, D] of one batch, length and head size")
    b, _, s, d = shape
    dtype, device = q.dtype, q.device
    ops.dtype_code(dtype)
    if k is not None and (k.dtype != dtype or k.device != device):
        raise TypeError(f"queries {dtype} on {device}, keys {k.dtype} on {k.device}")
    if positions.dtype != torch.int64 and positions.dtype != torch.int32:
        raise TypeError(f"positions of {positions.dtype}: want int32 or int64")
    at = positions.shape
    if len(at) not in (1, 2) or at[-1] != s or (len(at) == 2 and at[0] != 1 and at[0] != b):
        raise ValueError(f"positions {tuple(at)} for {b} x {s} tokens")
    pairs = freq.shape
    if len(pairs) != 2 or pairs[1] != 2 or freq.dtype != torch.float32 or not freq.is_contiguous() or 2 * pairs[0] > d:
        raise ValueError(f"frequencies {freq.dtype} {tuple(pairs)}: want contiguous fp32 [pairs, 2] with at most {d // 2} pairs")
    if positions.device != device or freq.device != device:
        raise ValueError(f"queries on {device}, positions on {positions.device}, frequencies on {freq.device}")
    if (q.requires_grad or (k is not None and k.requires_grad)) and torch.is_grad_enabled():
        return _Rotary.apply(q, k, positions, freq, how, False, float(scale))
    return ops.rotary(q, k, positions, freq, how, False, float(scale))


__all__ = ["LAYOUTS", "apply_rotary"]
