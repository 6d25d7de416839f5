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
    """The gradient of a turn is the turn back, with the same scale."""

    @staticmethod
    def forward(ctx, q, k, positions, freq, layout, scale):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions, freq)
        ctx.how = layout, scale
        q2, k2 = ops.rotary(q, k, positions, freq, layout, False, scale)
        return q2 if k2 is None else (q2, k2)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk=None):
        if dq is None and dk is None:
            return (None,) * 6
        positions, freq = ctx.saved_tensors
        layout, scale = ctx.how
        dq, dk = ops.rotary(dq, dk, positions, freq, layout, True, scale)
        return dq, dk, None, None, None, None


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, freq: torch.Tensor, *, layout: str = "half",
                 scale: float = 1.0) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``q [B, Hq, S, D]`` and ``k [B, Hkv, S, D]`` (or None) turned by their positions, as new tensors of the same type.

    ``positions``: int32 or int64, ``[B, S]``, ``[1, S]`` or ``[S]``.  ``freq``: fp32 ``[pairs, 2]``, every frequency (radians per
    position) as a high and a low part; the first ``2 * pairs`` elements of a head turn and are multiplied by ``scale``, the others are
    copied.  ``layout``: ``"half"`` turns element i with ``pairs + i``, ``"pairs"`` element 2i with 2i + 1.  Angles are exact to fp32 at
    any position, and a result is rounded once.  Any strides; the results are stored token by token (``[B, S, H, D]`` in memory).
    Differentiable in q and k."""
    if layout not in LAYOUTS:
        raise ValueError(f"layout {layout!r}: one of {sorted(LAYOUTS)}")
    if q.dim() != 4 or (k is not None and (k.dim() != 4 or k.shape[0] != q.shape[0] or k.shape[2:] != q.shape[2:])):
        raise ValueError(f"queries {tuple(q.shape)} and keys {None if k is None else tuple(k.shape)}: want [B, H, S, D] of one batch, length and head size")
    ops.dtype_code(q.dtype)
    if k is not None and (k.dtype != q.dtype or k.device != q.device):
        raise TypeError(f"queries {q.dtype} on {q.device}, keys {k.dtype} on {k.device}")
    b, _, s, d = q.shape
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"positions of {positions.dtype}: want int32 or int64")
    if positions.dim() == 1:
        positions = positions[None]
    if positions.dim() != 2 or positions.shape[1] != s or positions.shape[0] not in (1, b):
        raise ValueError(f"positions {tuple(positions.shape)} for {b} x {s} tokens")
    if freq.dim() != 2 or freq.shape[1] != 2 or freq.dtype != torch.float32 or not freq.is_contiguous() or 2 * freq.shape[0] > d:
        raise ValueError(f"frequencies {freq.dtype} {tuple(freq.shape)}: want contiguous fp32 [pairs, 2] with at most {d // 2} pairs")
    if positions.device != q.device or freq.device != q.device:
        raise ValueError(f"queries on {q.device}, positions on {positions.device}, frequencies on {freq.device}")
    positions = positions.expand(b, s)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        out = _Rotary.apply(q, k, positions, freq, LAYOUTS[layout], float(scale))
        return (out, None) if k is None else out
    return tuple(ops.rotary(q, k, positions, freq, LAYOUTS[layout], False, scale))


__all__ = ["LAYOUTS", "apply_rotary"]
