"""Rotary positions of queries and keys with their gradient, and the frequencies of checkpoints made for long contexts.

``apply_rotary`` is one kernel for queries and keys of any lengths, layouts and positions; ``RotaryPlan`` gives the frequencies and the
scale that a configuration's ``rope_parameters`` call for.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import ops

LAYOUTS = {"half": 0, "pairs": 1}


class _Rotary(torch.autograd.Function):
    """The gradient of a turn is the turn back, with the same scale; its gradient in turn is the turn itself.  A turn is linear: tangents are
    turned like what they belong to."""

    @staticmethod
    def forward(ctx, q, k, positions, freq, layout, inverse, scale):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions, freq)
        ctx.save_for_forward(positions, freq)
        ctx.how = layout, inverse, scale
        ctx.shapes = tuple(None if t is None else t.shape for t in (q, k))
        return ops.rotary(q, k, positions, freq, layout, inverse, scale)

    @staticmethod
    def jvp(ctx, *tangents):
        positions, freq = ctx.saved_tensors
        turn, given = _Rotary.apply if torch.is_grad_enabled() else ops.rotary, tangents[0] if tangents[0] is not None else tangents[1]
        turned = turn(*tangents[:2], positions, freq, *ctx.how)
        # where only one of the two has a tangent, the other's is zero (an output's may not be left out)
        return tuple(given.new_zeros(shape) if out is None and shape is not None else out for out, shape in zip(turned, ctx.shapes))

    @staticmethod
    def backward(ctx, dq, dk):
        if dq is None and dk is None:
            return (None,) * 7
        positions, freq = ctx.saved_tensors
        layout, inverse, scale = ctx.how
        turn = _Rotary.apply if torch.is_grad_enabled() else ops.rotary
        dq, dk = turn(dq, dk, positions, freq, layout, not inverse, scale)
        return dq, dk, None, None, None, None, None


def _has_tangent(t: torch.Tensor) -> bool:
    return forward_ad.unpack_dual(t).tangent is not None


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, freq: torch.Tensor, *, layout: str = "half",
                 scale: float = 1.0) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``q [B, Hq, S, D]`` and ``k [B, Hkv, S, D]`` (or None) turned by their positions, as new tensors of the same type.

    ``positions``: int32 or int64, ``[B, S]``, ``[1, S]`` or ``[S]``.  ``freq``: fp32 ``[pairs, 2]``, every frequency (radians per
    position) as a high and a low part; the first ``2 * pairs`` elements of a head turn and are multiplied by ``scale``, the others are
    copied.  ``layout``: ``"half"`` turns element i with ``pairs + i``, ``"pairs"`` element 2i with 2i + 1.  Angles are exact to fp32 at
    any position, and a result is rounded once.  Any strides; the results are stored token by token (``[B, S, H, D]`` in memory).
    Differentiable in q and k, in either mode."""
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
    if ((q.requires_grad or (k is not None and k.requires_grad)) and torch.is_grad_enabled()) or _has_tangent(q) or (k is not None and _has_tangent(k)):
        return _Rotary.apply(q, k, positions, freq, how, False, float(scale))
    return ops.rotary(q, k, positions, freq, how, False, float(scale))


def split_frequencies(f: torch.Tensor) -> torch.Tensor:
    """Frequencies in 64 bits as ``apply_rotary`` takes them: ``[pairs, 2]``, a high and a low part in fp32."""
    hi = f.float()
    return torch.stack([hi, (f - hi.double()).float()], dim=-1).contiguous()


class RotaryPlan:
    """Frequencies of the rotary positions of a head's first ``dims`` elements: ``base^(-2i / dims)``, changed as ``parameters["rope_type"]``
    says (the keys are those of transformers' ``rope_parameters``):

    * ``default``: as they are;
    * ``linear``: divided by ``factor``;
    * ``llama3``: waves longer than ``original_max_position_embeddings / low_freq_factor`` divided by ``factor``, shorter ones than
      ``.. / high_freq_factor`` kept, those between mixed in proportion;
    * ``yarn``: a ramp over the pairs between those that turn ``beta_fast`` and ``beta_slow`` times in the original length, kept on one side,
      divided by ``factor`` on the other; queries and keys scaled by ``attention_factor`` (default ``0.1 ln(factor) + 1``, or the quotient of
      that with ``mscale`` and ``mscale_all_dim``);
    * ``longrope``: divided by ``short_factor`` or, where the sequence is longer than the original length, ``long_factor`` (a number per
      pair); scaled by ``attention_factor`` (default ``sqrt(1 + ln(factor) / ln(original))``);
    * ``dynamic``: for sequences longer than ``max_positions`` the base grows with the length (``original_max_position_embeddings`` counts
      only where ``max_positions`` is not given, as in transformers).

    ``on(device, positions)`` is the table and the scale; where it depends on the length, that is the largest position plus one, and it is
    chosen on the device (recordable in a CUDA graph)."""

    KINDS = ("default", "linear", "llama3", "yarn", "longrope", "dynamic")

    def __init__(self, dims: int, base: float, parameters: Optional[dict] = None, max_positions: Optional[int] = None):
        p = dict(parameters or {})
        self.kind = p.get("rope_type", p.get("type", "default")) or "default"
        if self.kind not in self.KINDS:
            raise NotImplementedError(f"rope_type={self.kind!r}: one of {self.KINDS}")
        if dims < 0 or dims % 2:
            raise ValueError(f"{dims} rotary dims")
        self.dims, self.base, self.scale = dims, float(base), 1.0
        need = {"linear": ("factor",), "llama3": ("factor", "low_freq_factor", "high_freq_factor"), "yarn": ("factor",),
                "longrope": ("short_factor", "long_factor"), "dynamic": ("factor",)}.get(self.kind, ())
        missing = [k for k in need if p.get(k) is None]
        if missing:
            raise ValueError(f"rope_type={self.kind!r} without {missing}")
        self.original = p.get("original_max_position_embeddings") or max_positions
        if self.kind == "dynamic":
            self.original = max_positions or self.original
        if self.kind in ("llama3", "yarn", "longrope", "dynamic") and not self.original:
            raise ValueError(f"rope_type={self.kind!r} without original_max_position_embeddings")
        # On the CPU whatever the default device is: checkpoints are loaded into models that were built on "meta", where tables have no values.
        f = self.base ** (-torch.arange(0, dims, 2, dtype=torch.float64, device="cpu") / max(dims, 1))
        self.factor = float(p.get("factor") or 1.0)
        self._tables = [getattr(self, f"_{self.kind}")(f, p, max_positions)]
        if self.kind == "longrope":
            self._tables = list(self._tables[0])
        self._held = {}

    def _default(self, f, p, max_positions):
        return f

    def _linear(self, f, p, max_positions):
        return f / self.factor

    def _dynamic(self, f, p, max_positions):
        return f

    def _llama3(self, f, p, max_positions):
        lo, hi = float(p["low_freq_factor"]), float(p["high_freq_factor"])
        turns = self.original * f / (2 * math.pi)                      # of a pair in the original length
        mix = (turns - lo) / (hi - lo)
        mixed = (1 - mix) * f / self.factor + mix * f
        return torch.where(turns < lo, f / self.factor, torch.where(turns > hi, f, mixed))

    def _yarn(self, f, p, max_positions):
        factor = self.factor

        def magnitude(m=1.0):
            return 0.1 * m * math.log(factor) + 1.0 if factor > 1 else 1.0
        given = p.get("attention_factor")
        if given is not None:
            self.scale = float(given)
        elif p.get("mscale") and p.get("mscale_all_dim"):
            self.scale = magnitude(p["mscale"]) / magnitude(p["mscale_all_dim"])
        else:
            self.scale = magnitude()

        def pair_of(turns):                                            # the pair that turns this often in the original length
            return self.dims * math.log(self.original / (turns * 2 * math.pi)) / (2 * math.log(self.base))
        lo, hi = pair_of(float(p.get("beta_fast") or 32.0)), pair_of(float(p.get("beta_slow") or 1.0))
        if p.get("truncate", True):
            lo, hi = math.floor(lo), math.ceil(hi)
        lo, hi = max(lo, 0), min(hi, self.dims - 1)
        ramp = ((torch.arange(self.dims // 2, dtype=torch.float64, device="cpu") - lo) / ((hi - lo) or 0.001)).clamp(0, 1)
        return f / factor * ramp + f * (1 - ramp)

    def _longrope(self, f, p, max_positions):
        out = []
        for key in ("short_factor", "long_factor"):
            by = torch.tensor([float(x) for x in p[key]], dtype=torch.float64, device="cpu")
            if by.shape != f.shape:
                raise ValueError(f"{key} has {by.numel()} numbers for {f.numel()} pairs")
            out.append(f / by)
        factor = p.get("factor") or (max_positions / self.original if max_positions else 1.0)
        given = p.get("attention_factor")
        self.scale = float(given) if given is not None else 1.0 if factor <= 1 else math.sqrt(1 + math.log(factor) / math.log(self.original))
        return out

    def _on(self, device) -> list:
        held = self._held.get(device)
        if held is None:
            with torch.inference_mode(False):             # kept beyond this call: a training pass saves them for its gradients
                held = self._held[device] = [split_frequencies(t).to(device) for t in self._tables]
        return held

    def on(self, device, positions: torch.Tensor) -> Tuple[torch.Tensor, float]:
        """``(freq [pairs, 2], scale)`` for a pass over tokens at ``positions``."""
        held = self._on(device)
        if self.kind == "longrope":
            return torch.where(positions.max() >= self.original, held[1], held[0]), self.scale
        if self.kind == "dynamic" and self.dims > 2:
            length = (positions.max() + 1).clamp_min(self.original).double()
            grown = (self.factor * length / self.original - (self.factor - 1)) ** (self.dims / (self.dims - 2))
            i = torch.arange(0, self.dims, 2, dtype=torch.float64, device=device) / self.dims
            return split_frequencies((self.base * grown) ** -i), self.scale
        return held[0], self.scale


__all__ = ["LAYOUTS", "RotaryPlan", "apply_rotary", "split_frequencies"]
