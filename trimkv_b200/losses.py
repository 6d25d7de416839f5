"""Losses of scoring and training passes: cross entropy straight from the head's weight, and the balance of a router's experts."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import ops


def _once(backward):
    """A backward pass without a gradient of its own: asking for one raises.  (torch's guard alone costs several microseconds a pass, so it
    is put in front only where a graph of the backward pass is being made.)"""
    guarded = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        return (guarded if torch.is_grad_enabled() else backward)(ctx, *grads)
    return staticmethod(run)


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, labels, ignore, reduction, status):
        loss, reduced, plan = ops.vloss_forward(x, w, labels, ignore, reduction, status)
        ctx.save_for_backward(x, w, plan)
        ctx.how = reduction, status
        return reduced if reduction else loss

    @_once
    def backward(ctx, grad):
        x, w, plan = ctx.saved_tensors
        reduction, status = ctx.how
        dx, dw = ops.vloss_backward(x, w, plan, ops.as_float(grad), reduction, ctx.needs_input_grad[0], ctx.needs_input_grad[1], status)
        return dx, dw, None, None, None, None


def _autocast(t: torch.Tensor) -> torch.Tensor:
    return t.to(torch.get_autocast_dtype(t.device.type)) if t.is_floating_point() and t.dtype != torch.float64 else t


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, *, ignore_index: int = -100,
                         reduction: str = "mean", status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``cross_entropy(hidden @ weight.T, labels)`` in fp32 without the logits: ``hidden [..., H]``, ``weight [V, H]``, ``labels [...]``.

    The vocabulary goes by in pieces; what is kept for the gradient is a few numbers per token.  ``reduction``: ``"none"`` (fp32, the
    shape of ``labels``), ``"sum"``, or ``"mean"`` over the labels that are not ``ignore_index`` (NaN where there are none, as in
    ``torch.nn.functional.cross_entropy``).  Ignored tokens cost nothing; their rows are not read and get a gradient of zeros.  A label
    outside the vocabulary makes its token's loss NaN, leaves the token out of the gradients and is recorded in ``status``
    (``ops.new_status``).  Differentiable in hidden and weight; gradients are accumulated in fp32 and rounded once, with the
    gradients of the logits rounded to the inputs' type for the products (the label's, the largest of a token, counts in full for hidden,
    and for weight up to 256 tokens, the first eight of every 32 neighbouring words).  Under autocast hidden and weight are taken in its type, as
    ``torch.nn.functional.linear`` takes them."""
    if reduction not in ops.VLOSS_REDUCTIONS:
        raise ValueError(f"reduction {reduction!r}: one of {sorted(ops.VLOSS_REDUCTIONS)}")
    if weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1] or labels.shape != hidden.shape[:-1]:
        raise ValueError(f"hidden {tuple(hidden.shape)}, weight {tuple(weight.shape)}, labels {tuple(labels.shape)}")
    if weight.shape[0] == 0 or weight.shape[1] == 0:
        raise ValueError(f"an empty weight {tuple(weight.shape)}")
    if torch.is_autocast_enabled(hidden.device.type):
        hidden, weight = (_autocast(t) for t in (hidden, weight))
    ops.dtype_code(hidden.dtype)
    if weight.dtype != hidden.dtype:
        raise TypeError(f"hidden rows in {hidden.dtype}, weight in {weight.dtype}")
    if labels.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"labels of {labels.dtype}: want int32 or int64")
    if not hidden.device == weight.device == labels.device:
        raise ValueError(f"hidden rows on {hidden.device}, weight on {weight.device}, labels on {labels.device}")
    if status is not None and (status.dtype != torch.int32 or status.numel() < 1 or status.device != hidden.device):
        raise ValueError(f"status {status.dtype} {tuple(status.shape)} on {status.device}: want int32 on {hidden.device}, as ops.new_status gives it")
    x = hidden if hidden.dim() == 2 else hidden.reshape(-1, hidden.shape[-1])
    if x.stride(1) != 1 or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        x = x.contiguous()
    loss = _LinearCrossEntropy.apply(x, weight.contiguous(), labels.reshape(-1).to(torch.int64).contiguous(), int(ignore_index),
                                     ops.VLOSS_REDUCTIONS[reduction], status)
    return loss.view(labels.shape) if reduction == "none" and labels.dim() != 1 else loss


def logits_cross_entropy(logits: torch.Tensor, labels: torch.Tensor, *, ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """:func:`linear_cross_entropy` where the logits ``[..., V]`` are there already, in elementary operations on any device: the same loss and
    reductions, ignored rows not counted whatever is in them, NaN for labels outside the vocabulary."""
    live = labels != ignore_index
    counts = live & (labels >= 0) & (labels < logits.shape[-1])
    z = logits.to(torch.promote_types(logits.dtype, torch.float32)).masked_fill(~counts[..., None], 0.0)
    at = labels.long().masked_fill(~counts, 0)
    loss = (z.logsumexp(-1) - z.gather(-1, at[..., None])[..., 0]).masked_fill(~live, 0.0).masked_fill(live & ~counts, float("nan"))
    return loss if reduction == "none" else loss.sum() if reduction == "sum" else loss.sum() / counts.sum()


class _ExpertBalance(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, choice, valid):
        loss, counts, load = ops.moe_balance(logits, choice, valid)
        ctx.save_for_backward(logits, load) if valid is None else ctx.save_for_backward(logits, load, valid)
        ctx.mark_non_differentiable(counts)
        return loss, counts

    @_once
    def backward(ctx, grad, _):
        logits, load, *valid = ctx.saved_tensors
        return ops.moe_balance_grad(logits, valid[0] if valid else None, load, ops.as_float(grad)), None, None


def expert_balance(logits: torch.Tensor, choice: torch.Tensor, valid: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(loss, counts)`` of a router: with p = softmax(logits ``[..., E]``) and the experts chosen for every token (``choice [..., k]``,
    int32 or int64), ``loss = E * sum_e (counts_e / (n k)) * mean_t p_te`` over the n tokens where ``valid [...]`` (bool; None: all) is
    true: 1 where experts are equally used and equally likely, more where they are not, 0 without tokens.  ``counts [E]`` int32.  Entries
    of ``choice`` outside [0, E) count for no expert.  Differentiable in the logits; tokens that are not valid are not read and get zeros."""
    if logits.dim() < 1 or choice.dim() != logits.dim() or choice.shape[:-1] != logits.shape[:-1] or logits.shape[-1] == 0:
        raise ValueError(f"logits {tuple(logits.shape)}, choice {tuple(choice.shape)}")
    if valid is not None and (valid.shape != logits.shape[:-1] or valid.dtype != torch.bool):
        raise ValueError(f"valid {valid.dtype} {tuple(valid.shape)}: want bool {tuple(logits.shape[:-1])}")
    ops.dtype_code(logits.dtype)
    if choice.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"choices of {choice.dtype}: want int32 or int64")
    if choice.device != logits.device or (valid is not None and valid.device != logits.device):
        raise ValueError(f"logits on {logits.device}, choice on {choice.device}, valid on {None if valid is None else valid.device}")
    if logits.dim() != 2:                          # a reshape of two dimensions would only add a node to the graph
        logits, choice = logits.reshape(-1, logits.shape[-1]), choice.reshape(-1, choice.shape[-1])
        valid = None if valid is None else valid.reshape(-1)
    if logits.stride(1) != 1:
        logits = logits.contiguous()
    if choice.stride(1) != 1:
        choice = choice.contiguous()
    return _ExpertBalance.apply(logits, choice, valid)


__all__ = ["expert_balance", "linear_cross_entropy"]
