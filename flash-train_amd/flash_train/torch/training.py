"""Differentiable forms of the operators around a training step's products."""

from typing import NamedTuple, Optional

import torch

from ._flash_train_torch import (
    linear_cross_entropy_backward,
    linear_cross_entropy_forward,
    moe_route_backward,
    moe_route_forward,
)


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, target, ignore_index):
        loss, lse = linear_cross_entropy_forward(hidden, weight, target, ignore_index)
        ctx.save_for_backward(hidden, weight, target, lse)
        ctx.ignore_index = ignore_index
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        hidden, weight, target, lse = ctx.saved_tensors
        grads = linear_cross_entropy_backward(grad_loss, hidden, weight, target, lse, ctx.ignore_index)
        return grads[0], grads[1], None, None


def linear_cross_entropy(
    hidden: torch.Tensor,
    weight: torch.Tensor,
    target: torch.Tensor,
    ignore_index: int = -100,
    reduction: str = "mean",
) -> torch.Tensor:
    """Softmax cross entropy of ``hidden @ weight.T`` (tokens x classes) against ``target``.

    ``reduction`` is "none" (a loss for every token, 0 where ``target`` is
    ``ignore_index``), "sum" or "mean" (over the tokens that are not ignored;
    NaN when all are).  Losses are fp32.
    """
    if reduction not in ("none", "sum", "mean"):
        raise RuntimeError(f"reduction must be none, sum or mean, not {reduction!r}")
    loss = _LinearCrossEntropy.apply(hidden, weight, target, ignore_index)
    if reduction == "none":
        return loss
    if reduction == "sum":
        return loss.sum()
    return loss.sum() / (target != ignore_index).sum()


class Routing(NamedTuple):
    """What ``moe_route`` returns: the forward call's values, ``gates`` and
    ``balance_loss`` differentiable in the logits."""

    experts: torch.Tensor
    gates: torch.Tensor
    slots: torch.Tensor
    counts: torch.Tensor
    balance_loss: torch.Tensor


class _MoeRoute(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_k, normalize, mask):
        experts, gates, slots, counts, routed, loss = moe_route_forward(logits, top_k, normalize, mask)
        ctx.save_for_backward(logits, experts, counts, routed, mask)
        ctx.normalize = normalize
        ctx.mark_non_differentiable(experts, slots, counts)
        return experts, gates, slots, counts, loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, _experts, grad_gates, _slots, _counts, grad_loss):
        logits, experts, counts, routed, mask = ctx.saved_tensors
        grad = moe_route_backward(grad_gates, grad_loss, logits, experts, counts, routed, ctx.normalize, mask)
        return grad, None, None, None


def moe_route(
    logits: torch.Tensor, top_k: int, normalize: bool = False, mask: Optional[torch.Tensor] = None
) -> Routing:
    """The ``top_k`` experts of every row of ``logits`` (tokens x experts).

    ``slots`` are the rows that the choices take when they are packed by
    expert, and ``counts`` the rows of each expert's group: the packing that
    the grouped products read.  ``mask`` (bool) leaves rows out.
    """
    return Routing(*_MoeRoute.apply(logits, top_k, normalize, mask))
