"""What the operators' autograd functions share: they have first derivatives in reverse mode, and others are refused where
they would be lost."""
from __future__ import annotations

import torch
from torch.autograd import forward_ad


def recorded(*tensors):
    """Whether a call with these inputs goes through its autograd function: to record it, or to be refused there because
    one of them carries a forward-mode tangent (the functions have no jvp)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    if forward_ad._current_level >= 0:
        return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)
    return False


class _FirstOrder(torch.autograd.Function):
    """Gradients that depend on tensors, without the derivative of that dependence."""

    @staticmethod
    def forward(ctx, what, count, *tensors):
        ctx.what = what
        return tuple(g.view_as(g) for g in tensors[:count])

    @staticmethod
    def backward(ctx, *_):
        raise NotImplementedError(f"{ctx.what} has no second derivatives")


def first_order(what, grads, sources):
    """``grads``, computed from ``sources`` by kernels: under create_graph their own derivatives raise, rather than be
    taken for zero."""
    if not torch.is_grad_enabled():
        return grads
    held = [g for g in grads if g is not None]
    marked = iter(_FirstOrder.apply(what, len(held), *held, *(t for t in sources if t is not None)))
    return tuple(None if g is None else next(marked) for g in grads)
