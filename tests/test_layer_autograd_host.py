"""The autograd helpers of the operators around flat attention, without a GPU."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

from htrc_b200 import _autograd


class Square(torch.autograd.Function):
    """x ** 2, its gradient formed as a kernel would: with no graph of its own."""

    @staticmethod
    def forward(ctx, x, w):
        ctx.save_for_backward(x)
        return x * x

    @staticmethod
    def backward(ctx, g):
        (x,) = ctx.saved_tensors
        with torch.no_grad():
            dx = 2 * x * g
        return _autograd.first_order("square", (dx, None), (x, g))


def test_gradients_of_kernels_refuse_to_be_differentiated():
    x = torch.randn(5, requires_grad=True)
    (g,) = torch.autograd.grad(Square.apply(x, None).sum(), x)
    assert not g.requires_grad and torch.equal(g, 2 * x)
    (g,) = torch.autograd.grad(Square.apply(x, None).sum(), x, create_graph=True)
    assert torch.equal(g, 2 * x)
    with pytest.raises(NotImplementedError, match="square has no second derivatives"):
        (g.pow(2).sum() + x.sum()).backward()


def test_what_is_recorded():
    x, w = torch.randn(3), torch.randn(3, requires_grad=True)
    assert _autograd.recorded(x, None, w) and not _autograd.recorded(x, None)
    with torch.no_grad():
        assert not _autograd.recorded(x, w)
        with fwd.dual_level():
            assert not _autograd.recorded(x, w, None)
            assert _autograd.recorded(None, fwd.make_dual(x, torch.ones(3)))
