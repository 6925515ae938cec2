"""Derivatives that the operators around flat attention do not have are refused, not dropped: second ones (through a gradient
taken with create_graph) and forward-mode tangents."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda:0")


def _cross(dev):
    import htrc_b200
    gen = torch.Generator(device=dev).manual_seed(1)
    args = [torch.randn((1, r, h, 64), generator=gen, device=dev).bfloat16() for r, h in ((20, 4), (30, 2), (30, 2))]
    return args, lambda q, k, v: htrc_b200.cross_attention(q, k, v, return_lse=True)


def _rotary(dev):
    import htrc_b200
    gen = torch.Generator(device=dev).manual_seed(2)
    args = [torch.randn((1, 9, h, 64), generator=gen, device=dev) for h in (4, 2)]
    args += [torch.rand(64, generator=gen, device=dev) + 0.5 for _ in range(2)]
    pos = torch.arange(9, device=dev, dtype=torch.int32)[:, None]
    return args, lambda q, k, wq, wk: htrc_b200.rotary_qk(q, k, pos, axes=(64,), q_weight=wq, k_weight=wk)


CALLS = [_cross, _rotary]


@pytest.mark.parametrize("make", CALLS)
def test_second_derivatives_are_refused(dev, make):
    args, call = make(dev)
    for i in range(len(args)):
        leaves = [x.clone().requires_grad_(j == i) for j, x in enumerate(args)]
        loss = call(*leaves)[0].float().pow(2).sum() if i != 1 else sum(y.float().sum() for y in call(*leaves))
        (g,) = torch.autograd.grad(loss, leaves[i], create_graph=True)
        with pytest.raises(NotImplementedError, match="second"):
            (g.float().pow(2).sum() + leaves[i].float().sum()).backward()
    # an upstream gradient that is itself differentiated
    leaves = [x.clone().requires_grad_() for x in args]
    out = call(*leaves)[0]
    up = torch.ones_like(out).requires_grad_()
    (g,) = torch.autograd.grad(out, leaves[0], up, create_graph=True)
    with pytest.raises(NotImplementedError, match="second"):
        torch.autograd.grad(g.float().sum(), up)


@pytest.mark.parametrize("make", CALLS)
def test_create_graph_gives_the_same_first_derivatives(dev, make):
    args, call = make(dev)
    leaves = [x.clone().requires_grad_() for x in args]
    plain = torch.autograd.grad(sum(y.float().pow(2).sum() for y in call(*leaves)), leaves)
    graph = torch.autograd.grad(sum(y.float().pow(2).sum() for y in call(*leaves)), leaves, create_graph=True)
    assert all(torch.equal(x, y) for x, y in zip(plain, graph))


@pytest.mark.parametrize("make", CALLS)
@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(dev, make, grad):
    args, call = make(dev)
    for i in range(len(args)):
        with torch.set_grad_enabled(grad), fwd.dual_level():
            inputs = list(args)
            inputs[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(NotImplementedError):
                call(*inputs)
            assert all(torch.isfinite(y).all() for y in call(*args))       # no tangent in hand: as ever
