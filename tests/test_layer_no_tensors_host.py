"""Arguments that are no tensors are refused by the calls' own checks, whether gradients are recorded or not."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

import htrc_b200
from htrc_b200 import _autograd

x = torch.zeros((4, 64))
w = htrc_b200.Int8Rows(torch.zeros((8, 64), dtype=torch.int8), torch.ones(8))
CALLS = [lambda: htrc_b200.layer_norm([1.0]), lambda: htrc_b200.layer_norm(x, weight=[1.0] * 64),
         lambda: htrc_b200.layer_norm_int8("x"), lambda: htrc_b200.layer_norm_int8(x, scale=0.5), lambda: htrc_b200.quantize_rows(1),
         lambda: htrc_b200.int8_linear(x, w, bias=[0.0] * 8), lambda: htrc_b200.cross_attention([1], [1], [1])]


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("grad", [True, False])
def test_refused_by_a_value_error(call, grad):
    with torch.set_grad_enabled(grad), pytest.raises(ValueError):
        call()


def test_nothing_else_is_recorded():
    assert not _autograd.recorded([1.0], 2, "x", None)
    with fwd.dual_level():
        assert not _autograd.recorded([1.0], 2, "x", None)
