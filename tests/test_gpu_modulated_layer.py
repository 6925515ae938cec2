"""examples/video_layer.py behind its modulated norms: the branch in 8 bits against the same one in 16, and the gradients
that training sees against the same computation in float64."""
from __future__ import annotations

import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))


@pytest.fixture(scope="module")
def layer_and_inputs():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import video_layer
    return video_layer, video_layer.make((4, 8, 16), heads=6, kv_heads=2, keys=77, width=256, state_width=192,
                                         exact_leaves=8)


def test_served_branch_is_near_its_own(layer_and_inputs):
    """Bound: 8-bit rows of random values are off by a uniform half step of their largest value, about 4 standard deviations,
    over 127: 4 / 127 / sqrt(12) = 0.9 % of their size in the mean square, and so are the weights; the two products, and q and
    k in the logits of size 1, add four times that at most: below 2^-3 of the answer with the 16-bit roundings."""
    video_layer, (layer, *args) = layer_and_inputs
    served, plain, norms = video_layer.modulated(layer, *args)
    assert served.shape == plain.shape and served.dtype is plain.dtype
    off = (served.double() - plain.double()).pow(2).mean().sqrt()
    assert off <= 2.0 ** -3 * plain.double().pow(2).mean().sqrt(), float(off)
    assert norms and all(v > 0 and v < float("inf") for v in norms.values())


def test_gradients_through_the_modulated_norm(layer_and_inputs):
    """The modulation's and the rows' gradients for the same upstream gradient, against float64: each is a bfloat16 rounding
    (2^-8 per element) of a float32 sum."""
    import htrc_b200
    video_layer, (layer, x, positions, states, lengths) = layer_and_inputs
    torch.manual_seed(4)
    step = torch.randn((x.shape[0], 256), device="cuda").bfloat16()
    m = video_layer.Modulated(torch.nn.Identity(), x.shape[-1], 256).cuda().bfloat16()
    with torch.no_grad():
        scale, shift = m.terms(step).chunk(2, -1)
    leaves = [t.detach().clone().requires_grad_() for t in (x, scale, shift)]
    y = htrc_b200.layer_norm(leaves[0], scale=leaves[1], shift=leaves[2])
    assert torch.equal(y, m(x, step))
    dy = torch.randn_like(y)
    y.backward(dy)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    (torch.nn.functional.layer_norm(wide[0], (x.shape[-1],), eps=1e-6) * (1 + wide[1][:, None]) + wide[2][:, None]).backward(dy.double())
    for got, want in zip(leaves, wide):
        assert (got.grad.double() - want.grad).norm() <= 2.0 ** -8 * want.grad.norm()
