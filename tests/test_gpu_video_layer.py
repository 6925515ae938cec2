"""examples/video_layer.py: the operators together, against the same layer written in float64."""
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
    # 512 tokens are 8 leaves, all of them opened: flat attention is then softmax attention of 8-bit q and k
    return video_layer, video_layer.make((4, 8, 16), heads=6, kv_heads=2, keys=77, width=256, state_width=192,
                                         exact_leaves=8)


def _norm(x, w):
    return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6) * w.double()


def _turn(x, positions):
    per = [44, 42, 42]
    at = torch.cat([torch.full((w // 2,), i) for i, w in enumerate(per)]).to(x.device)
    f = torch.cat([10000.0 ** (-torch.arange(0, w, 2, dtype=torch.float64) / w) for w in per]).to(x.device)
    angle = (positions.double()[..., at] * f)[..., None, :]
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], -1).flatten(-2)


def _attend(q, k, v, lengths=None):
    g = q.shape[2] // k.shape[2]
    k, v = (x.repeat_interleave(g, 2) for x in (k, v))
    s = torch.einsum("bnhd,bmhd->bhnm", q, k) * 128 ** -0.5
    if lengths is not None:
        s = s.masked_fill(torch.arange(k.shape[1], device=q.device) >= lengths.view(-1, 1, 1, 1), -torch.inf)
    return torch.einsum("bhnm,bmhd->bnhd", s.softmax(-1), v).flatten(2)


def test_layer_matches_float64(layer_and_inputs):
    """Bound: every tensor that is rounded to bfloat16 on the way (q, k, v, the attention's answer, the projections'
    outputs: seven in a row at most) adds at most 2^-8 of its size in the mean square, the 8-bit q and k of the flat
    operator about 1 / 127 of theirs on logits of size 1; all of it together stays below 2^-4 of the answer's rms."""
    _, (layer, x, positions, states, lengths) = layer_and_inputs
    with torch.no_grad():
        y = layer(x, positions, states, lengths)
        own, pr = layer.own, layer.prompt
        d = x.double()
        q, k, v = (d @ own.qkv.weight.double().T).unflatten(-1, (3, 6, 128)).unbind(-3)
        a = _attend(_turn(_norm(q, own.norm[0]), positions), _turn(_norm(k, own.norm[1]), positions), v)
        d = d + a @ own.out.weight.double().T
        k, v = (states.double() @ pr.kv.weight.double().T).unflatten(-1, (2, 2, 128)).unbind(-3)
        q = (d @ pr.q.weight.double().T).unflatten(-1, (6, 128))
        a2 = _attend(_norm(q, pr.norm[0]), _norm(k, pr.norm[1]), v, lengths)
        add = a2 @ pr.out.weight.double().T
    both = d - x.double() + add
    err = (y.double() - (d + add)).pow(2).mean().sqrt()
    # x itself is carried in bfloat16: its rounding, twice
    assert err <= 2.0 ** -4 * both.pow(2).mean().sqrt() + 2 * 2.0 ** -8 * x.double().pow(2).mean().sqrt(), float(err)


def test_training_lowers_the_error(layer_and_inputs):
    video_layer, (layer, *args) = layer_and_inputs
    losses = video_layer.train(layer, *args, steps=12, rate=2e-3)
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in layer.prompt.parameters())
    assert losses[-1] < 0.8 * losses[0], losses
