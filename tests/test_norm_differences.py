"""Layer norm's gradients against differences of its results, coordinate by coordinate, so that the formula of the backward is
not used to test itself.

x: with u the normalised row and e the step over |x - mean|, a row's result is a constant plus sqrt(W) A (u + e d) / |u + e d|,
whose Taylor coefficients in e are u P_n + d P_(n-1), P_n Legendre polynomials of an angle's cosine: at most 2.  The differences
8 (f(t) - f(-t)) - (f(2 t) - f(-2 t)) over 12 t are off by at most 4 |a_5| h^4 + 20 |a_7| h^6 + ..  <= 9 h^4 of sqrt(W) |A dy|
for h = t / |x - mean| <= 0.1 (eps is a millionth of the variance).  The parameters: the result is linear in each, so a difference
over 2 t is exact.  Steps and inputs are on a grid that float32 holds.  What is left is rounding: a result is within 2^-15 of its
terms' sizes and half a step of float32, the gradients within twice 2^-15 of theirs (theirs and that of the statistics).

The first test plants mistakes in the float64 gradients and wants each of them seen under the same bounds."""
from __future__ import annotations

import pytest
import torch

import htrc_b200

NOISE, U, EPS = 2.0 ** -15, 2.0 ** -24, 1e-6
NAMES = ("weight", "bias", "scale", "shift")
STEP = 0.75


def _inputs(width, device, dtype):
    """x, dy [2, 3, width] and the parameters, multiples of 2^-12."""
    gen = torch.Generator().manual_seed(width)

    def grid(*shape, size=1.0, offset=0.0):
        t = torch.randn(shape, generator=gen).clamp(-3, 3) * size + offset
        return ((t * 4096).round() / 4096).to(device=device, dtype=dtype)
    x, dy = grid(2, 3, width, offset=0.25), grid(2, 3, width)
    return x, dy, dict(weight=grid(width, size=0.5, offset=1.0), bias=grid(width, size=0.5), scale=grid(2, width, size=0.3),
                       shift=grid(2, width, size=0.3))


def _sizes(x, kw):
    """In float64: A, u, rstd, and how far a float32 result may be off."""
    x, (w, b, s, t) = x.double(), (kw[k].double() for k in NAMES)
    mean = x.mean(-1, keepdim=True)
    rstd = (x - mean).pow(2).mean(-1, keepdim=True).add(EPS).rsqrt()
    u, a = (x - mean) * rstd, w * (1 + s[:, None])
    b = b * (1 + s[:, None])
    off = NOISE * (a.abs() * (u.abs() + rstd * x.abs().mean(-1, keepdim=True)) + b.abs() + t[:, None].abs())
    return a, u, rstd, off + U * (u * a + b + t[:, None]).abs()


def _by_x(call, x, dy, kw):
    """The derivatives by x, and what differences and rounding leave."""
    batch, tokens, width = x.shape
    one = torch.eye(width, device=x.device, dtype=x.dtype)[:, None] * STEP
    moved = x[:, :, None, None] + torch.cat([one * k for k in (-2, -1, 1, 2)], 1)      # [batch, tokens, coordinate, 4, width]
    rows = moved.reshape(batch, -1, width)

    def total(y):
        return (y.double().reshape(moved.shape) * dy.double()[:, :, None, None]).sum(-1)
    f = total(call(rows, **kw))
    off = (_sizes(rows, kw)[3].reshape(moved.shape) * dy.double().abs()[:, :, None, None]).sum(-1)
    a, _, rstd, _ = _sizes(x, kw)
    h = STEP * rstd / width ** 0.5
    assert float(h.max()) <= 0.1
    num = (8 * (f[..., 2] - f[..., 1]) - (f[..., 3] - f[..., 0])) / (12 * STEP)
    left = (8 * (off[..., 2] + off[..., 1]) + off[..., 3] + off[..., 0]) / (12 * STEP)
    return num, left + 9 * h ** 4 * rstd * (a * dy.double()).norm(dim=-1, keepdim=True)


def _by_parameter(call, x, dy, kw, name):
    value = kw[name]
    num, left = (torch.zeros(value.numel(), dtype=torch.float64, device=x.device) for _ in range(2))
    for i in range(value.numel()):
        f, off = [], 0.0
        for sign in (1, -1):
            moved = value.clone()
            moved.view(-1)[i] += sign
            new = {**kw, name: moved}
            f.append((call(x, **new).double() * dy.double()).sum())
            # the other columns' results are the same ones
            n, at = i % x.shape[-1], slice(None) if value.dim() == 1 else slice(i // x.shape[-1], i // x.shape[-1] + 1)
            off = off + (_sizes(x, new)[3][at, :, n] * dy[at, :, n].double().abs()).sum()
        num[i], left[i] = (f[0] - f[1]) / 2, off / 2
    return num.view(value.shape), left.view(value.shape)


def _gradients(x, dy, kw, without=None):
    """The formula in float64 (with a mistake), and each value's sizes."""
    a, u, rstd, _ = _sizes(x, kw)
    w, b, s = (kw[k].double() for k in NAMES[:3])
    dy, s = dy.double(), 1 + s[:, None]
    g = dy * (w if without == "modulation in dx" else s if without == "weight in dx" else a)
    gu = g * u
    mean, mean_u = g.mean(-1, keepdim=True), gu.mean(-1, keepdim=True)
    if without == "mean of g":
        mean = mean * 0
    if without == "mean of g u":
        mean_u = mean_u * 0
    one = 1 if without == "modulation of the sums" else s
    sum_u = (dy * u * one).sum((0, 1))
    got = [rstd * (g - mean - u * mean_u), sum_u, (dy * one).sum((0, 1)),
           (dy * (u * w + (0 if without == "bias in dscale" else b))).sum(1), dy.sum(1)]
    if without == "weight in dscale":
        got[3] = (dy * (u + b)).sum(1)
    if without == "last token":
        got[4] = dy[:, :-1].sum(1)
    sizes = [rstd * (g.abs() + g.abs().mean(-1, keepdim=True) + u.abs() * gu.abs().mean(-1, keepdim=True)), (dy * u * s).abs().sum((0, 1)),
             (dy * s).abs().sum((0, 1)), (dy * u * w).abs().sum(1) + (dy * b).abs().sum(1), dy.abs().sum(1)]
    return got, sizes


def _differences(call, x, dy, kw):
    return [_by_x(call, x, dy, kw), *(_by_parameter(call, x, dy, kw, k) for k in NAMES)]


def _worst(got, sizes, wants):
    """For each gradient the largest error over its bound: at most 1 where it is right."""
    return [float(((g.double() - num).abs() / (left + 2 * NOISE * size + U * g.double().abs())).max())
            for g, size, (num, left) in zip(got, sizes, wants)]


MISTAKES = {"mean of g": 0, "mean of g u": 0, "modulation in dx": 0, "weight in dx": 0, "modulation of the sums": 1,
            "bias in dscale": 3, "weight in dscale": 3, "last token": 4}


def test_a_missing_term_is_seen():
    x, dy, kw = _inputs(96, "cpu", torch.float64)

    def call(x, weight, bias, scale, shift):
        a, u, _, _ = _sizes(x, dict(zip(NAMES, (weight, bias, scale, shift))))
        return u * a + bias * (1 + scale[:, None]) + shift[:, None]
    wants = _differences(call, x, dy, kw)
    assert max(_worst(*_gradients(x, dy, kw), wants)) <= 1
    for mistake, at in MISTAKES.items():
        worst = _worst(*_gradients(x, dy, kw, mistake), wants)
        assert worst[at] > 2, mistake
    assert _worst(*_gradients(x, dy, kw, "modulation of the sums"), wants)[2] > 2


@pytest.mark.gpu
@pytest.mark.parametrize("width", [96, 97, 264])
def test_gradients_are_the_differences(width):
    """Rows of a warp, rows by elements and a CTA's rows."""
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    x, dy, kw = _inputs(width, "cuda", torch.float32)
    _, mean, rstd = htrc_b200.layer_norm(x, **kw, return_stats=True)
    got = htrc_b200.layer_norm_backward(dy, x, mean, rstd, **kw)
    worst = _worst(got, _gradients(x, dy, kw)[1], _differences(htrc_b200.layer_norm, x, dy, kw))
    assert max(worst) <= 1, worst
