"""Cross attention under additive masks so low that float32 logits lose their low bits, and rows that hold nothing else.

The operands are small integers and the scale a power of two, so every product and every logit s + bias is a float32
rounding of an exact number: ``Rounded`` takes that one rounding and is float64 otherwise.  The kernels' logits are then the
same numbers, and the bounds of test_gpu_cross.py hold as they stand, whatever the spacing of float32 is at the mask's value."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_cross import F, U, Plain, _keep_and_bias, _within

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
# float32's spacing: 2^-10 at 1e4, 2^-8 at float16's lowest value, 2^-4 at 1e6, 1 at 1e7, 8 at 1e8, 64 at 1e9
FILLS = [(-1e4, F32), (-1e5, F32), (-1e6, F32), (-1e7, F32), (-1e8, F32), (-1e9, F32), (-1e4, F16), (torch.finfo(F16).min, F16),
         (-1e6, BF16), (-1e9, BF16), (-1e30, F32), (torch.finfo(BF16).min, BF16), (torch.finfo(F32).min, F32)]
SCALE = 0.125


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda:0")


class Rounded(Plain):
    def __init__(self, q, k, v, mask):
        self.q, self.k, self.v = (x.double() for x in (q, k, v))
        self.group, self.scale = q.shape[1] // k.shape[1], SCALE
        keep, bias = _keep_and_bias((q.shape[0], q.shape[1], q.shape[2], k.shape[2]), None, mask, q.device)
        self.K, self.V = (x.repeat_interleave(self.group, 1) for x in (self.k, self.v))
        s = torch.where(keep, (self.q @ self.K.mT * SCALE + bias).float().double(), -math.inf)
        top = s.amax(-1, keepdim=True)
        e = torch.exp(s - top)
        total = e.sum(-1, keepdim=True)
        self.p = e / total
        self.lse = (top + total.log())[..., 0]
        self.out = self.p @ self.V
        self.out_bound = self.p @ self.V.abs()


def _operands(dev, size, dtype):
    b, n, m, hq, hk, d = size
    gen = torch.Generator(device=dev).manual_seed(sum(size))
    q, k = (torch.randint(-1, 2, (b, h, r, d), generator=gen, device=dev).to(dtype) for h, r in ((hq, n), (hk, m)))
    v = torch.randn((b, hk, m, d), generator=gen, device=dev).to(dtype)
    return q, k, v, gen


def _masks(kind, size, fill, mask_dtype, gen, dev):
    b, n, m, *_ = size
    rows = 1 if kind == "keys" else n
    soft = torch.randint(-8, 9, (b, 1, rows, m), generator=gen, device=dev) / 8
    bias = torch.where(torch.rand((b, 1, rows, m), generator=gen, device=dev) < 0.6, soft, fill)
    bias[..., 0] = 0.0
    if kind == "keys":
        bias[0] = fill                      # an empty prompt
    else:
        bias[:, :, ::5] = fill
    return bias.to(mask_dtype)


# many rows, a few, one, and few units whose keys are split
@pytest.mark.parametrize("size", [(3, 150, 203, 4, 2, 64), (2, 2, 131, 2, 1, 64), (2, 1, 300, 4, 2, 64), (1, 130, 6000, 1, 1, 64),
                                  (2, 40, 256, 6, 2, 128)])
@pytest.mark.parametrize("kind", ["keys", "pairs"])
@pytest.mark.parametrize("fill,mask_dtype", FILLS)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_rows_of_a_large_finite_bias(dev, dtype, fill, mask_dtype, kind, size):
    import htrc_b200
    q, k, v, gen = _operands(dev, size, dtype)
    mask = _masks(kind, size, fill, mask_dtype, gen, dev)
    kw = dict(mask=mask, scale=SCALE, heads_first=True)
    out, lse = htrc_b200.cross_attention(q, k, v, return_lse=True, **kw)
    ref = Rounded(q, k, v, mask)
    u = U[dtype]
    _within(out, ref.out, u * ref.out.abs() + (u + F) * ref.out_bound, "out")
    do = torch.randn(q.shape, generator=gen, device=dev).to(dtype)
    dlse = torch.randn(lse.shape, generator=gen, device=dev)
    grads = htrc_b200.cross_attention_backward(do, q, k, v, out, lse, dlse=dlse, **kw)
    for name, g, w, bound in zip(("dq", "dk", "dv"), grads, *ref.backward_bounds(do, dlse, u)):
        _within(g, w, bound, name)
    # each row's weights sum to one: the values' gradients are the upstream ones, shared out
    got, want = grads[2].double().sum(2), do.double().unflatten(1, (-1, ref.group)).sum((2, 3))
    assert ((got - want).abs() <= (2 * u + F) * do.double().abs().unflatten(1, (-1, ref.group)).sum((2, 3))).all()
    htrc_b200.cross_status()
