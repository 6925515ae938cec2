"""Rotary positions with a norm whose eps is zero: only a row of zeros may then divide by zero, never the rows that fill up
a warp's batch.  Bounds as in test_gpu_rotary.py."""
from __future__ import annotations

import pytest
import torch

from test_gpu_rotary import _close, _major, _plain, _plain_backward

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda:0")


# heads that fill a warp's batches of rows and heads that do not, rows shared between tokens (one and two heads), rows past
# the end, and a head size of the general kernel
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dim,axes", [(128, (44, 42, 42)), (64, (20, 22, 22)), (256, (64, 64, 64)), (37, (8, 6, 0))])
@pytest.mark.parametrize("b,n,hq,hk", [(1, 700, 24, 8), (2, 333, 4, 3), (1, 41, 40, 5), (3, 47, 2, 1), (1, 1, 1, 1), (1, 2500, 16, 7)])
def test_zero_eps(dev, dtype, dim, axes, b, n, hq, hk):
    import htrc_b200
    gen = torch.Generator(device=dev).manual_seed(n + hq + dim)
    q, k = (torch.randn((b, n, h, dim), generator=gen, device=dev).to(dtype) for h in (hq, hk))
    pos = torch.randint(0, 900, (b, n, 3), generator=gen, device=dev, dtype=torch.int32)
    wq, wk = (1 + 0.3 * torch.randn(dim, generator=gen, device=dev) for _ in range(2))
    kw = dict(axes=axes, q_weight=wq, k_weight=wk, eps=0.0, heads_first=True)
    got = htrc_b200.rotary_qk(q, k, pos, **kw)
    dy = [torch.randn(y.shape, generator=gen, device=dev).to(dtype) for y in got]
    dq, dk, dwq, dwk = htrc_b200.rotary_qk_backward(*dy, q, k, pos, **kw)
    for x, w, y, g, dx, dw in zip((q, k), (wq, wk), got, dy, (dq, dk), (dwq, dwk)):
        _close(_major(y, True), *_plain(x, pos, axes, "interleaved", w, eps=0.0))
        want, size, want_w, size_w = _plain_backward(_major(g, True), x, pos, axes, "interleaved", w, eps=0.0)
        _close(dx, want, size)
        _close(dw, want_w, size_w)
