"""Float16 gradients of cross attention whatever the size of the upstream gradient: what enters a product as float16 must not
fall into its subnormals long before the result does.

Bounds as in test_gpu_cross.py but for the subnormals: P and dS are to be carried times 2^t at least, with t the largest that
keeps 2^t (2 dim max|dout| max|v| + max|dlse|), a bound on dS, below 2^15, from 0 to 12.  A value that is still subnormal then
has an absolute error of 2^-25 2^-t, and the result one of 2^-25."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_cross import U, Plain, _mask, _rows

pytestmark = pytest.mark.gpu

F16 = torch.float16


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda:0")


def _subnormal(do, v, dlse, group):
    """2^-25 2^-t per batch entry and key head."""
    size = 2 * do.shape[-1] * do.double().abs().unflatten(1, (-1, group)).amax((2, 3, 4)) * v.double().abs().amax((2, 3))
    if dlse is not None:
        size = size + dlse.double().abs().unflatten(1, (-1, group)).amax((2, 3))
    # (one more than t's own rule allows, for a bound that the kernels' float32 puts on the other side of a power of two)
    t = (14 - torch.floor(torch.log2(size.clamp_min(1e-30))) - 1).clamp(0, 12)
    return 2.0 ** (-25 - t)


def _check(q, k, v, do, dlse=None, **kw):
    import htrc_b200
    out, lse = htrc_b200.cross_attention(q, k, v, heads_first=True, return_lse=True, **kw)
    got = htrc_b200.cross_attention_backward(do, q, k, v, out, lse, dlse=dlse, heads_first=True, **kw)
    ref = Plain(q, k, v, kw.get("key_lengths"), kw.get("mask"))
    eps = _subnormal(do, v, dlse, ref.group)
    each = eps.repeat_interleave(ref.group, 1)[..., None, None]
    seen = (ref.p > 0).double()
    fold = lambda x: x.unflatten(1, (-1, ref.group)).sum(2)  # noqa: E731
    more = (ref.scale * each * (seen @ ref.K.abs()), ref.scale * eps[..., None, None] * fold(seen.mT @ ref.q.abs()),
            eps[..., None, None] * fold(seen.mT @ do.double().abs()))
    for name, g, w, bound, extra in zip(("dq", "dk", "dv"), got, *ref.backward_bounds(do, dlse, U[F16]), more):
        assert torch.isfinite(g).all(), name
        over = (g.double() - w).abs() - bound - extra - 2.0 ** -25
        assert (over <= 0).all(), (name, float(over.max()))
    htrc_b200.cross_status()
    return got


# ordinary, long keys, one query, split keys, shared heads with an odd head size
SIZES = [(2, 150, 203, 4, 2, 64), (1, 64, 4000, 2, 2, 128), (2, 1, 300, 4, 2, 128), (1, 130, 6000, 1, 1, 64), (1, 2000, 40, 6, 3, 72)]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("upstream", [30.0, 1.0, 1e-2, 1e-3, 1e-4, 1e-5, 1e-6])
@pytest.mark.parametrize("with_dlse", [False, True])
def test_any_upstream_gradient(dev, size, upstream, with_dlse):
    gen = torch.Generator(device=dev).manual_seed(sum(size))
    q, k, v = _rows(dev, *size, F16, seed=sum(size))
    do = (torch.randn(q.shape, generator=gen, device=dev) * upstream).half()
    dlse = torch.randn(q.shape[:3], generator=gen, device=dev) * upstream if with_dlse else None
    _check(q, k, v, do, dlse)


@pytest.mark.parametrize("size", [(3, 150, 203, 4, 2, 128), (3, 40, 5000, 2, 1, 64), (3, 2, 131, 2, 1, 72)])
@pytest.mark.parametrize("kind", ["lengths", "keys", "keys of heads", "pairs", "key bias", "bias", "keys and lengths", "none kept"])
@pytest.mark.parametrize("upstream", [1.0, 1e-5])
def test_masks(dev, size, kind, upstream):
    b, n, m, h, hk, d = size
    gen = torch.Generator(device=dev).manual_seed(len(kind))
    lengths, mask = _mask(kind, b, h, n, m, F16, dev)
    q, k, v = _rows(dev, *size, F16, seed=len(kind))
    do = (torch.randn(q.shape, generator=gen, device=dev) * upstream).half()
    _check(q, k, v, do, key_lengths=lengths, mask=mask)


@pytest.mark.parametrize("size", [(2, 150, 203, 4, 2, 64), (1, 40, 5000, 2, 1, 128)])
@pytest.mark.parametrize("values", [1e-3, 300.0, 8000.0])
@pytest.mark.parametrize("upstream", [1e-6, 1e-4, 1e-2])
def test_large_and_small_values(dev, size, values, upstream):
    """The bound on dS goes by the values too: nothing overflows."""
    gen = torch.Generator(device=dev).manual_seed(sum(size))
    q, k, v = _rows(dev, *size, F16, seed=sum(size))
    v = (v.float() * values).half()
    do = (torch.randn(q.shape, generator=gen, device=dev) * upstream).half()
    _check(q, k, v, do)


@pytest.mark.parametrize("kind", ["lengths", "keys", "key bias"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, 60000.0])
def test_excluded_keys_and_empty_rows_do_not_count(dev, kind, bad):
    import htrc_b200
    b, n, m, h, hk, d = 3, 150, 203, 4, 2, 64
    gen = torch.Generator(device=dev).manual_seed(8)
    lengths, mask = _mask(kind, b, h, n, m, F16, dev)
    keep = torch.ones((b, 1, 1, m), dtype=torch.bool, device=dev)
    if lengths is not None:
        keep &= torch.arange(m, device=dev) < lengths.view(b, 1, 1, 1)
    if mask is not None:
        keep &= mask if mask.dtype == torch.bool else mask != -math.inf
    q, k, v = _rows(dev, b, n, m, h, hk, d, F16)
    do = (torch.randn(q.shape, generator=gen, device=dev) * 1e-5).half()
    kw = dict(key_lengths=lengths, mask=mask, heads_first=True)
    out, lse = htrc_b200.cross_attention(q, k, v, return_lse=True, **kw)
    want = htrc_b200.cross_attention_backward(do, q, k, v, out, lse, **kw)
    dirty = (~keep[:, 0, 0, :, None])[:, None].expand(k.shape)
    got = htrc_b200.cross_attention_backward(do, q, k.masked_fill(dirty, bad), v.masked_fill(dirty, bad), out, lse, **kw)
    assert all(torch.equal(x, y) for x, y in zip(want, got))


@pytest.mark.parametrize("size", [(2, 500, 300, 4, 2, 128), (1, 23, 3287, 3, 3, 128), (3, 777, 130, 12, 4, 64)])
def test_one_result_whatever_the_stream_or_the_run(dev, size):
    """Under a graph, on a side stream and right behind another call that reuses its workspace."""
    import htrc_b200
    q, k, v = _rows(dev, *size, F16)
    gen = torch.Generator(device=dev).manual_seed(9)
    do = (torch.randn(q.shape, generator=gen, device=dev) * 1e-4).half()
    mask = torch.randn((size[0], 1, 1, size[2]), generator=gen, device=dev).half()
    out, lse = htrc_b200.cross_attention(q, k, v, mask=mask, heads_first=True, return_lse=True)

    def grads():
        return htrc_b200.cross_attention_backward(do, q, k, v, out, lse, mask=mask, heads_first=True)

    first = grads()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = grads()
    torch.cuda.current_stream().wait_stream(side)
    htrc_b200.cross_attention_backward(do * 100, q, k, v * 50, out, lse, mask=mask, heads_first=True)
    third = grads()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        fourth = grads()
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    for other in (second, third, fourth):
        assert all(torch.equal(x, y) for x, y in zip(first, other))
    htrc_b200.cross_status()
