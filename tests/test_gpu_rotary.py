"""Rotary positions over several axes (htrc_b200.rotary_axes / rotary_qk) against a float64 implementation.

Bounds, derived before the first run.  The kernels compute in float32 and round once.  A rotated element is
a cos - b sin of two normalised elements: each carries the norm's relative error (a sum of at most 256 squares, a
reciprocal square root and two products: below 2^-18 with a wide margin over 256 * 2^-24 / 2), the cosine and sine an
absolute 2^-21 (an angle reduced to 2^-25 revolutions, then 2 ulp), so |error| <= 2^-17 * hypot(a, b) before the final
rounding, of relative u = 2^-8 (bfloat16), 2^-11 (float16) or 2^-24 (float32), plus float16's subnormal spacing.
The backward adds a mean over the row: its error is bounded by 2^-17 of the sum of the absolute terms."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
NOISE = 2.0 ** -17


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda:0")


def _turn(axes, positions, theta=10000.0, freqs=None):
    """cos and sin [.., 1, R / 2] in float64."""
    per = [torch.arange(0, w, 2, dtype=torch.float64, device=positions.device) for w in axes]
    f = torch.cat([theta ** (-a / w) for a, w in zip(per, axes) if w] or [positions.new_zeros(0, dtype=torch.float64)])
    if freqs is not None:
        f = torch.tensor(freqs, dtype=torch.float64, device=positions.device)
    at = torch.cat([torch.full((w // 2,), i, dtype=torch.long) for i, w in enumerate(axes)]).to(positions.device)
    angle = positions.double()[..., at] * f
    return angle.cos()[..., None, :], angle.sin()[..., None, :]


def _rotate(x, cos, sin, pairs):
    r = 2 * cos.shape[-1]
    y = x.clone()
    a, b = (slice(0, r, 2), slice(1, r, 2)) if pairs == "interleaved" else (slice(0, r // 2), slice(r // 2, r))
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., a] * sin + x[..., b] * cos
    return y


def _size(x, r, pairs):
    """hypot of each element's pair (the element itself past the rotated width)."""
    s = x.abs().clone()
    a, b = (slice(0, r, 2), slice(1, r, 2)) if pairs == "interleaved" else (slice(0, r // 2), slice(r // 2, r))
    s[..., a] = s[..., b] = torch.hypot(x[..., a], x[..., b])
    return s


def _plain(x, positions, axes, pairs, weight, eps=1e-6, **kw):
    """(result, size of what each element was formed from), float64 token-major."""
    cos, sin = _turn(axes, positions, **kw)
    u = x.double()
    if weight is not None:
        u = u * torch.rsqrt(u.pow(2).mean(-1, keepdim=True) + eps) * weight.double()
    return _rotate(u, cos, sin, pairs), _size(u, sum(axes), pairs)


def _plain_backward(dy, x, positions, axes, pairs, weight, eps=1e-6):
    """(dx, its bound's sum of absolute terms, dw, its bound's), float64 token-major."""
    cos, sin = _turn(axes, positions)
    g = _rotate(dy.double(), cos, -sin, pairs)
    gs = _size(dy.double(), sum(axes), pairs)
    if weight is None:
        return g, gs, None, None
    x, w = x.double(), weight.double()
    r = torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    lead = tuple(range(x.dim() - 1))
    dw, dws = (g * x * r).sum(lead), (gs * x.abs() * r).sum(lead)
    h, hs = g * w, gs * w.abs()
    dx = r * (h - x * r * r * (h * x).mean(-1, keepdim=True))
    dxs = r * (hs + x.abs() * r * r * (hs * x.abs()).mean(-1, keepdim=True))
    return dx, dxs, dw, dws


def _close(got, want, size, noise=NOISE):
    u = U[got.dtype]
    err = (got.double() - want).abs()
    bound = u * want.abs() + noise * size + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    assert torch.isfinite(got).all()
    assert (err <= bound).all(), float((err - bound).max())


def _major(x, heads_first):
    return x.transpose(-3, -2) if heads_first else x


# dim, axes: aligned, padded lanes, partial rotation, an odd number of pairs, an odd dim, one axis, four, none
SHAPES = [(128, (44, 42, 42)), (64, (20, 22, 22)), (80, (16, 24, 24)), (72, (24, 24, 24)), (128, (10, 6, 0)), (37, (8, 6)),
          (256, (256,)), (16, (4, 4, 4, 4)), (96, (0,)), (200, (64, 66, 66))]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("pairs", ["interleaved", "half"])
@pytest.mark.parametrize("dim,axes", SHAPES)
def test_forward_and_backward_match_float64(dev, dtype, pairs, dim, axes):
    import htrc_b200
    gen = torch.Generator(device=dev).manual_seed(dim * 7 + len(axes))
    for (b, n, hq, hk), norm, hf in [((2, 37, 5, 2), True, True), ((1, 130, 3, 3), False, False), ((3, 1, 1, 1), True, False)]:
        q = (torch.randn((b, n, hq, dim), generator=gen, device=dev) * 1.7).to(dtype)
        k = torch.randn((b, n, hk, dim), generator=gen, device=dev).to(dtype)
        pos = torch.randint(-300, 5000, (b, n, len(axes)), generator=gen, device=dev, dtype=torch.int32)
        wq = (1 + 0.3 * torch.randn(dim, generator=gen, device=dev)) if norm else None
        wk = (1 + 0.3 * torch.randn(dim, generator=gen, device=dev)).to(dtype) if norm else None
        kw = dict(axes=axes, pairs=pairs, q_weight=wq, k_weight=wk, heads_first=hf)
        got = htrc_b200.rotary_qk(q, k, pos, **kw)
        for x, w, y in zip((q, k), (wq, wk), got):
            want, size = _plain(x, pos, axes, pairs, w)
            assert y.is_contiguous() and y.dtype == dtype
            _close(_major(y, hf), want, size)
        dy = [torch.randn(y.shape, generator=gen, device=dev).to(dtype) for y in got]
        dq, dk, dwq, dwk = htrc_b200.rotary_qk_backward(*dy, q, k, pos, **kw)
        for x, w, g, dx, dw in zip((q, k), (wq, wk), dy, (dq, dk), (dwq, dwk)):
            want, size, want_w, size_w = _plain_backward(_major(g, hf), x, pos, axes, pairs, w)
            _close(dx, want, size)
            if norm:
                assert dw.dtype == w.dtype
                _close(dw, want_w, size_w)
            else:
                assert dw is None


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("b,n,hq,hk", [(2, 137, 2, 1), (3, 61, 1, 1), (1, 20011, 2, 2), (1, 20011, 3, 1), (5, 4001, 6, 2)])
def test_few_heads_and_many_tokens(dev, dtype, b, n, hq, hk):
    """Rows of several tokens per warp, and more rows than one pass over the grid takes."""
    import htrc_b200
    gen = torch.Generator(device=dev).manual_seed(n + hq)
    for dim, axes, pairs in [(64, (20, 22, 22), "half"), (72, (8, 16, 24), "interleaved"), (128, (44, 42, 42), "interleaved")]:
        q = torch.randn((b, n, hq, dim), generator=gen, device=dev).to(dtype)
        k = torch.randn((b, n, hk, dim), generator=gen, device=dev).to(dtype)
        pos = torch.randint(0, 3000, (b, n, 3), generator=gen, device=dev, dtype=torch.int32)
        wq = 1 + 0.3 * torch.randn(dim, generator=gen, device=dev)
        wk = 1 + 0.3 * torch.randn(dim, generator=gen, device=dev)
        kw = dict(axes=axes, pairs=pairs, q_weight=wq, k_weight=wk, heads_first=True)
        got = htrc_b200.rotary_qk(q, k, pos, **kw)
        for x, w, y in zip((q, k), (wq, wk), got):
            _close(_major(y, True), *_plain(x, pos, axes, pairs, w))
        dy = [torch.randn(y.shape, generator=gen, device=dev).to(dtype) for y in got]
        dq, dk, dwq, dwk = htrc_b200.rotary_qk_backward(*dy, q, k, pos, **kw)
        for x, w, g, dx, dw in zip((q, k), (wq, wk), dy, (dq, dk), (dwq, dwk)):
            want, size, want_w, size_w = _plain_backward(_major(g, True), x, pos, axes, pairs, w)
            _close(dx, want, size)
            _close(dw, want_w, size_w)


@pytest.mark.parametrize("pairs", ["interleaved", "half"])
def test_late_positions_keep_their_accuracy(dev, pairs):
    """int32 positions are reduced exactly: the last ones rotate as accurately as the first."""
    import htrc_b200
    x = torch.randn((6, 2, 64), device=dev)
    pos = torch.tensor([[0], [1], [2 ** 24 + 1], [2 ** 31 - 1], [-2 ** 31], [-77777777]], dtype=torch.int32, device=dev)
    want, size = _plain(x, pos, (64,), pairs, None)
    # float64's own angle: 2^31 radians carry 2^-22 of absolute error
    _close(htrc_b200.rotary_axes(x, pos, axes=(64,), pairs=pairs), want, size, NOISE + 2.0 ** -21)


def test_float_positions_and_frequencies(dev):
    import htrc_b200
    gen = torch.Generator(device=dev).manual_seed(5)
    x = torch.randn((2, 50, 3, 48), generator=gen, device=dev)
    pos = torch.rand((50, 2), generator=gen, device=dev) * 700 - 40
    freqs = [0.9 ** i for i in range(20)]
    for dt in (torch.float32, torch.float64):
        y = htrc_b200.rotary_axes(x, pos.to(dt), axes=(24, 16), freqs=freqs)
        want, size = _plain(x, pos, (24, 16), "interleaved", None, freqs=freqs)
        _close(y, want, size)
    ip = torch.randint(0, 2000, (50, 2), generator=gen, device=dev)                    # int64
    y = htrc_b200.rotary_axes(x, ip, axes=(24, 16), freqs=freqs, pairs="half")
    want, size = _plain(x, ip, (24, 16), "half", None, freqs=freqs)
    _close(y, want, size)
    y = htrc_b200.rotary_axes(x, ip, axes=[24, 16], theta=500.0, pairs="half")
    want, size = _plain(x, ip, (24, 16), "half", None, theta=500.0)
    _close(y, want, size)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_alignment_and_broadcast(dev, dtype):
    """Slices of a joint projection, rows off the 16-byte grid, a transposed and an expanded input, shared positions."""
    import htrc_b200
    gen = torch.Generator(device=dev).manual_seed(6)
    b, n, h, d = 2, 33, 4, 64
    axes, w = (20, 22, 22), 1 + 0.1 * torch.randn(64, generator=gen, device=dev)
    pos = torch.randint(0, 90, (1, n, 3), generator=gen, device=dev, dtype=torch.int32)
    joint = torch.randn((b, n, 3 * h * d + 1), generator=gen, device=dev).to(dtype)
    rows = {
        "slice": joint[..., h * d:2 * h * d].unflatten(-1, (h, d)),
        "odd slice": joint[..., 1:h * d + 1].unflatten(-1, (h, d)),
        "heads first": torch.randn((b, h, n, d), generator=gen, device=dev).to(dtype).transpose(1, 2),
        "expanded": torch.randn((1, n, 1, d), generator=gen, device=dev).to(dtype).expand(b, n, h, d),
        "column major": torch.randn((b, n, d, h), generator=gen, device=dev).to(dtype).transpose(-1, -2),
    }
    odd_pos = torch.randint(0, 90, (n, 5), generator=gen, device=dev, dtype=torch.int32)[:, 1:4]
    for name, x in rows.items():
        for p in (pos, odd_pos):
            want, size = _plain(x, p, axes, "half", w)
            _close(htrc_b200.rotary_axes(x, p, axes=axes, pairs="half", weight=w), want, size)
            dy = torch.randn(x.shape, generator=gen, device=dev).to(dtype)
            dx, dw = htrc_b200.rotary_axes_backward(dy, x, p, axes=axes, pairs="half", weight=w)
            want, size, want_w, size_w = _plain_backward(dy, x, p, axes, "half", w)
            _close(dx, want, size)
            _close(dw, want_w, size_w)


def test_what_is_not_rotated_is_not_touched(dev):
    """NaN and infinities past the rotated width stay where they are; a NaN stays in its own row."""
    import htrc_b200
    x = torch.randn((5, 2, 40), device=dev)
    x[1, 0, 39], x[2, 1, 38] = float("inf"), float("nan")
    pos = torch.arange(5, device=dev)[:, None].int() + 3
    for pairs in ("interleaved", "half"):
        y = htrc_b200.rotary_axes(x, pos, axes=(16,), pairs=pairs)
        assert torch.equal(y[..., 16:].nan_to_num(7.0), x[..., 16:].nan_to_num(7.0))
        assert torch.isfinite(y[..., :16]).all()
    x = torch.randn((4, 3, 128), device=dev).bfloat16()
    x[2, 1, 5] = float("nan")
    y = htrc_b200.rotary_axes(x, pos[:4].expand(4, 3).contiguous(), axes=(44, 42, 42), weight=torch.ones(128, device=dev))
    bad = ~torch.isfinite(y).all(-1)
    assert bad[2, 1] and int(bad.sum()) == 1


def test_zero_rows_and_empty_inputs(dev):
    import htrc_b200
    w = torch.ones(64, device=dev)
    pos = torch.zeros((3, 1), dtype=torch.int32, device=dev)
    y = htrc_b200.rotary_axes(torch.zeros((3, 2, 64), device=dev), pos, axes=(64,), weight=w)
    assert torch.equal(y, torch.zeros_like(y))
    for shape in ((0, 2, 64), (2, 0, 2, 64), (0, 3, 2, 64)):
        x = torch.empty(shape, device=dev)
        p = torch.empty((*shape[:-2], 1), dtype=torch.int32, device=dev)
        assert htrc_b200.rotary_axes(x, p, axes=(64,), weight=w, heads_first=True).shape == (*shape[:-3], 2, shape[-3], 64)
        dx, dw = htrc_b200.rotary_axes_backward(x, x, p, axes=(64,), weight=w)
        assert dx.shape == x.shape and torch.equal(dw, torch.zeros_like(w))


def test_gradients_against_differences(dev):
    """Autograd through both tensors and their weights against central differences of the float64 forward."""
    import htrc_b200
    gen = torch.Generator(device=dev).manual_seed(9)
    axes, pairs = (6, 4, 4), "half"
    q = torch.randn((1, 7, 2, 16), generator=gen, device=dev)
    k = torch.randn((1, 7, 1, 16), generator=gen, device=dev)
    wq, wk = (1 + 0.2 * torch.randn(16, generator=gen, device=dev) for _ in range(2))
    pos = torch.randint(0, 50, (7, 3), generator=gen, device=dev, dtype=torch.int32)
    leaves = [t.clone().requires_grad_() for t in (q, k, wq, wk)]
    yq, yk = htrc_b200.rotary_qk(leaves[0], leaves[1], pos, axes=axes, pairs=pairs, q_weight=leaves[2],
                                 k_weight=leaves[3], heads_first=True)
    cq, ck = (torch.randn(y.shape, generator=gen, device=dev) for y in (yq, yk))
    grads = torch.autograd.grad((yq * cq).sum() + (yk * ck).sum(), leaves)

    def value(a, b, c, d):
        return sum((_plain(x, pos, axes, pairs, w)[0].transpose(1, 2) * g.double()).sum()
                   for x, w, g in ((a, c, cq), (b, d, ck)))

    for i, (x, g) in enumerate(zip((q, k, wq, wk), grads)):
        way = torch.randn(x.shape, generator=gen, device=dev, dtype=torch.float64)
        args = [t.double() for t in (q, k, wq, wk)]
        h = 1e-5
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + h * way, args[i] - h * way
        want = (value(*up) - value(*down)) / (2 * h)
        # float32 gradients of at most a few hundred terms of order one; the differences' own error is order h^2
        assert abs(float((g.double() * way).sum() - want)) <= 1e-4 * float(way.abs().sum()) ** 0.5 + 1e-6


def test_one_result_whatever_the_stream_or_the_run(dev):
    import htrc_b200
    gen = torch.Generator(device=dev).manual_seed(11)
    q = torch.randn((1, 3000, 6, 128), generator=gen, device=dev).bfloat16()
    pos = htrc_b200.grid_positions((3, 25, 40), start=(1, 0, 2), device=dev)
    assert pos.shape == (3000, 3) and pos[41].tolist() == [1, 1, 3]
    w = torch.rand(128, generator=gen, device=dev) + 0.5
    kw = dict(axes=(44, 42, 42), weight=w)
    y = htrc_b200.rotary_axes(q, pos, **kw)
    dx, dw = htrc_b200.rotary_axes_backward(y, q, pos, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y2 = htrc_b200.rotary_axes(q, pos, **kw)
        dx2, dw2 = htrc_b200.rotary_axes_backward(y2, q, pos, **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, y2) and torch.equal(dx, dx2) and torch.equal(dw, dw2)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y3 = htrc_b200.rotary_axes(q, pos, **kw)
        dx3, dw3 = htrc_b200.rotary_axes_backward(y3, q, pos, **kw)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, y3) and torch.equal(dx, dx3) and torch.equal(dw, dw3)


def test_refusals(dev):
    import htrc_b200
    x = torch.randn((4, 2, 64), device=dev)
    pos = torch.zeros((4, 2), dtype=torch.int32, device=dev)
    f = htrc_b200.rotary_axes
    for kw in (dict(axes=(3, 4)), dict(axes=(64, 2)), dict(axes=()), dict(axes=(4, 4), pairs="both"), dict(axes=(4, 4), theta=0.0),
               dict(axes=(4, 4), eps=-1.0), dict(axes=(4, 4), freqs=[1.0]), dict(axes=(4, 4, 4)), dict(axes=(-2, 4)),
               dict(axes=(4, 4), weight=torch.ones(63, device=dev)), dict(axes=(4, 4), weight=torch.ones(64))):
        with pytest.raises(ValueError):
            f(x, pos, **kw)
    for bad in (pos[:3], pos.cpu(), pos[:, :1], pos.bool(), None):
        with pytest.raises(ValueError):
            f(x, bad, axes=(4, 4))
    with pytest.raises(ValueError):
        f(x.cpu(), pos.cpu(), axes=(4, 4))
    with pytest.raises(ValueError):
        f(x.double(), pos, axes=(4, 4))
    with pytest.raises(ValueError):
        f(x[0], pos, axes=(4, 4))
    with pytest.raises(NotImplementedError):
        f(torch.randn((4, 1, 264), device=dev), pos, axes=(4, 4))
    with pytest.raises(ValueError):
        htrc_b200.rotary_qk(x, x.bfloat16(), pos, axes=(4, 4))
    with pytest.raises(ValueError):
        htrc_b200.rotary_qk(x, x[:3], pos, axes=(4, 4))
    with pytest.raises(ValueError):
        htrc_b200.rotary_axes_backward(x, x, pos, axes=(4, 4), heads_first=True)
    assert math.isfinite(float(f(x, pos, axes=(4, 4)).sum()))
