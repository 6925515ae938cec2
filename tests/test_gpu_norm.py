"""Layer norm (htrc_b200.layer_norm and its backward, layer_norm_int8, quantize_rows) against float64.

Bounds, derived before the first run; u is half a step of the result's type.  A float32 sum over a row adds at most 64
elements in a lane, 32 lanes in 5 steps and 16 warps: fewer than 2^7 roundings of 2^-24, so a row's mean is within
2^-17 mean|x|, and its variance within a relative 2^-16 plus the square of the mean's error.  The normalised element is
then within 2^-16 (|u| + rstd mean|x|), a result within 2^-15 of the same with its terms' sizes, before its own rounding.
Sums over rows add at most 2^7 rows in a thread of these sizes, 2^5 parts in a lane and 2^5 of those: the same 2^-15 of the
sum of magnitudes.  8-bit codes of a given row are exact; of a norm they are within half a step and 127 times the result's
error over the row's largest."""
from __future__ import annotations

import pytest
import torch

import htrc_b200

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
NOISE = 2.0 ** -15
TYPES = list(U)
EPS = 1e-6


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda:0")


def _w(t):
    return None if t is None else t.double()


def _terms(weight, bias, scale, shift, like):
    """A and B [batch, 1, width] of y = u A + B, and the size of B's parts."""
    one = torch.ones((1, 1, like.shape[-1]), dtype=torch.float64, device=like.device)
    w = one if weight is None else _w(weight)[None, None]
    b = 0 * one if bias is None else _w(bias)[None, None]
    s = one if scale is None else 1 + _w(scale).reshape(like.shape[0], 1, -1)
    t = 0 * one if shift is None else _w(shift).reshape(like.shape[0], 1, -1)
    return w * s, b * s + t, (b * s).abs() + t.abs(), w, b, s


def _plain(x, kw):
    """(y, its bound without the rounding, mean, rstd, u) in float64 of x [batch, tokens, width]."""
    x = _w(x)
    mean = x.mean(-1, keepdim=True)
    rstd = (x - mean).pow(2).mean(-1, keepdim=True).add(EPS).rsqrt()
    u = (x - mean) * rstd
    a, b, bs, *_ = _terms(*(kw.get(k) for k in ("weight", "bias", "scale", "shift")), x)
    off = NOISE * (a.abs() * (u.abs() + rstd * x.abs().mean(-1, keepdim=True)) + bs)
    return u * a + b, off, mean[..., 0], rstd[..., 0], u


def _close(got, want, off):
    assert torch.isfinite(got).all()
    err = (got.double() - want).abs()
    bound = U[got.dtype] * want.abs() + off + (2.0 ** -25 if got.dtype is torch.float16 else 0.0)
    assert (err <= bound).all(), float((err - bound).max())


def _params(gen, dev, terms, batch, width, dtype):
    def normal(*shape, dt, size):
        return (torch.randn(shape, generator=gen, device=dev) * size).to(dt)
    kw = {}
    if "w" in terms:
        kw["weight"] = normal(width, dt=torch.float32, size=0.5) + 1
    if "b" in terms:
        kw["bias"] = normal(width, dt=dtype, size=0.5)
    if "s" in terms:
        kw["scale"] = normal(batch, width, dt=dtype, size=0.3)
    if "t" in terms:
        kw["shift"] = normal(batch, 1, width, dt=torch.bfloat16, size=0.3)
    return kw


# single elements, odd widths, a lane's, a warp's and a CTA's pieces and one more or less, the widest
WIDTHS = [1, 2, 7, 8, 63, 64, 96, 257, 511, 768, 1001, 1024, 2040, 2048, 2056, 4100, 5120, 8192, 8200, 10007, 16384]
TERMS = ["", "wb", "st", "wbst", "w", "t", "bs"]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_forward_and_backward_match_float64(dev, dtype, width):
    gen = torch.Generator(device=dev).manual_seed(width)
    for i, (batch, tokens) in enumerate([(2, 37), (1, 1), (3, 9)]):
        terms = TERMS[(WIDTHS.index(width) + i) % len(TERMS)]
        kw = _params(gen, dev, terms, batch, width, dtype)
        x = (torch.randn((batch, tokens, width), generator=gen, device=dev) * 1.7 + 0.4).to(dtype)
        y, mean, rstd = htrc_b200.layer_norm(x, **kw, return_stats=True)
        want, off, m, r, _ = _plain(x, kw)
        assert y.is_contiguous() and y.dtype is dtype and mean.shape == x.shape[:-1]
        _close(y, want, off)
        spread = _w(x).abs().mean(-1)
        assert ((mean.double() - m).abs() <= NOISE * spread).all()
        assert ((rstd.double() - r).abs() <= r * (NOISE + (NOISE * spread * r) ** 2)).all()

        dy = torch.randn(x.shape, generator=gen, device=dev).to(dtype)
        got = htrc_b200.layer_norm_backward(dy, x, mean, rstd, **kw)
        _check_backward(got, dy, x, mean, rstd, kw)


def _check_backward(got, dy, x, mean, rstd, kw):
    """The formula on the statistics that the call got."""
    args = [kw.get(k) for k in ("weight", "bias", "scale", "shift")]
    a, _, _, w, b, s = _terms(*args, x)
    dy, x, r = dy.double(), x.double(), rstd.double()[..., None]
    u = (x - mean.double()[..., None]) * r
    g = dy * a
    gu = g * u
    dx = r * (g - g.mean(-1, keepdim=True) - u * gu.mean(-1, keepdim=True))
    _close(got[0], dx, NOISE * r * (g.abs() + g.abs().mean(-1, keepdim=True) + u.abs() * gu.abs().mean(-1, keepdim=True)))
    p, q, ps, qs = (dy * u).sum(1, True), dy.sum(1, True), (dy * u).abs().sum(1, True), dy.abs().sum(1, True)
    wants = [((p * s).sum((0, 1)), (ps * s.abs()).sum((0, 1))), ((q * s).sum((0, 1)), (qs * s.abs()).sum((0, 1))),
             (p * w + q * b, ps * w.abs() + qs * b.abs()), (q, qs)]
    for t, d, (want, size) in zip(args, got[1:], wants):
        if t is None:
            assert d is None
            continue
        assert d.shape == t.shape and d.dtype is t.dtype
        _close(d, want.expand(*want.shape[:-1], want.shape[-1]).reshape(t.shape), NOISE * size.reshape(t.shape))


@pytest.mark.parametrize("dtype", TYPES)
def test_many_rows(dev, dtype):
    """Every chunk and part, a last chunk that is short, entries that share CTAs or have several."""
    gen = torch.Generator(device=dev).manual_seed(3)
    for batch, tokens, width, terms in [(1, 5003, 256, "wb"), (2, 2501, 320, "wbst"), (700, 3, 64, "st"), (1, 1, 512, "wbst"),
                                        (9000, 1, 40, "wb"), (5, 0, 64, "wbst"), (0, 4, 64, "wb")]:
        kw = _params(gen, dev, terms, batch, width, dtype)
        x = torch.randn((batch, tokens, width), generator=gen, device=dev).to(dtype)
        y, mean, rstd = htrc_b200.layer_norm(x, **kw, return_stats=True)
        want, off, *_ = _plain(x, kw)
        _close(y, want, off)
        dy = torch.randn(x.shape, generator=gen, device=dev).to(dtype)
        _check_backward(htrc_b200.layer_norm_backward(dy, x, mean, rstd, **kw), dy, x, mean, rstd, kw)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_shapes(dev, dtype):
    gen = torch.Generator(device=dev).manual_seed(5)
    big = torch.randn((3, 11, 5, 200), generator=gen, device=dev).to(dtype)
    kw = _params(gen, dev, "wb", 1, 64, dtype)
    views = [big[..., 8:72], big[..., 3:67], big[:, ::2, 1, :64], big[1, :, :, 64:128], big[0, 0, 0, 5:69],
             big.transpose(0, 2)[..., 100:164], big[:, :1, 0, :64].expand(3, 6, 64), big[:, :, 0, 0:128:2],
             big.permute(3, 0, 1, 2)[:, 0, 0, :][100:].T.contiguous()[..., :64]]
    for x in views:
        y, mean, rstd = htrc_b200.layer_norm(x, **kw, return_stats=True)
        flat = x.reshape(1, -1, 64)
        want, off, *_ = _plain(flat, kw)
        assert y.shape == x.shape and mean.shape == x.shape[:-1]
        _close(y.reshape(1, -1, 64), want, off)
        wide = torch.randn((*x.shape[:-1], 130), generator=gen, device=dev).to(dtype)
        dy = wide[..., 66:]
        got = htrc_b200.layer_norm_backward(dy, x, mean, rstd, **kw)
        _check_backward((got[0].reshape(1, -1, 64), *got[1:]), dy.reshape(1, -1, 64), flat, mean.reshape(1, -1),
                        rstd.reshape(1, -1), kw)
    # a modulation from a joint projection, for rows with more dimensions than two; and one for all rows
    joint = (torch.randn((3, 6 * 64), generator=gen, device=dev) * 0.2).to(dtype)
    scale, shift = joint.chunk(6, -1)[1], joint.chunk(6, -1)[4]
    x = big[..., 8:72]
    y = htrc_b200.layer_norm(x, scale=scale, shift=shift)
    want, off, *_ = _plain(x.reshape(3, -1, 64), dict(scale=scale, shift=shift))
    _close(y.reshape(3, -1, 64), want, off)
    y = htrc_b200.layer_norm(x[0, 0], scale=scale[0], shift=shift[:1].expand(1, 64)[0])
    want, off, *_ = _plain(x[0, :1], dict(scale=scale[:1], shift=shift[:1]))
    _close(y[None], want, off)


def test_repeated_calls_with_other_alignments_and_modulated_dimensions(dev):
    """What a call keeps for the next goes by shapes, strides and types: pointers of other alignments are read as they are."""
    gen = torch.Generator(device=dev).manual_seed(12)
    for dtype in TYPES:
        room = torch.randn(2 * 3 * 5 * 72 + 64, generator=gen, device=dev).to(dtype)
        kw = _params(gen, dev, "wbst", 2, 64, dtype)
        kw["shift"] = kw["shift"][:, 0]
        for start in (0, 8, 0, 1, 2, 8):
            x = room[start:].as_strided((2, 3, 5, 64), (3 * 5 * 72, 5 * 72, 72, 1))
            for _ in range(2):
                y, mean, rstd = htrc_b200.layer_norm(x, **kw, return_stats=True)
                flat = x.reshape(2, 15, 64)
                want, off, *_ = _plain(flat, kw)
                _close(y.reshape(2, 15, 64), want, off)
                dy = torch.randn((2, 3, 5, 80), generator=gen, device=dev).to(dtype)[..., start:start + 64]
                got = htrc_b200.layer_norm_backward(dy, x, mean, rstd, **kw)
                _check_backward((got[0].reshape(2, 15, 64), *got[1:]), dy.reshape(2, 15, 64), flat, mean.reshape(2, 15),
                                rstd.reshape(2, 15), kw)
                rows = htrc_b200.quantize_rows(x)
                assert torch.equal(rows.codes.double(), _codes(x)[0])


def test_large_offset_and_constant_rows(dev):
    """A mean far above the deviations loses no more than its own rounding; a constant row gives the shift."""
    gen = torch.Generator(device=dev).manual_seed(6)
    x = torch.randn((1, 8, 1024), generator=gen, device=dev) + 1000.0
    want, off, *_ = _plain(x, {})
    _close(htrc_b200.layer_norm(x), want, off)
    for dtype in TYPES:
        x = torch.full((1, 3, 512), 2.5, dtype=dtype, device=dev)
        shift = torch.arange(512, device=dev).to(dtype)[None]
        assert torch.equal(htrc_b200.layer_norm(x, shift=shift), shift[:, None].expand(1, 3, 512))


def test_bad_values_stay_in_their_rows(dev):
    for width in (1024, 1001):
        x = torch.ones((6, width), device=dev).bfloat16()
        x += torch.arange(width, device=dev) % 3
        x[1, 5] = float("nan")
        x[4, -1] = float("inf")
        y = htrc_b200.layer_norm(x)
        assert torch.isnan(y[1]).all() and torch.isnan(y[4]).all() and torch.isfinite(y[[0, 2, 3, 5]]).all()
        for rows in (htrc_b200.layer_norm_int8(x), htrc_b200.quantize_rows(x)):
            assert torch.isnan(rows.scales[[1, 4]]).all() and torch.isfinite(rows.scales[[0, 2, 3, 5]]).all()


def _codes(x):
    """The definition, each rounding to float32 by itself: codes and scales of x [.., width]."""
    x = x.double()
    top = x.abs().amax(-1).clamp_min(1e-30).float().double()
    by = (127.0 / top).float().double()
    return torch.round((x * by[..., None]).float().double()), top / 127.0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_quantized_rows_are_exact(dev, dtype, width):
    gen = torch.Generator(device=dev).manual_seed(width)
    x = torch.randn((3, 29, width), generator=gen, device=dev)
    x = (x * torch.logspace(-18, 4, 29, device=dev)[:, None]).to(dtype)
    x[0, 3] = 0
    x[1, 2] = -x[1, 2].abs()
    for rows in (x, x[:, ::3], x[..., width // 3:], x[2, 5]):
        if rows.shape[-1] == 0:
            continue
        got = htrc_b200.quantize_rows(rows)
        codes, scales = _codes(rows)
        assert got.codes.shape == rows.shape and torch.equal(got.codes.double(), codes)
        assert ((got.scales.double() - scales).abs() <= 2.0 ** -24 * scales).all()


def test_quantized_halves_round_to_even(dev):
    x = torch.arange(-127, 128, device=dev).float()
    x = torch.cat([x, x[:-1] + 0.5])
    assert torch.equal(htrc_b200.quantize_rows(x).codes.float(), torch.round(x))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_norm_in_8_bits(dev, dtype, width):
    gen = torch.Generator(device=dev).manual_seed(width + 1)
    for i, (batch, tokens) in enumerate([(2, 21), (1, 1)]):
        kw = _params(gen, dev, TERMS[(WIDTHS.index(width) + i + 2) % len(TERMS)], batch, width, dtype)
        x = (torch.randn((batch, tokens, width), generator=gen, device=dev) * 2 + 0.3).to(dtype)
        rows = htrc_b200.layer_norm_int8(x, **kw)
        want, off, *_ = _plain(x, kw)
        top = want.abs().amax(-1).clamp_min(1e-30)
        worst = off.amax(-1)
        # at a width of one, without a bias or shift, the result itself is nothing but rounding
        sure = top > 8 * worst
        assert ((rows.scales.double() * 127 - top).abs() <= worst + 2.0 ** -22 * top)[sure].all()
        z = want * (127 / top)[..., None]
        slack = 127 * (off + worst[..., None]) / top[..., None] + 127 * 2.0 ** -22
        assert ((rows.codes.double() - z).abs() <= 0.5 + slack)[sure].all()
        assert rows.codes.abs().amax() <= 127


def test_autograd(dev):
    gen = torch.Generator(device=dev).manual_seed(8)
    x = torch.randn((2, 19, 320), generator=gen, device=dev).bfloat16()
    kw = _params(gen, dev, "wbst", 2, 320, torch.bfloat16)
    leaves = [t.detach().clone().requires_grad_() for t in (x, *kw.values())]
    kw2 = dict(zip(kw, leaves[1:]))
    y, mean, rstd = htrc_b200.layer_norm(leaves[0], **kw2, return_stats=True)
    assert not mean.requires_grad and not rstd.requires_grad
    dy = torch.randn(y.shape, generator=gen, device=dev).bfloat16()
    y.backward(dy)
    want = htrc_b200.layer_norm_backward(dy, x, mean, rstd, **kw)
    for leaf, w in zip(leaves, want):
        assert torch.equal(leaf.grad, w)
    # only what is asked for; a frozen weight gets none
    y = htrc_b200.layer_norm(leaves[0], weight=kw["weight"], scale=leaves[3])
    (gx,) = torch.autograd.grad(y, leaves[0], dy)
    assert torch.equal(gx, htrc_b200.layer_norm_backward(dy, x, mean, rstd, weight=kw["weight"], scale=kw["scale"])[0])
    # a modulation shared by the batch: its gradient is summed outside
    one = kw["scale"][:1].detach().clone().requires_grad_()
    y = htrc_b200.layer_norm(x, scale=one.expand(2, -1))
    y.backward(dy)
    both = htrc_b200.layer_norm_backward(dy, x, mean, rstd, scale=one.detach().expand(2, -1))[3]
    assert torch.equal(one.grad, both.sum(0, keepdim=True))


def test_gradient_against_differences(dev):
    """Directional differences of float32 calls: the step h leaves h^2 / 6 of the third derivative and 2^-24 |y| / h of
    rounding per element; both are far below 1 % of the directional derivative at h = 2^-6 and unit sizes."""
    gen = torch.Generator(device=dev).manual_seed(9)
    x = torch.randn((2, 5, 96), generator=gen, device=dev)
    kw = _params(gen, dev, "wbst", 2, 96, torch.float32)
    kw["shift"] = kw["shift"].float()
    dy = torch.randn(x.shape, generator=gen, device=dev)
    _, mean, rstd = htrc_b200.layer_norm(x, **kw, return_stats=True)
    grads = htrc_b200.layer_norm_backward(dy, x, mean, rstd, **kw)
    given = [x, *kw.values()]
    for i, g in enumerate(grads):
        d = torch.randn(given[i].shape, generator=gen, device=dev)
        h = 2.0 ** -6

        def at(sign):
            moved = list(given)
            moved[i] = given[i] + sign * h * d
            y = htrc_b200.layer_norm(moved[0], **dict(zip(kw, moved[1:])))
            return (y.double() * dy.double()).sum()
        num, ana = float((at(1) - at(-1)) / (2 * h)), float((g.double() * d.double()).sum())
        assert abs(num - ana) <= 0.01 * float((g.double().norm() * d.double().norm())), (i, num, ana)


def test_derivatives_that_are_refused(dev):
    x = torch.randn((2, 3, 64), device=dev).requires_grad_()
    (g,) = torch.autograd.grad(htrc_b200.layer_norm(x).sum(), x, create_graph=True)
    with pytest.raises(NotImplementedError, match="second"):
        g.sum().backward()
    with torch.autograd.forward_ad.dual_level(), pytest.raises((NotImplementedError, RuntimeError)):
        htrc_b200.layer_norm(torch.autograd.forward_ad.make_dual(x.detach(), x.detach()))
    for call in (htrc_b200.layer_norm_int8, htrc_b200.quantize_rows):
        with pytest.raises(NotImplementedError, match="gradients"):
            call(x)
        with torch.no_grad():
            call(x)


def test_streams_and_graphs(dev):
    gen = torch.Generator(device=dev).manual_seed(10)
    x = torch.randn((2, 300, 512), generator=gen, device=dev).half()
    dy = torch.randn(x.shape, generator=gen, device=dev).half()
    kw = _params(gen, dev, "wbst", 2, 512, torch.float16)

    def step():
        y, mean, rstd = htrc_b200.layer_norm(x, **kw, return_stats=True)
        return (y, *htrc_b200.layer_norm_backward(dy, x, mean, rstd, **kw), *htrc_b200.layer_norm_int8(x, **kw))
    want = step()
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    x0 = x.clone()
    for k in range(2):
        x.copy_(x0 if k else torch.randn_like(x0))
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_empty_batches_and_broadcast_gradients(dev):
    gen = torch.Generator(device=dev).manual_seed(14)
    for shape in ((0, 4, 96), (3, 0, 96), (0, 96)):
        x = torch.empty(shape, device=dev)
        kw = _params(gen, dev, "wb" if len(shape) == 2 else "wbst", shape[0], 96, torch.float32)
        y, mean, rstd = htrc_b200.layer_norm(x, **kw, return_stats=True)
        assert y.shape == x.shape and mean.shape == rstd.shape == x.shape[:-1]
        dx, *grads = htrc_b200.layer_norm_backward(y, x, mean, rstd, **kw)
        assert dx.shape == x.shape and all(g is None or (g == 0).all() for g in grads)
        assert htrc_b200.layer_norm_int8(x, **kw).codes.shape == htrc_b200.quantize_rows(x).codes.shape == x.shape
    # an upstream gradient that is one value, and one that is the same row for all tokens
    x = torch.randn((2, 70, 520), generator=gen, device=dev).bfloat16().requires_grad_()
    row = torch.randn(520, generator=gen, device=dev).bfloat16()
    for dy in (torch.ones((), device=dev).bfloat16().expand(2, 70, 520), row.expand(2, 70, 520)):
        y, mean, rstd = htrc_b200.layer_norm(x, return_stats=True)
        (g,) = torch.autograd.grad(y, x, dy)
        _check_backward((g, None, None, None, None), dy, x.detach(), mean, rstd, {})


def test_offsets_past_32_bits(dev):
    gen = torch.Generator(device=dev).manual_seed(15)
    x = torch.randn((1, 140000, 16384), generator=gen, device=dev, dtype=torch.bfloat16)
    y, mean, rstd = htrc_b200.layer_norm(x, return_stats=True)
    dx = htrc_b200.layer_norm_backward(y, x, mean, rstd)[0]
    for a in (0, 131060, 139990):
        some = slice(a, a + 10)
        want, off, *_ = _plain(x[:, some], {})
        _close(y[:, some], want, off)
        _check_backward((dx[:, some], None, None, None, None), y[:, some], x[:, some], mean[:, some], rstd[:, some], {})


def test_calls_on_two_streams_at_once(dev):
    gen = torch.Generator(device=dev).manual_seed(16)
    cases = []
    for width in (2048, 768, 1001, 128):
        x = torch.randn((2, 900, width), generator=gen, device=dev).bfloat16()
        cases.append((x, torch.randn(x.shape, generator=gen, device=dev).bfloat16(),
                      _params(gen, dev, "wbst", 2, width, torch.bfloat16)))

    def step(x, dy, kw):
        y, mean, rstd = htrc_b200.layer_norm(x, **kw, return_stats=True)
        return (y, *htrc_b200.layer_norm_backward(dy, x, mean, rstd, **kw), *htrc_b200.layer_norm_int8(x, **kw))
    want = [step(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    got = []
    for k in range(3):
        for i, c in enumerate(cases):
            with torch.cuda.stream(streams[(i + k) % 2]):
                got.append((i, step(*c)))
    torch.cuda.synchronize()
    for i, g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want[i]))


def test_refusals(dev):
    x = torch.zeros((2, 3, 64), device=dev)
    w = torch.ones(64, device=dev)
    bad = [dict(weight=w[:63]), dict(bias=w.double()), dict(weight=w.cpu()), dict(scale=w), dict(scale=w.expand(3, 64)),
           dict(shift=w.expand(2, 3, 64)), dict(eps=-1.0), dict(eps=float("nan"))]
    for kw in bad:
        for call in (htrc_b200.layer_norm, htrc_b200.layer_norm_int8):
            with pytest.raises(ValueError):
                call(x, **kw)
    with pytest.raises(ValueError):
        htrc_b200.layer_norm(x.double())
    with pytest.raises(ValueError):
        htrc_b200.quantize_rows(x.int())
    for call in (htrc_b200.layer_norm, htrc_b200.layer_norm_int8, htrc_b200.quantize_rows):
        with pytest.raises(NotImplementedError):
            call(torch.zeros((2, 16385), device=dev))
        with pytest.raises(ValueError):
            call(torch.zeros((2, 0), device=dev))
    y, mean, rstd = htrc_b200.layer_norm(x, return_stats=True)
    for args in ((y.half(), x, mean, rstd), (y[:1], x, mean, rstd), (y, x, mean[:1], rstd), (y, x, mean, rstd.half())):
        with pytest.raises(ValueError):
            htrc_b200.layer_norm_backward(*args)
