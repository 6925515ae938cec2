"""Cross attention (htrc_b200.cross_attention and its backward) against a float64 implementation.

Bounds, derived before the first run, with u the unit roundoff of the operands' type (2^-8 bfloat16, 2^-11 float16):
the weights p enter the second product rounded to u, everything else is float32, the result is rounded once, so
  |out - exact| <= u |out| + (u + f) sum_j p_j |v_j|.
f covers float32: a logit of up to 128 products, the exponential, the sums (2^-12 is more than 16 times their worst).
With a_i = sum_d |dout out| (delta is formed from the rounded out: an error of u a_i) and e_ij = p_ij (|dP_ij| + a_i):
  dv: u |dv| + (u + f) sum_i p_ij |dout_i|
  dq: u |dq| + scale sum_j ((u + f) |dS_ij| + (u + f) p_ij a_i + f e_ij) |k_j|,   dk: the same over i with |q_i|.
(u enters twice: dS rounded, and delta.)  float16 adds its subnormal spacing 2^-25 for each rounded value."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F = 2.0 ** -12


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda:0")


def _keep_and_bias(shape, lengths, mask, dev):
    b, h, n, m = shape
    keep = torch.ones(shape, dtype=torch.bool, device=dev)
    bias = torch.zeros(shape, dtype=torch.float64, device=dev)
    if lengths is not None:
        keep &= torch.arange(m, device=dev) < lengths.to(dev).view(b, 1, 1, 1)
    if mask is not None and mask.dtype == torch.bool:
        keep &= mask
    elif mask is not None:
        bias = bias + mask.double()
        keep &= bias != -math.inf
    return keep, bias


class Plain:
    """Forward and backward in float64, head-major, from the definition; excluded keys and values are never used."""

    def __init__(self, q, k, v, lengths=None, mask=None, scale=None):
        dev = q.device
        self.q, self.k, self.v = (x.double() for x in (q, k, v))
        self.group = q.shape[1] // k.shape[1]
        self.scale = scale or q.shape[-1] ** -0.5
        shape = (q.shape[0], q.shape[1], q.shape[2], k.shape[2])
        keep, bias = _keep_and_bias(shape, lengths, mask, dev)
        used = keep.unflatten(1, (k.shape[1], self.group)).any(2).any(2)[..., None]      # keys that any query sees
        self.k, self.v = torch.where(used, self.k, 0.0), torch.where(used, self.v, 0.0)
        self.K, self.V = (x.repeat_interleave(self.group, 1) for x in (self.k, self.v))
        s = torch.where(keep, self.q @ self.K.mT * self.scale + bias, -math.inf)
        top = s.amax(-1, keepdim=True) if shape[3] else s.new_full((*shape[:3], 1), -math.inf)
        e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        total = e.sum(-1, keepdim=True)
        self.p = e / torch.where(total == 0, 1.0, total)
        self.lse = (top + total.log())[..., 0]
        self.out = self.p @ self.V
        self.out_bound = self.p @ self.V.abs()
        self.s = torch.where(s == -math.inf, 0.0, s)

    def backward(self, do, dlse=None):
        do = do.double()
        dp = do @ self.V.mT
        delta = (do * self.out).sum(-1, keepdim=True)
        a = (do * self.out).abs().sum(-1, keepdim=True)
        if dlse is not None:
            delta = delta - dlse.double()[..., None]
        ds = self.p * (dp - delta)
        fold = lambda x: x.unflatten(1, (-1, self.group)).sum(2)  # noqa: E731
        g = (ds @ self.K * self.scale, fold(ds.mT @ self.q) * self.scale, fold(self.p.mT @ do))
        return g, ds.abs(), self.p * a, self.p * (dp.abs() + delta.abs() + a), do, fold

    def backward_bounds(self, do, dlse, u):
        g, ds, pa, e, do, fold = self.backward(do, dlse)
        t = (u + F) * ds + (u + F) * pa + F * e
        return g, (u * g[0].abs() + self.scale * (t @ self.K.abs()),
                   u * g[1].abs() + self.scale * fold(t.mT @ self.q.abs()),
                   u * g[2].abs() + (u + F) * fold(self.p.mT @ do.abs()))


def _within(got, want, bound, what=""):
    assert torch.isfinite(got).all(), what
    tiny = 2.0 ** -25 * (1 + got.shape[-2]) if got.dtype == torch.float16 else 1e-30
    over = (got.double() - want).abs() - bound - tiny
    assert (over <= 0).all(), (what, float(over.max()))


def _check(q, k, v, *, lengths=None, mask=None, scale=None, heads_first=True, backward=True, with_dlse=False, seed=0):
    """q, k, v head-major; runs the operator in either order."""
    import htrc_b200
    major = (lambda x: x) if heads_first else (lambda x: x.transpose(1, 2))
    kw = dict(key_lengths=lengths, mask=mask, scale=scale, heads_first=heads_first)
    args = [major(x) for x in (q, k, v)]
    out, lse = htrc_b200.cross_attention(*args, return_lse=True, **kw)
    ref = Plain(q, k, v, lengths, mask, scale)
    u = U[q.dtype]
    assert out.shape == args[0].shape and out.dtype == q.dtype and lse.shape == q.shape[:3]
    _within(major(out), ref.out, u * ref.out.abs() + (u + F) * ref.out_bound, "out")
    empty = ref.lse == -math.inf
    assert torch.equal(empty, lse == -math.inf)
    assert (major(out)[empty] == 0).all()
    # float32 sums of logits: their size times a few roundings
    top = ref.s.abs().amax(-1) if ref.s.shape[-1] else torch.zeros_like(ref.lse)
    lerr = (lse.double() - ref.lse).abs()
    assert (torch.where(empty, 0.0, lerr) <= 2.0 ** -18 * (1 + top)).all(), float(torch.where(empty, 0.0, lerr).max())
    if backward:
        gen = torch.Generator(device=q.device).manual_seed(seed + 1)
        do = torch.randn(q.shape, generator=gen, device=q.device).to(q.dtype)
        dlse = torch.randn(lse.shape, generator=gen, device=q.device) if with_dlse else None
        got = htrc_b200.cross_attention_backward(major(do).contiguous(), *args, out, lse, dlse=dlse, **kw)
        want, bounds = ref.backward_bounds(do, dlse, u)
        for name, g, w, bnd in zip(("dq", "dk", "dv"), got, want, bounds):
            _within(major(g), w, bnd, name)
    htrc_b200.cross_status()
    return out, lse


def _rows(dev, b, n, m, hq, hk, d, dtype, seed=0, spread=2.0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    q = (torch.randn((b, hq, n, d), generator=gen, device=dev) * spread).to(dtype)
    k, v = (torch.randn((b, hk, m, d), generator=gen, device=dev).to(dtype) for _ in range(2))
    return q, k, v


# batch, queries, keys, heads, key heads, dim: around the tiles' edges, one of each, shared heads, every dim rule
SIZES = [(1, 1, 1, 1, 1, 128), (2, 128, 128, 2, 2, 128), (1, 129, 127, 2, 1, 128), (2, 77, 65, 4, 2, 64), (1, 300, 257, 3, 1, 72),
         (1, 64, 640, 2, 2, 8), (3, 5, 200, 6, 2, 128), (1, 1, 1000, 8, 2, 128), (2, 2, 513, 4, 4, 64), (1, 1000, 33, 1, 1, 96),
         (1, 3, 4100, 2, 1, 40), (2, 1, 77, 12, 4, 64), (1, 4, 300, 8, 8, 128), (1, 16, 129, 2, 2, 32),
         (3, 40, 50, 1, 1, 64), (4, 1, 90, 1, 1, 128)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", SIZES)
def test_sizes_match_float64(dev, dtype, size):
    q, k, v = _rows(dev, *size, dtype, seed=sum(size))
    _check(q, k, v, heads_first=size[1] % 2 == 0, with_dlse=size[2] % 2 == 0)


# more units than SMs (each CTA walks several), keys split over CTAs, more entries than one pass of the lengths' sums
MANY = [(40, 300, 150, 6, 3, 64), (7, 700, 390, 16, 16, 128), (230, 1, 70, 4, 2, 64), (260, 3, 130, 2, 1, 128),
        (300, 5, 90, 4, 4, 64), (100, 2, 200, 24, 12, 64), (30, 24, 150, 6, 6, 128), (20, 9, 333, 24, 8, 128),
        (3, 32, 4243, 1, 1, 72), (2, 200, 1500, 4, 2, 128), (1, 300, 400, 2, 2, 64),
        (2, 40, 9000, 2, 1, 64), (1, 130, 12000, 1, 1, 128), (2, 1, 30000, 4, 1, 128), (5, 4, 2000, 24, 8, 64)]


@pytest.mark.parametrize("kind", ["none", "lengths", "pairs", "bias"])
@pytest.mark.parametrize("size", MANY)
def test_many_units_and_dead_ones(dev, size, kind):
    b, n, m, h, hk, d = size
    q, k, v = _rows(dev, *size, torch.bfloat16, seed=sum(size))
    gen = torch.Generator(device=dev).manual_seed(b + m)
    lengths = mask = None
    if kind != "none":
        lengths = torch.randint(0, m + 1, (b,), generator=gen, device=dev, dtype=torch.int32)
        lengths[b // 3] = 0                       # entries without a key, at the start, in the middle and at the end
        if b > 4:
            lengths[0] = lengths[b // 2] = lengths[b // 2 + 1] = lengths[-1] = 0
    if kind == "pairs":
        mask = torch.rand((b, 1, n, m), generator=gen, device=dev) < 0.5
        mask[:, :, ::5] = False
    elif kind == "bias":
        mask = torch.randn((1, h, n, m), generator=gen, device=dev)
    _check(q, k, v, lengths=lengths, mask=mask)


def _mask(kind, b, h, n, m, dtype, dev, seed=3):
    gen = torch.Generator(device=dev).manual_seed(seed)
    keys = torch.rand((b, 1, 1, m), generator=gen, device=dev) < 0.6
    pairs = torch.rand((b, 1, n, m), generator=gen, device=dev) < 0.5
    pairs[:, :, ::7] = False                                  # rows with nothing left
    noise = torch.randn((b, h, n, m), generator=gen, device=dev)
    if kind == "lengths":
        return torch.arange(b, device=dev) * (m + 3) // max(1, b - 1), None        # 0 .. beyond the keys
    if kind == "keys":
        return None, keys
    if kind == "keys of heads":
        return None, torch.rand((h, 1, m), generator=gen, device=dev) < 0.5
    if kind == "pairs":
        return None, pairs
    if kind == "pairs of a head":
        return None, noise > 0
    if kind == "shared pairs, transposed":
        return None, (noise[0, 0].mT.contiguous().mT > 0.3)
    if kind == "key bias":
        return None, torch.where(keys, noise[:, :1, :1], -math.inf)
    if kind == "lowest":
        low = torch.finfo(dtype).min
        return None, torch.where(keys, noise[:, :1, :1], low).to(dtype)
    if kind == "lowest rows":
        # entry 0 holds nothing but the lowest value: the softmax of equal logits; float32
        bias = torch.where(keys, noise[:, :1, :1], torch.finfo(torch.float32).min)
        bias[0] = torch.finfo(torch.float32).min
        return None, bias
    if kind == "bias":
        return None, torch.where(pairs, noise, -math.inf)
    if kind == "bias, lowest rows":
        bias = noise[:, :1].clone()
        bias[:, :, ::5] = torch.finfo(torch.float32).min
        return None, bias
    if kind == "keys and lengths":
        return torch.tensor([m // 2, m, 1][:b], device=dev, dtype=torch.int32), keys
    if kind == "pairs and lengths":
        return torch.tensor([m // 2, m, 0][:b], device=dev, dtype=torch.int32), pairs
    if kind == "none kept":
        return None, torch.zeros((m,), dtype=torch.bool, device=dev)
    raise AssertionError(kind)


MASKS = ["lengths", "keys", "keys of heads", "pairs", "pairs of a head", "shared pairs, transposed", "key bias", "lowest",
         "lowest rows", "bias", "bias, lowest rows", "keys and lengths", "pairs and lengths", "none kept"]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [(3, 150, 203, 4, 2, 128), (2, 130, 64, 2, 2, 64), (3, 1, 300, 4, 2, 128), (2, 2, 131, 2, 1, 72)])
@pytest.mark.parametrize("kind", MASKS)
def test_masks_match_float64(dev, dtype, size, kind):
    b, n, m, hq, hk, d = size
    lengths, mask = _mask(kind, b, hq, n, m, dtype, dev)
    q, k, v = _rows(dev, *size, dtype, seed=len(kind))
    _check(q, k, v, lengths=lengths, mask=mask, heads_first=len(kind) % 2 == 0)


@pytest.mark.parametrize("rows", [1, 2, 150])
@pytest.mark.parametrize("kind", ["lengths", "keys", "key bias"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_excluded_keys_may_hold_anything(dev, rows, kind, bad):
    import htrc_b200
    b, m, hq, hk, d = 3, 203, 4, 2, 128
    lengths, mask = _mask(kind, b, hq, rows, m, torch.bfloat16, dev)
    q, k, v = _rows(dev, b, rows, m, hq, hk, d, torch.bfloat16)
    keep, _ = _keep_and_bias((b, 1, 1, m), lengths, mask, dev)
    out = ~keep[:, :, 0, :, None].expand(k.shape)
    dirty_k, dirty_v = k.masked_fill(out, bad), v.masked_fill(out, bad)
    kw = dict(key_lengths=lengths, mask=mask, heads_first=True)
    clean = htrc_b200.cross_attention(q, k, v, return_lse=True, **kw)
    dirty = htrc_b200.cross_attention(q, dirty_k, dirty_v, return_lse=True, **kw)
    for x, y in zip(clean, dirty):
        assert torch.equal(x, y)
    do = torch.randn_like(q)
    want = htrc_b200.cross_attention_backward(do, q, k, v, *clean, **kw)
    got = htrc_b200.cross_attention_backward(do, q, dirty_k, dirty_v, *clean, **kw)
    for x, y in zip(want, got):
        assert torch.equal(x, y)
    assert (got[1][out] == 0).all() and (got[2][out] == 0).all()


def test_strides_alignment_and_broadcast(dev):
    """Slices of a joint projection, rows off the 16-byte grid, one prompt for a whole batch, one head for all."""
    gen = torch.Generator(device=dev).manual_seed(2)
    b, n, m, h, d = 2, 140, 70, 4, 64
    wide = torch.randn((b, m, 2 * h * d + 8), generator=gen, device=dev).bfloat16()
    q = torch.randn((b, h, n, d), generator=gen, device=dev).bfloat16()
    k, v = (wide[..., i * h * d:(i + 1) * h * d].unflatten(-1, (h, d)).transpose(1, 2) for i in range(2))
    _check(q, k, v)
    odd = [wide[..., i * h * d + 1:(i + 1) * h * d + 1].unflatten(-1, (h, d)).transpose(1, 2) for i in range(2)]
    _check(q, *odd)
    one = [x[:1].expand(b, h, m, d) for x in (k, v)]
    _check(q, *one, heads_first=False)
    single = [x[:, :1].expand(b, h, m, d) for x in (k, v)]
    _check(q, *single)
    _check(q[:, :, :1].expand(b, h, 9, d), k[:, :, :1].expand(b, h, 5, d), v[:, :, :5])
    _check(q[:, :, ::2], k[:, :, 0:69:3], v[:, :, 1:70:3])


def test_empty_sides(dev):
    import htrc_b200
    for n, m in ((0, 5), (5, 0), (0, 0)):
        q, k, v = _rows(dev, 2, n, m, 2, 1, 64, torch.bfloat16)
        out, lse = htrc_b200.cross_attention(q, k, v, heads_first=True, return_lse=True)
        assert (out == 0).all() and (lse == -math.inf).all()
        grads = htrc_b200.cross_attention_backward(torch.randn_like(q), q, k, v, out, lse, heads_first=True)
        assert [g.shape for g in grads] == [q.shape, k.shape, v.shape] and all((g == 0).all() for g in grads)
    q = torch.empty((0, 4, 2, 64), device=dev, dtype=torch.bfloat16)
    assert htrc_b200.cross_attention(q, q, q).shape == q.shape


def test_large_logits_and_scale(dev):
    """A maximum that keeps growing along the keys (the running maximum's rescaling) and a caller's scale."""
    q, k, v = _rows(dev, 1, 200, 700, 2, 2, 128, torch.float16, spread=1.0)
    k = (k * torch.linspace(0.05, 3.0, 700, device=dev)[:, None]).half()
    _check(q, k, v, scale=0.7)
    _check(q, k, v, scale=3e-3)
    _check(q[:, :, :1], k, v, scale=0.7)


def test_gradients_against_differences(dev):
    """Autograd against central differences of the float64 forward, through shared heads and an expanded prompt."""
    import htrc_b200
    gen = torch.Generator(device=dev).manual_seed(4)
    b, n, m, hq, hk, d = 2, 20, 30, 4, 2, 16
    q = torch.randn((b, hq, n, d), generator=gen, device=dev).half()
    k, v = (torch.randn((1, hk, m, d), generator=gen, device=dev).half() for _ in range(2))
    mask = torch.rand((b, 1, n, m), generator=gen, device=dev) < 0.7
    co = torch.randn((b, hq, n, d), generator=gen, device=dev).half()
    cl = torch.randn((b, hq, n), generator=gen, device=dev)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    out, lse = htrc_b200.cross_attention(leaves[0], leaves[1].expand(b, -1, -1, -1), leaves[2].expand(b, -1, -1, -1),
                                         mask=mask, heads_first=True, return_lse=True)
    live = torch.isfinite(lse)
    grads = torch.autograd.grad((out.double() * co.double()).sum() + (torch.where(live, lse, 0.0) * cl).sum(), leaves)

    def value(q, k, v):
        r = Plain(q, k.expand(b, -1, -1, -1), v.expand(b, -1, -1, -1), None, mask)
        return (r.out * co.double()).sum() + (torch.where(live, r.lse, 0.0) * cl.double()).sum()

    ref = Plain(q, k.expand(b, -1, -1, -1), v.expand(b, -1, -1, -1), None, mask)
    _, bounds = ref.backward_bounds(co, torch.where(live, cl, 0.0), U[torch.float16])
    for i, (x, g, bound) in enumerate(zip((q, k, v), grads, bounds)):
        way = torch.randn(x.shape, generator=gen, device=dev, dtype=torch.float64)
        args = [t.double() for t in (q, k, v)]
        h = 1e-4
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + h * way, args[i] - h * way
        want = (value(*up) - value(*down)) / (2 * h)
        # the bound of the batch entries' sum, its own rounding, and the differences' h^2
        allowed = (bound if i == 0 else bound.sum(0, keepdim=True) + U[torch.float16] * g.double().abs()) * way.abs()
        assert abs(float((g.double() * way).sum() - want)) <= float(allowed.sum()) + 1e-5


def test_no_batch_dimension_and_order(dev):
    import htrc_b200
    q, k, v = _rows(dev, 1, 50, 40, 2, 2, 64, torch.bfloat16)
    a, la = htrc_b200.cross_attention(q, k, v, heads_first=True, return_lse=True)
    b, lb = htrc_b200.cross_attention(q[0], k[0], v[0], heads_first=True, return_lse=True)
    c = htrc_b200.cross_attention(q[0].transpose(0, 1), k[0].transpose(0, 1), v[0].transpose(0, 1))
    assert torch.equal(a[0], b) and torch.equal(la[0], lb) and torch.equal(c.transpose(0, 1), b)
    do = torch.randn_like(q)
    ga = htrc_b200.cross_attention_backward(do, q, k, v, a, la, heads_first=True)
    gb = htrc_b200.cross_attention_backward(do[0], q[0], k[0], v[0], b, lb, heads_first=True)
    assert all(torch.equal(x[0], y) for x, y in zip(ga, gb))
    for x in (q, k, v):
        x.requires_grad_()
    out = htrc_b200.cross_attention(q, k, v, heads_first=True)
    assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(out, (q, k, v), do), ga))


@pytest.mark.parametrize("size", [(2, 500, 300, 4, 2, 128), (3, 1, 3000, 4, 2, 128), (1, 3000, 200, 2, 2, 64),
                                  (2, 40, 5000, 2, 1, 128)])
def test_one_result_whatever_the_stream_or_the_run(dev, size):
    import htrc_b200
    q, k, v = _rows(dev, *size, torch.bfloat16)
    do = torch.randn_like(q)

    def both():
        out, lse = htrc_b200.cross_attention(q, k, v, heads_first=True, return_lse=True)
        return (out, lse, *htrc_b200.cross_attention_backward(do, q, k, v, out, lse, heads_first=True))

    first = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = both()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        third = both()
    g.replay()
    torch.cuda.synchronize()
    for other in (second, third):
        assert all(torch.equal(x, y) for x, y in zip(first, other))
    htrc_b200.cross_status()


def test_refusals(dev):
    import htrc_b200
    f = htrc_b200.cross_attention
    q, k, v = (x.transpose(1, 2) for x in _rows(dev, 2, 8, 6, 4, 2, 64, torch.bfloat16))
    with pytest.raises(NotImplementedError):
        f(q.float(), k.float(), v.float())
    with pytest.raises(NotImplementedError):
        f(q, k.half(), v)
    with pytest.raises(NotImplementedError):
        f(*(torch.zeros((1, 4, 1, 136), device=dev, dtype=torch.bfloat16),) * 3)
    with pytest.raises(NotImplementedError):
        f(q[..., :60], k[..., :60], v[..., :60])
    for bad in ((q, k[:1], v[:1]), (q, k, v[:, :5]), (q[:, :, :3], k, v), (q[0], k, v), (q.cpu(), k, v), (q, k[..., :32], v)):
        with pytest.raises(ValueError):
            f(*bad)
    for kw in (dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(key_lengths=torch.ones(3, device=dev).int()),
               dict(key_lengths=torch.ones(2, device=dev)), dict(key_lengths=torch.ones(2).int()),
               dict(mask=torch.ones((8, 5), device=dev).bool()), dict(mask=torch.ones((8, 6), device=dev).int()),
               dict(mask=torch.ones((1, 2, 4, 8, 6), device=dev).bool()), dict(mask=torch.ones((8, 6)).bool())):
        with pytest.raises(ValueError):
            f(q, k, v, **kw)
    out, lse = f(q, k, v, return_lse=True)
    back = htrc_b200.cross_attention_backward
    for args in ((out[:1], q, k, v, out, lse), (out, q, k, v, out.half(), lse), (out, q, k, v, out, lse[:, :1]),
                 (out, q, k, v, out, lse.double())):
        with pytest.raises(ValueError):
            back(*args)
    with pytest.raises(ValueError):
        back(out, q, k, v, out, lse, dlse=lse[..., :3])
    htrc_b200.cross_status()
