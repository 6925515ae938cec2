"""The 8-bit product (htrc_b200.int8_linear) against float64.

Bound, derived before the first run: the sum is an exact integer; its conversion, two products and the bias's sum round to
float32 (below 2^-22 of the parts' sizes together), and the result once to its type (u, half a step of it)."""
from __future__ import annotations

import pytest
import torch

import htrc_b200
from htrc_b200 import Int8Rows, _lib
from htrc_b200.linear8 import _DTYPES

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TYPES = list(U)


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda:0")


def _rows(gen, dev, *shape, low=-127):
    """Rows of arbitrary codes."""
    codes = torch.randint(low, 128, shape, generator=gen, device=dev, dtype=torch.int8)
    return Int8Rows(codes, torch.rand(shape[:-1], generator=gen, device=dev) * 0.02 + 0.001)


def _check(got, x, w, bias, dtype):
    parts = (x.codes.double() @ w.codes.double().T) * x.scales.double()[..., None] * w.scales.double()
    want = parts if bias is None else parts + bias.double()
    size = parts.abs() + (0 if bias is None else bias.double().abs())
    assert got.shape == want.shape and got.dtype is dtype and got.is_contiguous()
    assert torch.isfinite(got).all() or not got.numel()
    err = (got.double() - want).abs()
    bound = U[dtype] * want.abs() + 2.0 ** -22 * size + (2.0 ** -25 if dtype is torch.float16 else 0.0)
    assert (err <= bound).all(), float((err - bound).max())


# tokens, width, channels: single ones, tiles and one more or less in every direction, widths that end inside 16 and 128
# bytes, tiles that are split over the width, several tiles
SIZES = [(1, 1, 1), (1, 2048, 515), (2, 16, 128), (15, 17, 127), (16, 128, 129), (17, 129, 300), (32, 4100, 64), (33, 255, 2),
         (64, 1000, 1000), (65, 777, 515), (128, 512, 256), (129, 130, 130), (255, 384, 1023), (256, 64, 256), (300, 2048, 2048),
         (1001, 777, 515), (513, 4096, 384), (2049, 96, 1025), (7, 16384, 40), (5, 65536, 33),
         # pairs of SMs: several tiles each, ends in every direction, rows that are not 16-byte aligned
         (5000, 384, 1100), (2049, 96, 2308), (3001, 777, 2051), (19000, 130, 304), (300, 1000, 20000), (4096, 2048, 4096)]


@pytest.mark.parametrize("size", SIZES)
def test_codes_match_float64(dev, size):
    tokens, width, channels = size
    gen = torch.Generator(device=dev).manual_seed(sum(size))
    x, w = _rows(gen, dev, tokens, width, low=-128), _rows(gen, dev, channels, width, low=-128)
    for dtype, kind in zip(TYPES, (torch.float32, None, torch.bfloat16)):
        bias = None if kind is None else torch.randn(channels, generator=gen, device=dev).to(kind)
        _check(htrc_b200.int8_linear(x, w, bias=bias, dtype=dtype), x, w, bias, dtype)
    htrc_b200.int8_linear_status()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [s for s in SIZES if s[1] <= 16384])
def test_floats_are_quantised_on_the_way(dev, size, dtype):
    tokens, width, channels = size
    gen = torch.Generator(device=dev).manual_seed(sum(size) + 1)
    x = torch.randn((tokens, width), generator=gen, device=dev).to(dtype)
    w = htrc_b200.quantize_rows(torch.randn((channels, width), generator=gen, device=dev))
    bias = torch.randn(channels, generator=gen, device=dev).half()
    rows = htrc_b200.quantize_rows(x)
    got = htrc_b200.int8_linear(x, w, bias=bias)
    _check(got, rows, w, bias, dtype)
    assert torch.equal(got, htrc_b200.int8_linear(rows, w, bias=bias, dtype=dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [1, 5, 128, 130, 1000, 4096, 4104, 8200, 16384])
def test_few_float_rows(dev, width, dtype):
    """Up to 16 rows are quantised by the product itself (up to a width): the same codes as the rows' own kernel's, rows of
    any alignment and stride, split over the width or not."""
    gen = torch.Generator(device=dev).manual_seed(width)
    for channels in (100, 3000, 20000 if width < 1000 else 9000):
        w = htrc_b200.quantize_rows(torch.randn((channels, width), generator=gen, device=dev))
        for shape in ((1, 1), (16, 1), (3, 5)):
            room = torch.randn((*shape, width + 17), generator=gen, device=dev).to(dtype)
            for x in (room[..., :width], room[..., 17:], room[..., 1:1 + width].contiguous()):
                want = htrc_b200.int8_linear(htrc_b200.quantize_rows(x), w, dtype=dtype)
                assert torch.equal(htrc_b200.int8_linear(x, w), want)
    htrc_b200.int8_linear_status()


def test_extreme_codes_and_widest_rows(dev):
    """Sums at the ends of what the width allows: 65,536 products of 128 * 128 are 2^30."""
    for width in (65536, 1024):
        for a, b in ((-128, -128), (-128, 127), (127, 127)):
            x = Int8Rows(torch.full((3, width), a, dtype=torch.int8, device=dev), torch.ones(3, device=dev))
            w = Int8Rows(torch.full((5, width), b, dtype=torch.int8, device=dev), torch.ones(5, device=dev))
            assert torch.equal(htrc_b200.int8_linear(x, w, dtype=torch.float32),
                               torch.full((3, 5), float(a * b * width), device=dev))


def test_shapes_and_strides(dev):
    gen = torch.Generator(device=dev).manual_seed(4)
    w = htrc_b200.quantize_rows(torch.randn((200, 96), generator=gen, device=dev))
    big = torch.randn((3, 10, 4, 224), generator=gen, device=dev).bfloat16()
    for x in (big[..., 16:112], big[..., 3:99], big[:, ::2, 1, :96], big[0, 0, 0, 5:101], big.transpose(0, 2)[..., :96],
              big[:, :1, 0, :96].expand(3, 5, 96), big[..., 0:192:2], big[:0, :, 0, :96], big[:, :0, 0, :96], big[:0, ..., :96]):
        got = htrc_b200.int8_linear(x, w)
        assert got.shape == (*x.shape[:-1], 200)
        _check(got, htrc_b200.quantize_rows(x), w, None, torch.bfloat16)
    # codes of any layout: broadcast rows, odd starts, transposed, unit dimensions with any stride
    codes = torch.randint(-127, 128, (4, 6, 131), generator=gen, device=dev, dtype=torch.int8)
    scales = torch.rand((4, 6), generator=gen, device=dev)
    for c in (codes[..., 3:99], codes[..., :96], codes.transpose(0, 1)[..., 32:128], codes[:, :1, :96].expand(4, 6, 96),
              codes[:1, :, 7:103], codes.permute(2, 0, 1).contiguous().permute(1, 2, 0)[..., :96]):
        s = scales.T if c.shape[0] == 6 else scales[:c.shape[0]]
        x = Int8Rows(c, s)
        _check(htrc_b200.int8_linear(x, w, dtype=torch.float32), x, w, None, torch.float32)
        v = Int8Rows(c[0], s[0])
        _check(htrc_b200.int8_linear(big[0, 0, :, :96], v), htrc_b200.quantize_rows(big[0, 0, :, :96]), v, None, torch.bfloat16)
    bias = torch.randn(400, generator=gen, device=dev)[::2]
    _check(htrc_b200.int8_linear(big[0, 0, :, :96], w, bias=bias), htrc_b200.quantize_rows(big[0, 0, :, :96]), w, bias,
           torch.bfloat16)
    laid = htrc_b200.int8_rows(codes[0, :, 3:99], scales[0])
    assert laid.codes.stride(0) % 16 == 0 and torch.equal(laid.codes, codes[0, :, 3:99])
    assert htrc_b200.int8_rows(*laid).codes.data_ptr() == laid.codes.data_ptr()


def test_repeated_calls_with_other_alignments(dev):
    """What a call keeps for the next goes by shapes, strides and types, and no pointer is taken to be aligned."""
    gen = torch.Generator(device=dev).manual_seed(13)
    room = torch.randint(-127, 128, (90 * 112 + 64,), generator=gen, device=dev, dtype=torch.int8)
    scales = torch.rand(90, generator=gen, device=dev)
    for start in (0, 16, 0, 3, 32, 1, 0):
        x = Int8Rows(room[start:].as_strided((90, 96), (112, 1)), scales)
        w = Int8Rows(x.codes[:70], scales[:70])
        f = torch.randn(90 * 96 + 64, generator=gen, device=dev).bfloat16()[start:start + 90 * 96].view(90, 96)
        for _ in range(2):
            _check(htrc_b200.int8_linear(x, w, dtype=torch.float32), x, w, None, torch.float32)
            _check(htrc_b200.int8_linear(f, w), htrc_b200.quantize_rows(f), w, None, torch.bfloat16)


@pytest.mark.parametrize("tokens,channels", [(1, 1), (3, 77), (130, 130), (300, 520), (2100, 1030), (700, 2048),
                                             (5000, 1032), (9000, 515)])
def test_what_lies_around_the_result_is_left_alone(dev, tokens, channels):
    """Through the C entry, into the middle of a larger buffer."""
    gen = torch.Generator(device=dev).manual_seed(5)
    x, w = _rows(gen, dev, tokens, 256), _rows(gen, dev, channels, 256)
    for dtype in TYPES:
        buf = torch.full((tokens * channels + 8192,), 7.0, dtype=dtype, device=dev)
        out = buf[4096:4096 + tokens * channels]
        status = torch.zeros(64, dtype=torch.int32, device=dev)
        args = _lib.LINEAR8_ARGS.pack(x.codes.data_ptr(), 0, 256, x.scales.data_ptr(), 1, tokens, 256, channels, _lib.LAYER_I8,
                                      w.codes.data_ptr(), 256, w.scales.data_ptr(), 0, 0, _DTYPES[dtype], out.data_ptr(),
                                      status.data_ptr(), 0, 0)
        assert _lib.lib().htrc_linear8_forward(args, _lib.stream_ptr()) == _lib.HTRC_OK
        _check(out.view(tokens, channels), x, w, None, dtype)
        assert (buf[:4096] == 7).all() and (buf[4096 + tokens * channels:] == 7).all() and status[0] == 0


def test_offsets_past_32_bits(dev):
    gen = torch.Generator(device=dev).manual_seed(11)
    x, w = _rows(gen, dev, 70000, 64), _rows(gen, dev, 32768, 64)
    got = htrc_b200.int8_linear(x, w)
    for a in (0, 35000, 65500, 69990):
        some = slice(a, a + 10)
        _check(got[some], Int8Rows(x.codes[some], x.scales[some]), w, None, torch.bfloat16)
    x = torch.randn((140000, 16384), generator=gen, device=dev, dtype=torch.bfloat16)
    rows = htrc_b200.quantize_rows(x)
    w = htrc_b200.quantize_rows(x[:40])
    got = htrc_b200.int8_linear(x, w)
    for a in (0, 131060, 139990):
        some = slice(a, a + 10)
        _check(got[some], Int8Rows(rows.codes[some], rows.scales[some]), w, None, torch.bfloat16)


def test_bad_rows_stay_by_themselves(dev):
    gen = torch.Generator(device=dev).manual_seed(6)
    w = htrc_b200.quantize_rows(torch.randn((150, 300), generator=gen, device=dev))
    for tokens in (5, 400):
        x = torch.randn((tokens, 300), generator=gen, device=dev).half()
        x[1, 3], x[3, 0] = float("inf"), float("nan")
        x[2] = 0
        y = htrc_b200.int8_linear(x, w)
        rest = torch.ones(tokens, dtype=torch.bool, device=dev)
        rest[[1, 3]] = False
        assert torch.isnan(y[~rest]).all() and torch.isfinite(y[rest]).all() and (y[2] == 0).all()


def test_norm_then_product(dev):
    """What a layer runs: the norm's 8-bit rows into the product, against the two calls' own definitions and, within the
    8-bit steps, against float64: an element is off by at most half a step of its row and of its channel."""
    gen = torch.Generator(device=dev).manual_seed(7)
    for batch, tokens, width, channels in ((2, 70, 320, 200), (16, 1, 1024, 512), (2, 700, 512, 1030)):
        x = torch.randn((batch, tokens, width), generator=gen, device=dev).bfloat16()
        scale, shift = ((torch.randn((batch, width), generator=gen, device=dev) * 0.2).bfloat16() for _ in range(2))
        full = torch.randn((channels, width), generator=gen, device=dev) * width ** -0.5
        w = htrc_b200.quantize_rows(full)
        rows = htrc_b200.layer_norm_int8(x, scale=scale, shift=shift)
        got = htrc_b200.int8_linear(rows, w)
        _check(got, rows, w, None, torch.bfloat16)
        d = x.double()
        u = (d - d.mean(-1, keepdim=True)) * (d.var(-1, unbiased=False, keepdim=True) + 1e-6).rsqrt()
        y = u * (1 + scale.double()[:, None]) + shift.double()[:, None]
        want = y @ full.double().T
        step = 0.51 * rows.scales.double()[..., None]
        off = step * full.double().abs().sum(-1) + 0.51 * w.scales.double() * y.abs().sum(-1, keepdim=True) + \
            step * 0.51 * w.scales.double() * width
        assert ((got.double() - want).abs() <= off + 2.0 ** -8 * want.abs()).all()


def test_streams_graphs_and_repeats(dev):
    gen = torch.Generator(device=dev).manual_seed(8)
    cases = []
    for tokens, width, channels in ((1, 2048, 512), (40, 640, 640), (700, 384, 1100), (4000, 512, 2048)):
        x = torch.randn((tokens, width), generator=gen, device=dev).bfloat16()
        w = htrc_b200.quantize_rows(torch.randn((channels, width), generator=gen, device=dev))
        cases.append((x, w))

    def step():
        # products straight after the kernels that write their rows and weights, and after one another
        out = []
        for x, w in cases:
            y = htrc_b200.int8_linear(x, w)
            back = htrc_b200.quantize_rows(w.codes.float())
            out += [y, htrc_b200.int8_linear(htrc_b200.quantize_rows(x), back), htrc_b200.int8_linear(x, back)]
        return out
    want = step()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(step(), want))
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    keep = [x.clone() for x, _ in cases]
    for k in range(2):
        for (x, _), x0 in zip(cases, keep):
            x.copy_(x0 if k else torch.randn_like(x0))
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    htrc_b200.int8_linear_status()


def test_no_rows_and_calls_on_two_streams_at_once(dev):
    gen = torch.Generator(device=dev).manual_seed(17)
    w = _rows(gen, dev, 300, 256)
    none = Int8Rows(w.codes[:0], w.scales[:0])
    assert htrc_b200.int8_linear(none, w).shape == (0, 300)
    assert htrc_b200.int8_linear(torch.empty((2, 0, 256), device=dev), w).shape == (2, 0, 300)
    cases = [(torch.randn((n, k), generator=gen, device=dev).half(), _rows(gen, dev, m, k))
             for n, k, m in ((5, 512, 700), (16, 4096, 300), (40, 1000, 520), (900, 256, 8200), (5000, 384, 1100))]
    want = [htrc_b200.int8_linear(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    got = []
    for k in range(4):
        for i, c in enumerate(cases):
            with torch.cuda.stream(streams[(i + k) % 2]):
                got.append((i, htrc_b200.int8_linear(*c)))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i, g in got)
    htrc_b200.int8_linear_status()


def test_refusals(dev):
    x = torch.zeros((4, 64), device=dev).bfloat16()
    w = htrc_b200.quantize_rows(torch.ones((8, 64), device=dev))
    ones = torch.ones(8, device=dev)
    with pytest.raises(ValueError):
        htrc_b200.int8_linear(x[:, :63], w)
    with pytest.raises(ValueError):
        htrc_b200.int8_linear(x.double(), w)
    with pytest.raises(ValueError):
        htrc_b200.int8_linear(x, w.codes)
    with pytest.raises(ValueError):
        htrc_b200.int8_linear(x, (w.codes.int(), w.scales))
    with pytest.raises(ValueError):
        htrc_b200.int8_linear(x, (w.codes, w.scales[:7]))
    with pytest.raises(ValueError):
        htrc_b200.int8_linear(x, (w.codes.cpu(), w.scales.cpu()))
    with pytest.raises(ValueError):
        htrc_b200.int8_linear(x, w, bias=ones[:7])
    with pytest.raises(ValueError):
        htrc_b200.int8_linear(x, w, bias=ones.int())
    with pytest.raises(ValueError):
        htrc_b200.int8_linear(x, w, dtype=torch.int8)
    with pytest.raises(ValueError):
        htrc_b200.int8_linear((w.codes, w.scales.half()), w)
    with pytest.raises(NotImplementedError, match="gradients"):
        htrc_b200.int8_linear(x.float().requires_grad_(), w)
    with pytest.raises(NotImplementedError, match="gradients"):
        htrc_b200.int8_linear(x, w, bias=ones.requires_grad_())
    wide = Int8Rows(torch.zeros((2, 65537), dtype=torch.int8, device=dev), torch.ones(2, device=dev))
    with pytest.raises(NotImplementedError):
        htrc_b200.int8_linear(wide, wide)
    wide = Int8Rows(torch.zeros((2, 16400), dtype=torch.int8, device=dev), torch.ones(2, device=dev))
    with pytest.raises(NotImplementedError):
        htrc_b200.int8_linear(torch.zeros((2, 16400), device=dev), wide)
