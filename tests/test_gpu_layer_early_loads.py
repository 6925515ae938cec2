"""Products that start under the kernel before them: what that kernel writes into memory which earlier products read (rows,
scales, bias, weights) is what they use, without anything waiting between the calls."""
from __future__ import annotations

import pytest
import torch

import htrc_b200
from htrc_b200 import Int8Rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda:0")


@pytest.mark.parametrize("tokens,width,channels", [(1, 512, 300), (16, 1024, 2048), (40, 640, 640), (100, 256, 200), (300, 512, 300)])
def test_inputs_that_change_between_calls(dev, tokens, width, channels):
    gen = torch.Generator(device=dev).manual_seed(tokens + width)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev)
    rounds = 6
    xs = [normal(tokens, width).bfloat16() * 2.0 ** k for k in range(rounds)]
    full = [htrc_b200.quantize_rows(normal(channels, width)) for _ in range(rounds)]
    biases = [normal(channels) for _ in range(rounds)]
    x, w, bias = xs[0].clone(), Int8Rows(*(t.clone() for t in full[0])), biases[0].clone()
    codes, scales = (t.clone() for t in htrc_b200.quantize_rows(x))

    def put(k):
        """Everything that a call reads changes in place, each by a kernel or a copy just before the call that reads it."""
        x.copy_(xs[k])
        for mine, new in zip(w, full[k]):
            mine.copy_(new)
        bias.copy_(biases[k])

    def calls():
        first = htrc_b200.int8_linear(x, w, bias=bias)
        rows = htrc_b200.layer_norm_int8(x)
        second = htrc_b200.int8_linear(rows, w, bias=bias)
        again = htrc_b200.quantize_rows(x)
        codes.copy_(again.codes)
        scales.copy_(again.scales)
        return first, second, htrc_b200.int8_linear(Int8Rows(codes, scales), w)

    want = []
    for k in range(rounds):
        put(k)
        torch.cuda.synchronize()
        out = []
        for y in calls():
            torch.cuda.synchronize()
            out.append(y)
        want.append(out)
    for _ in range(4):
        got = []
        for k in range(rounds):
            put(k)
            got.append(calls())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, h in zip(got, want) for a, b in zip(g, h))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = calls()
    for k in (0, 3, 5, 1):
        put(k)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[k]))
    htrc_b200.int8_linear_status()
