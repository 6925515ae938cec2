"""Products that may start under the kernel before them, captured where no kernel is before them on their stream: first in the
graph, behind a fill or a copy, behind another stream's work."""
from __future__ import annotations

import pytest
import torch

import htrc_b200

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [1, 16, 40])
@pytest.mark.parametrize("before", ["nothing", "fill", "copy", "other stream", "gradients"])
def test_captured_behind(tokens, before):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev).manual_seed(tokens)
    x = torch.randn((tokens, 512), generator=gen, device=dev)
    w = htrc_b200.quantize_rows(torch.randn((300, 512), generator=gen, device=dev))
    rows = htrc_b200.quantize_rows(x)
    new, bias, full = torch.randn_like(x), torch.zeros(300, device=dev), torch.randn(300, generator=gen, device=dev)
    ones, side = torch.ones_like(x), torch.cuda.Stream(dev)

    def step():
        main = torch.cuda.current_stream(dev)
        if before == "fill":
            bias.zero_()
        elif before == "copy":
            bias.copy_(full)
        elif before == "other stream":
            side.wait_stream(main)
            with torch.cuda.stream(side):
                x.copy_(new)
            main.wait_stream(side)
        elif before == "gradients":
            _, mean, rstd = htrc_b200.layer_norm(new, return_stats=True)
            htrc_b200.layer_norm_backward(ones, new, mean, rstd)
        return htrc_b200.int8_linear(x, w, bias=bias), htrc_b200.int8_linear(rows, w, bias=bias), \
            htrc_b200.int8_linear(htrc_b200.layer_norm_int8(x), w, dtype=torch.float32)
    want = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        for t in got:
            t.fill_(7.0)
        if before in ("fill", "copy"):
            bias.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    htrc_b200.int8_linear_status()
