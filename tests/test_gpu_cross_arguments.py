"""Arguments that cross attention takes in every form its documentation names."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda:0")


@pytest.mark.parametrize("dtype,keys", [(torch.uint8, 300), (torch.int8, 200), (torch.int16, 33000), (torch.int64, 300)])
def test_lengths_of_narrow_types(dev, dtype, keys):
    """A type that cannot hold the number of keys still says how many of them an entry has."""
    import htrc_b200
    gen = torch.Generator(device=dev).manual_seed(3)
    q = torch.randn((4, 3, 2, 64), generator=gen, device=dev).bfloat16()
    k, v = (torch.randn((4, keys, 2, 64), generator=gen, device=dev).bfloat16() for _ in range(2))
    lengths = torch.tensor([100, 0, 127, 7], device=dev)
    want = htrc_b200.cross_attention(q, k, v, key_lengths=lengths.int(), return_lse=True)
    got = htrc_b200.cross_attention(q, k, v, key_lengths=lengths.to(dtype), return_lse=True)
    assert all(torch.equal(x, y) for x, y in zip(want, got))


@pytest.mark.parametrize("name", ["cuda", "cuda:0", 0, None])
def test_status_of_a_device_by_any_name(dev, name):
    """A bit in the device's status word is reported, and cleared, whatever the device is called."""
    import htrc_b200
    from htrc_b200 import _lib, cross
    htrc_b200.cross_status(dev)
    cross._status_word(dev)[0] = 1
    with pytest.raises(_lib.HtrcError, match="bounded wait"):
        htrc_b200.cross_status(name)
    htrc_b200.cross_status(dev)


def _operands(dev):
    gen = torch.Generator(device=dev).manual_seed(4)
    return [torch.randn((2, 40, 2, 64), generator=gen, device=dev).bfloat16() for _ in range(3)]


def test_status_word_is_zeroed_before_any_stream_sees_it(dev):
    """The word is made by the first call; a bit that another stream sets right after it is not lost under the zero fill."""
    import htrc_b200
    from htrc_b200 import _lib, cross
    args = _operands(dev)
    htrc_b200.cross_attention(*args)
    torch.cuda.synchronize()
    cross._status.clear()
    busy, other = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(busy):
        torch.cuda._sleep(50_000_000)               # some 30 ms before anything else of this stream runs
        htrc_b200.cross_attention(*args)
    with torch.cuda.stream(other):
        cross._status_word(dev)[0] = 1
    torch.cuda.synchronize()
    with pytest.raises(_lib.HtrcError, match="bounded wait"):
        htrc_b200.cross_status(dev)
    htrc_b200.cross_status(dev)


def test_first_call_in_a_graph(dev):
    """A capture does not make the word: no replay then clears what other calls reported."""
    import htrc_b200
    from htrc_b200 import _lib, cross
    args = _operands(dev)
    want = htrc_b200.cross_attention(*args)
    torch.cuda.synchronize()
    cross._status.clear()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = htrc_b200.cross_attention(*args)
    htrc_b200.cross_status(dev)
    cross._status_word(dev)[0] = 1
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(want, got)
    with pytest.raises(_lib.HtrcError, match="bounded wait"):
        htrc_b200.cross_status(dev)
    htrc_b200.cross_status(dev)


def test_odd_strides_of_single_rows(dev):
    """A dimension of one is never stepped along: its stride may be anything (a token cut from a wider buffer)."""
    import htrc_b200
    gen = torch.Generator(device=dev).manual_seed(5)
    wide = torch.randn((4, 1, 1, 1, 67), generator=gen, device=dev).bfloat16()
    q, k, v, do = (x[..., :64] for x in wide.unbind())
    assert q.stride(1) % 8 and q.is_contiguous()
    for heads_first in (False, True):
        out, lse = htrc_b200.cross_attention(q, k, v, heads_first=heads_first, return_lse=True)
        assert torch.equal(out, v) and (lse.double() - (q.double() * k.double()).sum() * 0.125).abs().max() < 1e-5
        dq, dk, dv = htrc_b200.cross_attention_backward(do, q, k, v, out, lse, heads_first=heads_first)
        assert torch.equal(dv, do) and dq.abs().max() < 1e-2 and dk.abs().max() < 1e-2
    x = torch.randn((1, 9 * 64 + 1), generator=gen, device=dev).bfloat16()[:, :9 * 64]
    rows = x.as_strided((1, 9, 1, 64), (9 * 64 + 1, 64, 3, 1))          # one entry, one head, by any stride
    dense = x.reshape(1, 9, 1, 64).clone()
    for a, b in zip(htrc_b200.cross_attention(rows, rows, rows, return_lse=True),
                    htrc_b200.cross_attention(dense, dense, dense, return_lse=True)):
        assert torch.equal(a, b)
