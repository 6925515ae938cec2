"""Key masks that differ between the query heads that share a key head: what one of them excludes it never computes with,
even where another one does, whatever the number of queries."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_cross import _check, _rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda:0")


SIZES = [(3, 1, 203, 4, 2, 128), (2, 2, 77, 6, 2, 64), (2, 4, 1300, 8, 2, 128), (2, 5, 40, 6, 2, 72), (1, 16, 300, 4, 2, 64),
         (40, 1, 500, 24, 8, 128), (2, 150, 203, 4, 2, 128)]


def _head_mask(b, h, m, additive, gen, dev):
    keep = torch.rand((b, h, 1, m), generator=gen, device=dev) < 0.6
    if not additive:
        return keep, keep
    return keep, torch.where(keep, torch.randn((b, h, 1, m), generator=gen, device=dev), -math.inf)


@pytest.mark.parametrize("additive", [False, True])
@pytest.mark.parametrize("size", SIZES)
def test_masks_of_heads_match_float64(dev, size, additive):
    b, n, m, h, hk, d = size
    gen = torch.Generator(device=dev).manual_seed(sum(size))
    q, k, v = _rows(dev, *size, torch.bfloat16, seed=sum(size))
    _, mask = _head_mask(b, h, m, additive, gen, dev)
    _check(q, k, v, mask=mask)
    lengths = torch.randint(0, m + 1, (b,), generator=gen, device=dev, dtype=torch.int32)
    _check(q, k, v, mask=mask, lengths=lengths)


@pytest.mark.parametrize("additive", [False, True])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("size", SIZES)
def test_a_head_never_reads_what_it_excludes(dev, size, bad, additive):
    import htrc_b200
    b, n, m, h, hk, d = size
    group = h // hk
    gen = torch.Generator(device=dev).manual_seed(sum(size))
    q, k, v = _rows(dev, *size, torch.bfloat16, seed=sum(size))
    keep, mask = _head_mask(b, h, m, additive, gen, dev)
    dirty = torch.rand((b, hk, m), generator=gen, device=dev) < 0.2       # keys that the first head of each group excludes
    first = torch.arange(h, device=dev) % group == 0
    off = dirty.repeat_interleave(group, 1)[:, :, None] & first.view(1, h, 1, 1)
    mask = mask & ~off if mask.dtype == torch.bool else mask.masked_fill(off, -math.inf)
    kw = dict(mask=mask, heads_first=True)
    clean = htrc_b200.cross_attention(q, k, v, return_lse=True, **kw)
    got = htrc_b200.cross_attention(q, k.masked_fill(dirty[..., None], bad), v.masked_fill(dirty[..., None], bad),
                                    return_lse=True, **kw)
    for x, y in zip(clean, got):
        assert torch.equal(x[:, first], y[:, first])
    do = torch.randn(q.shape, generator=gen, device=dev).to(q.dtype)
    want = htrc_b200.cross_attention_backward(do, q, k, v, *clean, **kw)
    back = htrc_b200.cross_attention_backward(do, q, k.masked_fill(dirty[..., None], bad),
                                              v.masked_fill(dirty[..., None], bad), *clean, **kw)
    assert torch.equal(want[0][:, first], back[0][:, first])
    htrc_b200.cross_status()
