"""The 8-bit product refuses the same pairs after calls of the same shapes as before them."""
from __future__ import annotations

import pytest
import torch

import htrc_b200

pytestmark = pytest.mark.gpu


def test_lists_are_refused_after_tuples_were_taken():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    x = torch.randn((4, 64), device="cuda").bfloat16()
    w, rows = htrc_b200.quantize_rows(torch.randn((8, 64), device="cuda")), htrc_b200.quantize_rows(x)
    for _ in range(2):
        assert torch.equal(htrc_b200.int8_linear(x, tuple(w)), htrc_b200.int8_linear(tuple(rows), w))
        for args in ((x, list(w)), (list(rows), w), (rows, list(w))):
            with pytest.raises(ValueError):
                htrc_b200.int8_linear(*args)
