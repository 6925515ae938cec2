"""A layer's norm and projection in 8 bits on batches without a token: each call gives what the next one takes."""
from __future__ import annotations

import pytest
import torch

import htrc_b200

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda:0")


@pytest.mark.parametrize("shape", [(0, 32), (3, 0, 32), (0, 3, 32), (3, 0, 20), (2, 3, 0, 32), (2, 0, 3, 17)])
def test_rows_of_an_empty_batch_go_through_the_product(dev, shape):
    width = shape[-1]
    x = torch.empty(shape, device=dev, dtype=torch.bfloat16)
    w = htrc_b200.quantize_rows(torch.randn((48, width), device=dev))
    for rows in (htrc_b200.layer_norm_int8(x), htrc_b200.quantize_rows(x), htrc_b200.int8_rows(*htrc_b200.quantize_rows(x)), x):
        for _ in range(2):
            y = htrc_b200.int8_linear(rows, w)
            assert y.shape == (*shape[:-1], 48) and y.dtype is torch.bfloat16
    htrc_b200.int8_linear_status()
