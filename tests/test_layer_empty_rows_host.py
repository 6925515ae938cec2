"""Codes without a row: whichever dimension is the empty one, they have a pitch, so that no call lays them out or fails on them."""
from __future__ import annotations

import pytest
import torch

from htrc_b200 import linear8


@pytest.mark.parametrize("shape", [(0, 32), (3, 0, 32), (0, 3, 32), (3, 0, 20), (2, 3, 0, 32), (2, 0, 3, 32), (2, 0, 0, 1), (0, 0, 17)])
def test_pitch_of_no_rows(shape):
    dense = torch.zeros(shape, dtype=torch.int8)
    laid, pitch = linear8._new_codes(shape, dense)
    want = (shape[-1] + 15) // 16 * 16
    assert linear8._pitch(dense) == linear8._pitch(laid) == pitch == want
    # a slice of more rows keeps their strides
    room = torch.zeros((*(n + 1 for n in shape[:-1]), want), dtype=torch.int8)
    if not room.data_ptr() & 15:
        assert linear8._pitch(room[tuple(slice(n) for n in shape)]) == want
