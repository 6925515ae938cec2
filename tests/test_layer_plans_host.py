"""What the 8-bit product keeps of a call for the next one of the same shapes changes nothing of what it refuses."""
from __future__ import annotations

import pytest
import torch

import htrc_b200
from htrc_b200 import Int8Rows, linear8


class Everything(dict):
    """A kept plan for whatever is asked for."""

    def get(self, key):
        raise AssertionError("a kept plan was used before the arguments were checked")


@pytest.mark.parametrize("x,weight", [
    (torch.zeros((4, 64)), [torch.zeros((8, 64), dtype=torch.int8), torch.ones(8)]),
    ([torch.zeros((4, 64), dtype=torch.int8), torch.ones(4)], Int8Rows(torch.zeros((8, 64), dtype=torch.int8), torch.ones(8)))])
def test_pairs_of_another_type_are_refused_whatever_was_called_before(monkeypatch, x, weight):
    monkeypatch.setattr(linear8, "_plans", Everything())
    with pytest.raises(ValueError):
        htrc_b200.int8_linear(x, weight)
