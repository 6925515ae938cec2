"""Kernels that are launched while the one before them still runs (griddepcontrol.wait in their source) read what it may have
written by ordinary loads: those of the read-only path (__ldg, ld.global.nc) are defined only for data that nothing writes
while the kernel lives."""
from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "htrc_b200" / "csrc"
READ_ONLY = re.compile(r"__ldg|ld\.global\.nc")


def _function(source, name):
    """A device function's definition, up to the brace that closes it."""
    start = re.search(rf"\b{name}\s*\([^;{{]*\)\s*{{", source)
    assert start, name
    depth, at = 1, start.end()
    while depth:
        depth += {"{": 1, "}": -1}.get(source[at], 0)
        at += 1
    return source[start.start():at]


@pytest.mark.parametrize("file,kernel,uses", [
    ("linear8.cu", "linear8_small_kernel", ["quantise_row", "bias_at"]), ("cross_few.cu", "cross_few_join_kernel", [])])
def test_no_read_only_loads(file, kernel, uses):
    source = (CSRC / file).read_text()
    body = _function(source, kernel)
    assert "griddepcontrol.wait" in body
    for part in [body] + [_function(source, f) for f in uses]:
        assert not READ_ONLY.search(part), READ_ONLY.search(part)


def test_the_sums_of_the_norms_parts():
    """Only the parts are written by the kernel before: the parameters (term_at) are older than that kernel's own launch."""
    body = _function((CSRC / "norm.cu").read_text(), "norm_terms_kernel")
    assert "griddepcontrol.wait" in body and not READ_ONLY.search(body) and body.count("__ldcg(") == 4
