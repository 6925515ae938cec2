"""No module of the package defines a function or class twice: the first would never be called."""
from __future__ import annotations

import ast
from collections import Counter
from pathlib import Path

import pytest

FILES = sorted((Path(__file__).resolve().parents[1] / "htrc_b200").glob("*.py"))


@pytest.mark.parametrize("file", FILES, ids=lambda f: f.name)
def test_defined_once(file):
    names = Counter(n.name for n in ast.parse(file.read_text()).body if isinstance(n, (ast.FunctionDef, ast.ClassDef)))
    assert not [name for name, n in names.items() if n > 1]
