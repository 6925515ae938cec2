"""Host-side checks of the operators around the flat attention that need no GPU: the structs' layouts against
include/htrc_layer.h, the C entries' refusals (which come before the device is asked for), and the Python layer's."""
from __future__ import annotations

import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import htrc_b200
from htrc_b200 import _lib

ROOT = Path(__file__).resolve().parents[1]
HEADER = (ROOT / "include" / "htrc_layer.h").read_text()


def test_every_declared_symbol_is_bound():
    names = set(re.findall(r"\bint (htrc_\w+)\(", HEADER))
    assert names and names <= set(_lib.SIGNATURES)


def test_struct_layouts_match_c(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    lines = []
    for cls in (_lib.HtrcRotaryTensor, _lib.HtrcRotaryArgs, _lib.HtrcCrossArgs):
        name = cls.__name__
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        for f, *_ in cls._fields_:
            lines.append(f'printf("{name}.{f} %zu\\n", offsetof({name}, {f.rstrip("_")}));')
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "htrc_layer.h"\nint main(void) {\n' + "\n".join(lines) +
                   "\nreturn 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run([cc, "-std=c99", "-Wall", "-Werror", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for cls in (_lib.HtrcRotaryTensor, _lib.HtrcRotaryArgs, _lib.HtrcCrossArgs):
        assert int(got[cls.__name__]) == ctypes.sizeof(cls)
        for f, *_ in cls._fields_:
            assert int(got[f"{cls.__name__}.{f}"]) == getattr(cls, f).offset, f
    assert _lib.ROTARY_ARGS.size == ctypes.sizeof(_lib.HtrcRotaryArgs)
    assert _lib.CROSS_ARGS.size == ctypes.sizeof(_lib.HtrcCrossArgs)


def test_packed_structs_hold_the_fields_in_order():
    values = list(range(1, 1 + len(_lib.CROSS_ARGS.unpack(bytes(_lib.CROSS_ARGS.size)))))
    a = _lib.HtrcCrossArgs.from_buffer_copy(_lib.CROSS_ARGS.pack(*values))
    flat = []
    for f, t in _lib.HtrcCrossArgs._fields_:
        v = getattr(a, f)
        flat += list(v) if hasattr(v, "__len__") else [v]
    assert flat == values
    values = list(range(1, 1 + len(_lib.ROTARY_ARGS.unpack(bytes(_lib.ROTARY_ARGS.size)))))
    r = _lib.HtrcRotaryArgs.from_buffer_copy(_lib.ROTARY_ARGS.pack(*values))
    assert r.tensor[0].in_ == 1 and r.tensor[1].in_ == 17 and r.tensor[1].heads == 32 and r.n_tensors == 33
    assert r.dim == 37 and r.axis_width[3] == 42 and r.theta == 49.0 and r.eps == 51.0 and r.workspace_bytes == 53


def _rotary(**kw):
    a = _lib.HtrcRotaryArgs()
    a.n_tensors, a.dtype, a.batch, a.tokens, a.dim, a.n_axes = 1, _lib.LAYER_BF16, 1, 4, 64, 2
    a.axis_width[:] = (32, 32, 0, 0)
    a.position_dtype, a.theta, a.eps, a.positions = _lib.LAYER_I32, 1e4, 1e-6, 256
    t = a.tensor[0]
    t.in_ = t.out = 256
    t.heads = 2
    for k, v in kw.items():
        if k == "axis_width":
            a.axis_width[:] = v
        else:
            setattr(t if hasattr(t, k) and k not in ("dim",) else a, k, v)
    return a


@pytest.mark.parametrize("kw,rc", [
    (dict(n_tensors=0), _lib.HTRC_ERR_ARG), (dict(n_tensors=3), _lib.HTRC_ERR_ARG), (dict(dtype=3), _lib.HTRC_ERR_ARG),
    (dict(tokens=-1), _lib.HTRC_ERR_ARG), (dict(batch=1 << 39), _lib.HTRC_ERR_UNSUPPORTED), (dict(dim=1), _lib.HTRC_ERR_ARG),
    (dict(dim=257), _lib.HTRC_ERR_UNSUPPORTED), (dict(n_axes=0), _lib.HTRC_ERR_ARG), (dict(n_axes=5), _lib.HTRC_ERR_UNSUPPORTED),
    (dict(axis_width=(31, 32, 0, 0)), _lib.HTRC_ERR_ARG), (dict(axis_width=(64, 2, 0, 0)), _lib.HTRC_ERR_ARG),
    (dict(pairs=2), _lib.HTRC_ERR_ARG), (dict(position_dtype=_lib.LAYER_BF16), _lib.HTRC_ERR_ARG), (dict(theta=0.0), _lib.HTRC_ERR_ARG),
    (dict(theta=float("nan")), _lib.HTRC_ERR_ARG), (dict(eps=-1.0), _lib.HTRC_ERR_ARG), (dict(heads=0), _lib.HTRC_ERR_ARG),
    (dict(heads=1025), _lib.HTRC_ERR_UNSUPPORTED), (dict(weight_dtype=4), _lib.HTRC_ERR_ARG), (dict(in_=None), _lib.HTRC_ERR_ARG),
    (dict(out=None), _lib.HTRC_ERR_ARG), (dict(positions=None), _lib.HTRC_ERR_ARG)])
def test_rotary_entries_refuse(kw, rc):
    L = _lib.lib()
    a = _rotary(**kw)
    assert L.htrc_rotary_forward(ctypes.byref(a), None) == rc
    assert L.htrc_rotary_backward(ctypes.byref(a), None) == rc


def test_rotary_backward_wants_its_operands_and_workspace():
    L = _lib.lib()
    assert L.htrc_rotary_forward(None, None) == _lib.HTRC_ERR_ARG
    assert L.htrc_rotary_backward(ctypes.byref(_rotary(weight=256)), None) == _lib.HTRC_ERR_ARG          # x, dweight missing
    n = ctypes.c_size_t()
    assert L.htrc_rotary_workspace_size(ctypes.byref(_rotary()), ctypes.byref(n)) == _lib.HTRC_OK and n.value >= 2 * 64 * 4
    assert L.htrc_rotary_workspace_size(ctypes.byref(_rotary(dim=0)), ctypes.byref(n)) == _lib.HTRC_ERR_ARG
    assert L.htrc_rotary_workspace_size(ctypes.byref(_rotary()), None) == _lib.HTRC_ERR_ARG


def _cross(**kw):
    a = _lib.HtrcCrossArgs()
    a.q = a.k = a.v = a.out = a.lse = a.dout = a.dq = a.dk = a.dv = 256
    for f in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
        getattr(a, f + "_stride")[:] = (1 << 16, 64, 64)
    a.batch, a.queries, a.keys, a.heads, a.kv_heads, a.dim = 2, 9, 7, 4, 2, 64
    a.dtype, a.scale = _lib.LAYER_BF16, 0.125
    for k, v in kw.items():
        if k.endswith("_stride"):
            getattr(a, k)[:] = v
        else:
            setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,rc", [
    (dict(batch=-1), _lib.HTRC_ERR_ARG), (dict(queries=-1), _lib.HTRC_ERR_ARG), (dict(keys=-1), _lib.HTRC_ERR_ARG),
    (dict(heads=0), _lib.HTRC_ERR_ARG), (dict(heads=5), _lib.HTRC_ERR_ARG), (dict(kv_heads=0), _lib.HTRC_ERR_ARG),
    (dict(dtype=_lib.LAYER_F32), _lib.HTRC_ERR_ARG), (dict(dim=60), _lib.HTRC_ERR_ARG), (dict(dim=0), _lib.HTRC_ERR_ARG),
    (dict(dim=136), _lib.HTRC_ERR_UNSUPPORTED), (dict(queries=1 << 31), _lib.HTRC_ERR_UNSUPPORTED), (dict(scale=0.0), _lib.HTRC_ERR_ARG),
    (dict(scale=float("inf")), _lib.HTRC_ERR_ARG), (dict(mask=256, mask_dtype=_lib.LAYER_I32), _lib.HTRC_ERR_ARG),
    (dict(q=None), _lib.HTRC_ERR_ARG), (dict(k=None), _lib.HTRC_ERR_ARG), (dict(out=None), _lib.HTRC_ERR_ARG), (dict(q=264), _lib.HTRC_ERR_ARG),
    (dict(k_stride=(64, 60, 64)), _lib.HTRC_ERR_ARG), (dict(v_stride=(64, 0, 64)), _lib.HTRC_ERR_ARG),
    (dict(out_stride=(64, -64, 64)), _lib.HTRC_ERR_ARG)])
def test_cross_entries_refuse(kw, rc):
    L = _lib.lib()
    a = _cross(**kw)
    assert L.htrc_cross_forward(ctypes.byref(a), None) == rc
    assert L.htrc_cross_backward(ctypes.byref(a), None) == rc


@pytest.mark.parametrize("name", ["lse", "dout", "dq", "dk", "dv"])
def test_cross_backward_wants_its_operands(name):
    assert _lib.lib().htrc_cross_backward(ctypes.byref(_cross(**{name: None})), None) == _lib.HTRC_ERR_ARG


def test_cross_workspace_size():
    L = _lib.lib()
    n = ctypes.c_size_t()
    assert L.htrc_cross_backward_workspace_size(ctypes.byref(_cross()), ctypes.byref(n)) == _lib.HTRC_OK and n.value >= 2 * 4 * 9 * 8
    assert L.htrc_cross_backward_workspace_size(ctypes.byref(_cross(dim=12)), ctypes.byref(n)) == _lib.HTRC_ERR_ARG
    assert L.htrc_cross_backward_workspace_size(ctypes.byref(_cross()), None) == _lib.HTRC_ERR_ARG
    assert L.htrc_cross_forward(None, None) == _lib.HTRC_ERR_ARG


def test_python_layer_refuses_without_a_device():
    q = torch.zeros((1, 4, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        htrc_b200.cross_attention(q, q, q)
    with pytest.raises(ValueError, match="CUDA"):
        htrc_b200.rotary_axes(q, torch.zeros((4, 1)), axes=(64,))
    with pytest.raises(ValueError, match="even"):
        htrc_b200.rotary_axes(q, torch.zeros((4, 1)), axes=(63,))
    with pytest.raises(ValueError):
        htrc_b200.grid_positions((2, -1), device="cpu")
    with pytest.raises(ValueError):
        htrc_b200.grid_positions((2, 2), start=(0,), device="cpu")


def test_grid_positions_are_row_major():
    p = htrc_b200.grid_positions((2, 3, 4), start=(5, 0, 1), device="cpu")
    assert p.dtype == torch.int32 and p.shape == (24, 3)
    assert p[0].tolist() == [5, 0, 1] and p[1].tolist() == [5, 0, 2] and p[4].tolist() == [5, 1, 1] and p[23].tolist() == [6, 2, 4]
    assert htrc_b200.grid_positions((0, 3), device="cpu").shape == (0, 2)
