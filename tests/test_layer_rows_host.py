"""Host-side checks of the layer norm and the 8-bit product that need no GPU: the structs' layouts against
include/htrc_layer.h, the C entries' refusals (which come before the device is asked for), and the Python layer's."""
from __future__ import annotations

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import htrc_b200
from htrc_b200 import _lib, linear8

ROOT = Path(__file__).resolve().parents[1]
STRUCTS = ((_lib.HtrcNormArgs, _lib.NORM_ARGS), (_lib.HtrcLinear8Args, _lib.LINEAR8_ARGS))


def test_struct_layouts_match_c(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    lines = []
    for cls, _ in STRUCTS:
        name = cls.__name__
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, *_ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "htrc_layer.h"\nint main(void) {\n' + "\n".join(lines) +
                   "\nreturn 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run([cc, "-std=c99", "-Wall", "-Werror", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for cls, packed in STRUCTS:
        assert int(got[cls.__name__]) == ctypes.sizeof(cls) == packed.size
        for f, *_ in cls._fields_:
            assert int(got[f"{cls.__name__}.{f}"]) == getattr(cls, f).offset, f


def test_packed_structs_hold_the_fields_in_order():
    for cls, packed in STRUCTS:
        values = list(range(1, 1 + len(packed.unpack(bytes(packed.size)))))
        a = cls.from_buffer_copy(packed.pack(*values))
        flat = []
        for f, _ in cls._fields_:
            v = getattr(a, f)
            flat += list(v) if hasattr(v, "__len__") else [v]
        assert flat == values


def _norm(**kw):
    a = _lib.HtrcNormArgs()
    a.x = a.out = a.dy = a.dx = a.mean = a.rstd = 256
    for f in ("x", "out", "dy", "dx"):
        getattr(a, f + "_stride")[:] = (1 << 12, 64)
    a.batch, a.tokens, a.width, a.dtype, a.eps = 2, 5, 64, _lib.LAYER_BF16, 1e-6
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,rc", [
    (dict(batch=-1), _lib.HTRC_ERR_ARG), (dict(tokens=-1), _lib.HTRC_ERR_ARG), (dict(width=0), _lib.HTRC_ERR_ARG),
    (dict(width=16385), _lib.HTRC_ERR_UNSUPPORTED), (dict(batch=1 << 31), _lib.HTRC_ERR_UNSUPPORTED), (dict(dtype=3), _lib.HTRC_ERR_ARG),
    (dict(dtype=_lib.LAYER_I8), _lib.HTRC_ERR_ARG), (dict(eps=-1.0), _lib.HTRC_ERR_ARG), (dict(eps=float("inf")), _lib.HTRC_ERR_ARG),
    (dict(weight_dtype=4), _lib.HTRC_ERR_ARG), (dict(shift_dtype=-1), _lib.HTRC_ERR_ARG), (dict(x=None), _lib.HTRC_ERR_ARG)])
def test_norm_entries_refuse(kw, rc):
    L = _lib.lib()
    a = _norm(**kw)
    assert L.htrc_norm_forward(ctypes.byref(a), None) == rc
    assert L.htrc_norm_backward(ctypes.byref(a), None) == rc


@pytest.mark.parametrize("kw", [dict(out=None), dict(codes=256, codes_pitch=64), dict(codes=256, codes_pitch=48, scales=256),
                                dict(codes=256, codes_pitch=72, scales=256), dict(codes=264, codes_pitch=64, scales=256)])
def test_norm_forward_wants_its_outputs(kw):
    assert _lib.lib().htrc_norm_forward(ctypes.byref(_norm(**kw)), None) == _lib.HTRC_ERR_ARG


@pytest.mark.parametrize("kw", [dict(dy=None), dict(dx=None), dict(mean=None), dict(rstd=None), dict(dweight=256), dict(dshift=256)])
def test_norm_backward_wants_its_operands(kw):
    assert _lib.lib().htrc_norm_backward(ctypes.byref(_norm(**kw)), None) == _lib.HTRC_ERR_ARG


def test_norm_workspace_size():
    L = _lib.lib()
    n = ctypes.c_size_t(1)
    assert L.htrc_norm_workspace_size(ctypes.byref(_norm()), ctypes.byref(n)) == _lib.HTRC_OK and n.value == 0
    assert L.htrc_norm_workspace_size(ctypes.byref(_norm(weight=256, dweight=256)), ctypes.byref(n)) == _lib.HTRC_OK
    assert n.value >= 2 * 64 * 4
    assert L.htrc_norm_workspace_size(ctypes.byref(_norm(width=0)), ctypes.byref(n)) == _lib.HTRC_ERR_ARG
    assert L.htrc_norm_workspace_size(ctypes.byref(_norm()), None) == _lib.HTRC_ERR_ARG
    assert L.htrc_norm_forward(None, None) == L.htrc_norm_backward(None, None) == _lib.HTRC_ERR_ARG


def _quantize(x=256, dtype=_lib.LAYER_F32, batch=1, tokens=2, width=64, stride=(0, 64), codes=256, pitch=64, scales=256):
    return _lib.lib().htrc_quantize_rows(x, dtype, batch, tokens, width, None if stride is None else (ctypes.c_int64 * 2)(*stride),
                                         codes, pitch, scales, None)


@pytest.mark.parametrize("kw,rc", [
    (dict(x=None), _lib.HTRC_ERR_ARG), (dict(codes=None), _lib.HTRC_ERR_ARG), (dict(scales=None), _lib.HTRC_ERR_ARG),
    (dict(stride=None), _lib.HTRC_ERR_ARG), (dict(pitch=48), _lib.HTRC_ERR_ARG), (dict(pitch=72), _lib.HTRC_ERR_ARG),
    (dict(codes=260), _lib.HTRC_ERR_ARG), (dict(dtype=5), _lib.HTRC_ERR_ARG), (dict(width=0), _lib.HTRC_ERR_ARG),
    (dict(width=16385, pitch=16400), _lib.HTRC_ERR_UNSUPPORTED), (dict(batch=-1), _lib.HTRC_ERR_ARG),
    (dict(batch=1 << 30, tokens=2), _lib.HTRC_ERR_UNSUPPORTED)])
def test_quantize_entry_refuses(kw, rc):
    assert _quantize(**kw) == rc


def _linear(**kw):
    a = _lib.HtrcLinear8Args()
    a.x = a.x_scales = a.w = a.w_scales = a.out = 256
    a.x_stride[:] = (320, 64)
    a.batch, a.tokens, a.width, a.channels = 2, 5, 64, 7
    a.dtype, a.out_dtype, a.w_pitch = _lib.LAYER_I8, _lib.LAYER_BF16, 64
    for k, v in kw.items():
        if k == "x_stride":
            a.x_stride[:] = v
        else:
            setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,rc", [
    (dict(batch=-1), _lib.HTRC_ERR_ARG), (dict(tokens=-1), _lib.HTRC_ERR_ARG), (dict(width=0), _lib.HTRC_ERR_ARG),
    (dict(channels=0), _lib.HTRC_ERR_ARG), (dict(dtype=4), _lib.HTRC_ERR_ARG), (dict(out_dtype=_lib.LAYER_I8), _lib.HTRC_ERR_ARG),
    (dict(bias_dtype=3), _lib.HTRC_ERR_ARG), (dict(width=65537, w_pitch=65552), _lib.HTRC_ERR_UNSUPPORTED),
    (dict(dtype=_lib.LAYER_F32, width=16385, w_pitch=16400), _lib.HTRC_ERR_UNSUPPORTED),
    (dict(batch=1 << 31), _lib.HTRC_ERR_UNSUPPORTED), (dict(w=None), _lib.HTRC_ERR_ARG), (dict(w_scales=None), _lib.HTRC_ERR_ARG),
    (dict(w=264), _lib.HTRC_ERR_ARG), (dict(w_pitch=48), _lib.HTRC_ERR_ARG), (dict(w_pitch=72), _lib.HTRC_ERR_ARG),
    (dict(x=None), _lib.HTRC_ERR_ARG), (dict(out=None), _lib.HTRC_ERR_ARG), (dict(x_scales=None), _lib.HTRC_ERR_ARG),
    (dict(x=257), _lib.HTRC_ERR_ARG), (dict(x_stride=(360, 72)), _lib.HTRC_ERR_ARG), (dict(x_stride=(240, 48)), _lib.HTRC_ERR_ARG),
    (dict(x_stride=(384, 64)), _lib.HTRC_ERR_ARG)])
def test_linear8_entry_refuses(kw, rc):
    assert _lib.lib().htrc_linear8_forward(ctypes.byref(_linear(**kw)), None) == rc


def test_linear8_workspace_size():
    L = _lib.lib()
    n = ctypes.c_size_t(1)
    assert L.htrc_linear8_workspace_size(ctypes.byref(_linear()), ctypes.byref(n)) == _lib.HTRC_OK and n.value == 0
    assert L.htrc_linear8_workspace_size(ctypes.byref(_linear(dtype=_lib.LAYER_F32, tokens=20)), ctypes.byref(n)) == _lib.HTRC_OK
    assert n.value >= 40 * 64 + 40 * 4
    assert L.htrc_linear8_workspace_size(ctypes.byref(_linear()), None) == _lib.HTRC_ERR_ARG
    assert L.htrc_linear8_forward(None, None) == _lib.HTRC_ERR_ARG


def test_python_layer_refuses_without_a_device():
    x = torch.zeros((4, 64), dtype=torch.bfloat16)
    rows = htrc_b200.Int8Rows(torch.zeros((8, 64), dtype=torch.int8), torch.ones(8))
    for call in (lambda: htrc_b200.layer_norm(x), lambda: htrc_b200.layer_norm_int8(x), lambda: htrc_b200.quantize_rows(x),
                 lambda: htrc_b200.int8_linear(x, rows), lambda: htrc_b200.int8_rows(*rows),
                 lambda: htrc_b200.layer_norm_backward(x, x, x, x)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


@pytest.mark.parametrize("view,pitch", [
    (lambda c: c, 160), (lambda c: c[..., :100], 160), (lambda c: c[:, :1], 3 * 160), (lambda c: c[:, 1:2, :5], 3 * 160),
    (lambda c: c[:1], 160), (lambda c: c[1, 2], 160), (lambda c: c[1, 2, :33], 48), (lambda c: c[:, :, 1:17], None),
    (lambda c: c[:, :2], None), (lambda c: c.transpose(0, 1), None), (lambda c: c[:1, :1].expand(4, 3, 160), None),
    (lambda c: c[..., ::2], None), (lambda c: c[::2, 0], 6 * 160), (lambda c: c[..., 16:49], 160)])
def test_pitch_of_codes(view, pitch):
    """Rows that stand evenly 16-byte aligned are read in place, others are laid out."""
    room = torch.zeros(4 * 3 * 160 + 16, dtype=torch.int8)
    start = -room.data_ptr() % 16
    assert linear8._pitch(view(room[start:start + 4 * 3 * 160].view(4, 3, 160))) == pitch
