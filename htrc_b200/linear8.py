"""The matrix product in 8-bit integers with a scale for each token and each channel (``csrc/linear8.cu``, tcgen05), as a
layer's projections use it, and the 8-bit rows that it reads.

    w = quantize_rows(weight)                                 # once: [channels, width] -> codes and a scale per channel
    y = int8_linear(x, w, bias=bias)                          # rows quantised on the way: [.., width] -> [.., channels]
    y = int8_linear(layer_norm_int8(x, scale=s, shift=t), w)  # rows that a norm wrote in 8 bits

A row's codes are the integers nearest ``x * (127 / top)``, ties to even, and its scale is ``top / 127``, with ``top`` its
largest magnitude (at least 1e-30), all in float32; a row with a NaN or an infinity has the scale NaN, and so do its
products.  The product's sums are exact 32-bit integers; scales and bias are applied in float32 and rounded once.

These functions are for inference: they have no gradients and refuse inputs that record them.  There is no CPU path.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib
from ._autograd import recorded
from ._lib import check, lib
from .cross import _on, _status_word, cross_status

_DTYPES = {torch.float32: _lib.LAYER_F32, torch.bfloat16: _lib.LAYER_BF16, torch.float16: _lib.LAYER_F16}


class Int8Rows(NamedTuple):
    """Rows in 8-bit integers: ``codes`` [.., width] int8 and ``scales`` [..] float32, a row's values codes * scale."""
    codes: torch.Tensor
    scales: torch.Tensor


def _check_codes(rows, name):
    if not isinstance(rows, tuple) or len(rows) != 2:
        raise ValueError(f"{name}: Int8Rows (codes, scales) expected")
    codes, scales = rows
    if not isinstance(codes, torch.Tensor) or not isinstance(scales, torch.Tensor) or codes.dtype is not torch.int8 or \
            codes.dim() < 1 or scales.dtype is not torch.float32 or scales.shape != codes.shape[:-1]:
        raise ValueError(f"{name}: int8 codes [.., width] and float32 scales [..] expected")
    if not codes.is_cuda or scales.device != codes.device:
        raise ValueError(f"{name} must be on one CUDA device (there is no CPU path)")
    return codes, scales


def _pitch(codes):
    """The even distance between the rows of codes [.., width] as the kernels read them, or None."""
    shape, stride = codes.shape, codes.stride()
    if codes.data_ptr() & 15 or (stride[-1] != 1 and shape[-1] != 1):
        return None
    if 0 in shape[:-1]:                   # no rows, whatever their strides
        return (shape[-1] + 15) // 16 * 16
    pitch = covered = None
    for i in range(len(shape) - 2, -1, -1):
        n = shape[i]
        if n == 1:
            continue
        s = stride[i]
        if pitch is None:
            pitch = s
        elif s != covered:
            return None
        covered = s * n
    if pitch is None:
        return (shape[-1] + 15) // 16 * 16
    return pitch if pitch >= shape[-1] and not pitch & 15 else None


def _dense(shape):
    """The strides of a dense tensor (with them ``empty_strided`` is the cheapest allocation there is)."""
    strides, n = [], 1
    for size in reversed(shape):
        strides.append(n)
        n *= max(1, size)
    return tuple(reversed(strides))


def _new_codes(shape, like):
    """Codes [.., width] on the tensor's device whose rows start at multiples of 16 bytes: (codes, pitch)."""
    width = shape[-1]
    pitch = (width + 15) // 16 * 16
    if pitch == width:
        return torch.empty_strided(shape, _dense(shape), dtype=torch.int8, device=like.device), pitch
    return like.new_empty((*shape[:-1], pitch), dtype=torch.int8)[..., :width], pitch


def int8_rows(codes, scales):
    """``Int8Rows`` laid out as the kernels read them (codes whose rows start at even multiples of 16 bytes are taken as
    they are), so that no product has to."""
    codes, scales = _check_codes((codes, scales), "rows")
    if _pitch(codes) is None:
        laid, _ = _new_codes(codes.shape, codes)
        codes = laid.copy_(codes)
    return Int8Rows(codes, scales.contiguous())


def _two_strides(x):
    """x [.., width] as (tensor, batch, tokens, width, batch stride, token stride); a copy only where its strides need one."""
    d = x.dim()
    if d > 3:
        x = x.reshape(-1, x.shape[-2], x.shape[-1]) if x.numel() else x.new_empty((0, 1, x.shape[-1]))
    shape, stride = x.shape, x.stride()
    w = shape[-1]
    if w < 1:
        raise ValueError("rows of at least one element expected")
    if stride[-1] != 1 and w != 1:
        x = x.contiguous()
        stride = x.stride()
    if d >= 3:
        return x, shape[0], shape[1], w, stride[0], stride[1]
    if d == 2:
        return x, 1, shape[0], w, 0, stride[0]
    return x, 1, 1, w, 0, 0


def _check_float_rows(x):
    if not isinstance(x, torch.Tensor) or x.dtype not in _DTYPES or x.dim() < 1:
        raise ValueError("x: float32, bfloat16 or float16 rows [.., width] expected")
    if not x.is_cuda:
        raise ValueError("x must be a CUDA tensor (there is no CPU path)")


def _refuse_gradients(what, *tensors):
    if recorded(*tensors):
        raise NotImplementedError(f"{what} has no gradients: call it under torch.no_grad() or with detached tensors")


def quantize_rows(x):
    """``Int8Rows`` of float32, bfloat16 or float16 rows x [.., width] (any strides), a scale per row."""
    _check_float_rows(x)
    _refuse_gradients("quantize_rows", x)
    guard = _on(x.device)
    if guard is not None:
        with guard:
            return quantize_rows(x)
    shape = x.shape
    kept, b, n, w, sb, sn = _two_strides(x)
    if w > _lib.NORM_MAX_WIDTH:
        raise NotImplementedError(f"rows of up to {_lib.NORM_MAX_WIDTH} elements are supported, got {w}")
    codes, pitch = _new_codes(shape, x)
    scales = torch.empty_strided(shape[:-1], _dense(shape[:-1]), dtype=torch.float32, device=x.device)
    check(lib().htrc_quantize_rows(kept.data_ptr(), _DTYPES[x.dtype], b, n, w, (ctypes.c_int64 * 2)(sb, sn),
                                   codes.data_ptr(), pitch, scales.data_ptr(), _lib.raw_stream(x.device.index)),
          "htrc_quantize_rows")
    return Int8Rows(codes, scales)


def int8_linear_status(device=None):
    """Raise if a kernel of this library's layer operators on the device reported a failed guard since the last check
    (synchronises); the same word as ``cross_status``."""
    return cross_status(device)


_plans = {}


def _meta(t):
    return (t.shape, t.stride(), t.dtype, t.device)


def int8_linear(x, weight, *, bias=None, dtype=None):
    """x [.., width], as float rows (quantised on the way) or ``Int8Rows``, times weight (``Int8Rows`` of
    [channels, width]) -> [.., channels] in ``dtype``: x's by default, bfloat16 for ``Int8Rows``.

    bias: [channels] float32, bfloat16 or float16."""
    floats = isinstance(x, torch.Tensor)
    # what follows from shapes, strides and types alone is kept for calls that repeat them: the checks cost more host time
    # than the rest of a small call
    try:
        wc, ws = weight
        rows, xs = (x, None) if floats else x
        key = (_meta(rows), None if floats else _meta(xs), _meta(wc), _meta(ws), None if bias is None else _meta(bias), dtype)
        kept = isinstance(weight, tuple) and (floats or isinstance(x, tuple))       # (pairs of another type are refused)
        plan = _plans.get(key) if kept and not (wc.data_ptr() & 15 or (not floats and rows.data_ptr() & 15)) else None
        _refuse_gradients("int8_linear", rows, xs, ws, bias)
    except (AttributeError, TypeError, ValueError):       # no tensors: the checks say so
        key = plan = None
    if plan is None:
        rows, xs, wc, ws, bias, plan, whole = _plan(x, weight, bias, dtype, floats)
        if whole and key is not None:
            if len(_plans) >= 1024:
                _plans.clear()
            _plans[key] = plan
    dev, sizes, wpitch, kinds, shape, strides, dtype, need = plan
    guard = _on(dev)
    if guard is not None:
        with guard:
            return int8_linear(x, weight, bias=bias, dtype=dtype)
    out = torch.empty_strided(shape, strides, dtype=dtype, device=dev)
    wp = 0
    if need:
        workspace = torch.empty_strided((need,), (1,), dtype=torch.uint8, device=dev)
        wp = workspace.data_ptr()
    status = _status_word(dev)
    sb, sn, *rest = sizes
    rc = lib().htrc_linear8_forward(
        _lib.LINEAR8_ARGS.pack(rows.data_ptr(), sb, sn, 0 if floats else xs.data_ptr(), *rest, wc.data_ptr(), wpitch,
                               ws.data_ptr(), 0 if bias is None else bias.data_ptr(), *kinds, out.data_ptr(),
                               0 if status is None else status.data_ptr(), wp, need), _lib.raw_stream(dev.index))
    if rc:
        check(rc, "htrc_linear8_forward")
    return out


def _plan(x, weight, bias, dtype, floats):
    """The call's operands as the kernels read them, what follows from their shapes, strides and types, and whether every
    operand is read as it was given."""
    wc, ws = _check_codes(weight, "weight")
    if wc.dim() != 2 or wc.shape[0] < 1 or wc.shape[1] < 1:
        raise ValueError("weight: Int8Rows of [channels, width] expected")
    if floats:
        _check_float_rows(x)
        rows, xs = x, None
    else:
        rows, xs = _check_codes(x, "x")
    dev = rows.device
    channels, width = wc.shape
    if rows.shape[-1] != width:
        raise ValueError(f"x: rows of {width} elements expected, got {rows.shape[-1]}")
    most = _lib.NORM_MAX_WIDTH if floats else _lib.LINEAR8_MAX_WIDTH
    if width > most:
        raise NotImplementedError(f"rows of up to {most} elements are supported, got {width}")
    if wc.device != dev:
        raise ValueError("weight: x's device expected")
    if bias is not None and (not isinstance(bias, torch.Tensor) or bias.shape != (channels,) or bias.dtype not in _DTYPES or
                             bias.device != dev):
        raise ValueError(f"bias: [{channels}] float32, bfloat16 or float16 on x's device expected")
    if dtype is None:
        dtype = x.dtype if floats else torch.bfloat16
    elif dtype not in _DTYPES:
        raise ValueError("dtype: float32, bfloat16 or float16 expected")
    given = (rows, xs, wc, ws, bias)
    shape = (*rows.shape[:-1], channels)
    with torch.cuda.device(dev):
        wpitch = _pitch(wc)
        if wpitch is None:
            wc, ws = int8_rows(wc, ws)
            wpitch = _pitch(wc)
        ws = ws.contiguous()
        bias = None if bias is None else bias.contiguous()
        if floats:
            rows, b, n, _, sb, sn = _two_strides(rows)
        else:
            sn = _pitch(rows)
            if sn is None:
                rows, xs = int8_rows(rows, xs)
                sn = _pitch(rows)
            xs = xs.contiguous()
            b, n, sb = 1, xs.numel(), 0
    sizes = (sb, sn, b, n, width, channels, _DTYPES[rows.dtype] if floats else _lib.LAYER_I8)
    kinds = (0 if bias is None else _DTYPES[bias.dtype], _DTYPES[dtype])
    size = ctypes.c_size_t()
    with torch.cuda.device(dev):
        check(lib().htrc_linear8_workspace_size(_lib.LINEAR8_ARGS.pack(0, sb, sn, 0, *sizes[2:], 0, wpitch, 0, 0, *kinds, 0, 0, 0, 0),
                                                size), "htrc_linear8_workspace_size")
    need = size.value
    used = (rows, xs, wc, ws, bias)
    whole = all(a is b or (a is not None and b is not None and a.data_ptr() == b.data_ptr() and a.numel() == b.numel())
                for a, b in zip(given, used))
    return *used, (dev, sizes, wpitch, kinds, shape, _dense(shape), dtype, need), whole
