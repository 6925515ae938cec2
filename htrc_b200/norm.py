"""Layer norm of a video transformer's residual stream, with a learned affine and the modulation that its timestep gives
each batch entry, forward and backward (``csrc/norm.cu``).

    y = layer_norm(x, weight=w, bias=b)                      # [.., width]
    y = layer_norm(x, scale=s, shift=t)                      # s, t [batch, width]: norm(x) (1 + s) + t
    rows = layer_norm_int8(x, scale=s, shift=t)              # the same in 8-bit rows, for int8_linear

``u = (x - mean) * rstd`` with ``rstd = rsqrt(variance + eps)`` over the width, then
``y = (u * weight + bias) * (1 + scale) + shift``; what is None is left out.  x: float32, bfloat16 or float16 with any
strides but a unit last one, parameters in any of these types; arithmetic is float32, rounded once.  ``layer_norm`` takes
part in autograd (first derivatives, reverse mode); its backward can also be called by itself.  There is no CPU path.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from ._autograd import first_order, recorded
from ._lib import check, lib
from .cross import _on, _status_word
from .linear8 import Int8Rows, _check_float_rows, _DTYPES, _new_codes, _refuse_gradients, _two_strides


class _Call:
    """The checked arguments of one call: rows and parameters as the kernels take them."""
    __slots__ = ("x", "shape", "dtype", "device", "batch", "tokens", "width", "head", "terms", "keep", "params")

    def __init__(self, x, weight, bias, scale, shift, eps):
        _check_float_rows(x)
        if not (eps >= 0 and math.isfinite(eps)):
            raise ValueError("eps must be non-negative and finite")
        self.shape, self.dtype, self.device = x.shape, x.dtype, x.device
        self.params = (weight, bias, scale, shift)
        modulated = scale is not None or shift is not None
        if modulated and x.dim() > 3:
            x = x.reshape(x.shape[0], math.prod(x.shape[1:-1]), x.shape[-1])
        x, self.batch, self.tokens, self.width, sb, sn = _two_strides(x)
        width = self.width
        if width > _lib.NORM_MAX_WIDTH:
            raise NotImplementedError(f"rows of up to {_lib.NORM_MAX_WIDTH} elements are supported, got {width}")
        self.x = x
        pointers, strides, kinds, self.keep = [], [], [], []
        for name, t in (("weight", weight), ("bias", bias)):
            if t is None:
                pointers.append(0)
                kinds.append(0)
                continue
            if not isinstance(t, torch.Tensor) or t.shape != (width,) or t.dtype not in _DTYPES or t.device != x.device:
                raise ValueError(f"{name}: [{width}] float32, bfloat16 or float16 on x's device expected")
            t = t.contiguous()
            self.keep.append(t)
            pointers.append(t.data_ptr())
            kinds.append(_DTYPES[t.dtype])
        # a modulation per entry of the first dimension; of rows without one, a single vector
        want = (self.batch, width) if len(self.shape) > 2 else (width,)
        for name, t in (("scale", scale), ("shift", shift)):
            if t is None:
                pointers.append(0)
                kinds.append(0)
                strides.append(0)
                continue
            if not isinstance(t, torch.Tensor) or t.shape not in (want, (*want[:-1], 1, width)) or \
                    t.dtype not in _DTYPES or t.device != x.device:
                raise ValueError(f"{name}: {list(want)} float32, bfloat16 or float16 on x's device expected")
            if t.stride(-1) != 1 and width != 1:
                t = t.contiguous()
            self.keep.append(t)
            pointers.append(t.data_ptr())
            kinds.append(_DTYPES[t.dtype])
            strides.append(t.stride(0) if len(want) == 2 else 0)
        self.head = (x.data_ptr(), sb, sn, self.batch, self.tokens, width, _DTYPES[x.dtype])
        self.terms = (*pointers, *strides, *kinds, eps)

    def rows(self):
        """(batch, token) strides of dense rows."""
        return self.tokens * self.width, self.width

    def statistics(self):
        return (torch.empty(self.shape[:-1], dtype=torch.float32, device=self.device) for _ in range(2))


_NO_BACK = (0,) * 13


def _forward(c, stats):
    guard = _on(c.device)
    if guard is not None:
        with guard:
            return _forward(c, stats)
    out = torch.empty(c.shape, dtype=c.dtype, device=c.device)
    mean, rstd = c.statistics() if stats else (None, None)
    args = _lib.NORM_ARGS.pack(*c.head, *c.terms, out.data_ptr(), *c.rows(), 0, 0, 0, mean.data_ptr() if stats else 0,
                               rstd.data_ptr() if stats else 0, *_NO_BACK)
    rc = lib().htrc_norm_forward(args, _lib.raw_stream(c.device.index))
    if rc:
        check(rc, "htrc_norm_forward")
    return out, mean, rstd


def _backward(c, dy, mean, rstd, wanted=(True,) * 4):
    """dx and the gradients of weight, bias, scale and shift: None for those that are none or not wanted."""
    if not isinstance(dy, torch.Tensor) or dy.shape != c.shape or dy.dtype != c.dtype or dy.device != c.device:
        raise ValueError(f"dy: {list(c.shape)} {c.dtype} on x's device expected")
    for name, t in (("mean", mean), ("rstd", rstd)):
        if not isinstance(t, torch.Tensor) or t.shape != c.shape[:-1] or t.dtype is not torch.float32 or t.device != c.device:
            raise ValueError(f"{name}: {list(c.shape[:-1])} float32 on x's device expected")
    guard = _on(c.device)
    if guard is not None:
        with guard:
            return _backward(c, dy, mean, rstd, wanted)
    mean, rstd = mean.contiguous(), rstd.contiguous()
    if dy.dim() > 3:
        dy = dy.reshape(c.batch, c.tokens, c.width)
    dy, _, _, _, gb, gn = _two_strides(dy)
    dx = torch.empty(c.shape, dtype=c.dtype, device=c.device)
    grads = [torch.empty(t.shape, dtype=t.dtype, device=c.device) if t is not None and want else None
             for t, want in zip(c.params, wanted)]
    status = _status_word(c.device)
    tail = (dy.data_ptr(), gb, gn, dx.data_ptr(), *c.rows(), *(0 if g is None else g.data_ptr() for g in grads),
            0 if status is None else status.data_ptr())
    head = (*c.head, *c.terms, 0, 0, 0, 0, 0, 0, mean.data_ptr(), rstd.data_ptr(), *tail)
    ws, wp, need = None, 0, 0
    if any(g is not None for g in grads):
        size = ctypes.c_size_t()
        check(lib().htrc_norm_workspace_size(_lib.NORM_ARGS.pack(*head, 0, 0), size), "htrc_norm_workspace_size")
        need = size.value
        ws = torch.empty(need, dtype=torch.uint8, device=c.device)
        wp = ws.data_ptr()
    rc = lib().htrc_norm_backward(_lib.NORM_ARGS.pack(*head, wp, need), _lib.raw_stream(c.device.index))
    if rc:
        check(rc, "htrc_norm_backward")
    return (dx, *grads)


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, scale, shift, eps):
        y, mean, rstd = _forward(_Call(x, weight, bias, scale, shift, eps), True)
        ctx.save_for_backward(x, weight, bias, scale, shift, mean, rstd)
        ctx.eps = eps
        ctx.mark_non_differentiable(mean, rstd)
        ctx.set_materialize_grads(False)
        return y, mean, rstd

    @staticmethod
    def backward(ctx, dy, *_):
        if dy is None:
            return (None,) * 6
        *given, mean, rstd = ctx.saved_tensors
        grads = _backward(_Call(*given, ctx.eps), dy, mean, rstd, ctx.needs_input_grad[1:5])
        return (*first_order("layer_norm", grads, (*given, dy)), None)


def layer_norm(x, *, weight=None, bias=None, scale=None, shift=None, eps=1e-6, return_stats=False):
    """x [.., width] normalised, in x's type, dense.  weight, bias: [width]; scale, shift: [batch, width] (or
    [batch, 1, width]), batch being x's first dimension, or [width] where x is [tokens, width].

    return_stats: also the rows' float32 mean and rstd [..], which ``layer_norm_backward`` takes and no gradient
    passes."""
    if recorded(x, weight, bias, scale, shift):
        y, mean, rstd = _Norm.apply(x, weight, bias, scale, shift, eps)
    else:
        y, mean, rstd = _forward(_Call(x, weight, bias, scale, shift, eps), return_stats)
    return (y, mean, rstd) if return_stats else y


def layer_norm_backward(dy, x, mean, rstd, *, weight=None, bias=None, scale=None, shift=None):
    """(dx, dweight, dbias, dscale, dshift) of ``layer_norm`` for its result's gradient dy and its statistics, each in
    its tensor's type, None for what is None."""
    return _backward(_Call(x, weight, bias, scale, shift, 0.0), dy, mean, rstd)


def layer_norm_int8(x, *, weight=None, bias=None, scale=None, shift=None, eps=1e-6):
    """``layer_norm``'s float32 result as ``Int8Rows``, without its rows ever being written."""
    _refuse_gradients("layer_norm_int8", x, weight, bias, scale, shift)
    return _codes(_Call(x, weight, bias, scale, shift, eps))


def _codes(c):
    guard = _on(c.device)
    if guard is not None:
        with guard:
            return _codes(c)
    codes, pitch = _new_codes(c.shape, c.device)
    scales = torch.empty(c.shape[:-1], dtype=torch.float32, device=c.device)
    args = _lib.NORM_ARGS.pack(*c.head, *c.terms, 0, 0, 0, codes.data_ptr(), pitch, scales.data_ptr(), 0, 0, *_NO_BACK)
    rc = lib().htrc_norm_forward(args, _lib.raw_stream(c.device.index))
    if rc:
        check(rc, "htrc_norm_forward")
    return Int8Rows(codes, scales)
