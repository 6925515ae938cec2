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


def _term(t, name, shapes, width, device):
    """(tensor, pointer, type) of a parameter of one of the shapes, its last dimension dense; (None, 0, 0) of None."""
    if t is None:
        return None, 0, 0
    if not isinstance(t, torch.Tensor) or t.shape not in shapes or t.dtype not in _DTYPES or t.device != device:
        raise ValueError(f"{name}: {list(shapes[0])} float32, bfloat16 or float16 on x's device expected")
    if width != 1 and t.stride(-1) != 1:
        t = t.contiguous()
    return t, t.data_ptr(), _DTYPES[t.dtype]


class _Call:
    """The checked arguments of one call: rows and parameters as the kernels take them."""
    __slots__ = ("x", "given", "device", "head", "terms", "keep", "params", "dense")

    def __init__(self, x, weight, bias, scale, shift, eps):
        _check_float_rows(x)
        if not (eps >= 0 and math.isfinite(eps)):
            raise ValueError("eps must be non-negative and finite")
        self.given = x
        dev = self.device = x.device
        dims = x.dim()
        modulated = scale is not None or shift is not None
        if modulated and dims > 3:
            x = x.reshape(x.shape[0], math.prod(x.shape[1:-1]), x.shape[-1])
        x, batch, tokens, width, sb, sn = _two_strides(x)
        if width > _lib.NORM_MAX_WIDTH:
            raise NotImplementedError(f"rows of up to {_lib.NORM_MAX_WIDTH} elements are supported, got {width}")
        self.x = x
        self.params = (weight, bias, scale, shift)
        self.keep = ()
        self.terms = (0, 0, 0, 0, 0, 0, 0, 0, 0, 0, eps)
        if modulated or weight is not None or bias is not None:
            w, wp, wk = _term(weight, "weight", ((width,),), width, dev)
            b, bp, bk = _term(bias, "bias", ((width,),), width, dev)
            sp = sk = ss = tp = tk = ts = 0
            s = t = None
            if modulated:
                # a modulation per entry of the first dimension; of rows without one, a single vector
                shapes = ((batch, width), (batch, 1, width)) if dims > 2 else ((width,), (1, width))
                s, sp, sk = _term(scale, "scale", shapes, width, dev)
                t, tp, tk = _term(shift, "shift", shapes, width, dev)
                if dims > 2:
                    ss = 0 if s is None else s.stride(0)
                    ts = 0 if t is None else t.stride(0)
            self.keep = (w, b, s, t)
            self.terms = (wp, bp, sp, tp, ss, ts, wk, bk, sk, tk, eps)
        self.head = (x.data_ptr(), sb, sn, batch, tokens, width, _DTYPES[x.dtype])
        self.dense = (tokens * width, width)         # (batch, token) strides of dense rows


_NO_BACK = (0,) * 13


def _like(x):
    """A dense tensor of x's shape and type."""
    return torch.empty_like(x) if x.is_contiguous() else torch.empty_like(x, memory_format=torch.contiguous_format)


def _forward(c, stats):
    guard = _on(c.device)
    if guard is not None:
        with guard:
            return _forward(c, stats)
    x = c.given
    out = _like(x)
    mean = rstd = None
    mp = rp = 0
    if stats:
        mean = x.new_empty(x.shape[:-1], dtype=torch.float32)
        rstd = torch.empty_like(mean)
        mp, rp = mean.data_ptr(), rstd.data_ptr()
    args = _lib.NORM_ARGS.pack(*c.head, *c.terms, out.data_ptr(), *c.dense, 0, 0, 0, mp, rp, *_NO_BACK)
    rc = lib().htrc_norm_forward(args, _lib.raw_stream(c.device.index))
    if rc:
        check(rc, "htrc_norm_forward")
    return out, mean, rstd


_workspaces = {}


def _workspace_bytes(key, args):
    """What the backward asks for: it goes by sizes, strides and alignments alone (``key``)."""
    need = _workspaces.get(key)
    if need is None:
        size = ctypes.c_size_t()
        check(lib().htrc_norm_workspace_size(args, size), "htrc_norm_workspace_size")
        if len(_workspaces) >= 1024:
            _workspaces.clear()
        need = _workspaces[key] = size.value
    return need


def _backward(c, dy, mean, rstd, wanted=(True,) * 4):
    """dx and the gradients of weight, bias, scale and shift: None for those that are none or not wanted."""
    x, dev = c.given, c.device
    shape = x.shape
    if not isinstance(dy, torch.Tensor) or dy.shape != shape or dy.dtype != x.dtype or dy.device != dev:
        raise ValueError(f"dy: {list(shape)} {x.dtype} on x's device expected")
    for t in (mean, rstd):
        if not isinstance(t, torch.Tensor) or t.shape != shape[:-1] or t.dtype is not torch.float32 or t.device != dev:
            raise ValueError(f"mean and rstd: {list(shape[:-1])} float32 on x's device expected")
    guard = _on(dev)
    if guard is not None:
        with guard:
            return _backward(c, dy, mean, rstd, wanted)
    mean, rstd = mean.contiguous(), rstd.contiguous()
    if dy.dim() > 3:
        dy = dy.reshape(c.x.shape)
    dy, _, _, _, gb, gn = _two_strides(dy)
    dx = _like(x)
    grads = [_like(t) if t is not None and want else None for t, want in zip(c.params, wanted)]
    pointers = [0 if g is None else g.data_ptr() for g in grads]
    status = _status_word(dev)
    gp = dy.data_ptr()
    head = (*c.head, *c.terms, 0, 0, 0, 0, 0, 0, mean.data_ptr(), rstd.data_ptr(), gp, gb, gn, dx.data_ptr(), *c.dense,
            *pointers, 0 if status is None else status.data_ptr())
    ws, wp, need = None, 0, 0
    if any(pointers):
        w, _, s, t = (p != 0 for p in c.terms[:4])
        need = _workspace_bytes((*c.head[1:], gb, gn, c.head[0] & 15, gp & 15, w, s, t, dev.index),
                                _lib.NORM_ARGS.pack(*head, 0, 0))
        ws = x.new_empty((need,), dtype=torch.uint8)
        wp = ws.data_ptr()
    rc = lib().htrc_norm_backward(_lib.NORM_ARGS.pack(*head, wp, need), _lib.raw_stream(dev.index))
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
    x = c.given
    codes, pitch = _new_codes(x.shape, x)
    scales = x.new_empty(x.shape[:-1], dtype=torch.float32)
    args = _lib.NORM_ARGS.pack(*c.head, *c.terms, 0, 0, 0, codes.data_ptr(), pitch, scales.data_ptr(), 0, 0, *_NO_BACK)
    rc = lib().htrc_norm_forward(args, _lib.raw_stream(c.device.index))
    if rc:
        check(rc, "htrc_norm_forward")
    return Int8Rows(codes, scales)
