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
from .linear8 import Int8Rows, _check_float_rows, _dense, _DTYPES, _new_codes, _refuse_gradients, _two_strides


def _term(t, name, shapes, width, device):
    """(tensor, type) of a parameter of one of the shapes, its last dimension dense; (None, 0) of None."""
    if t is None:
        return None, 0
    if not isinstance(t, torch.Tensor) or t.shape not in shapes or t.dtype not in _DTYPES or t.device != device:
        raise ValueError(f"{name}: {list(shapes[0])} float32, bfloat16 or float16 on x's device expected")
    if width != 1 and t.stride(-1) != 1:
        t = t.contiguous()
    return t, _DTYPES[t.dtype]


class _Call:
    """The checked arguments of one call: rows and parameters as the kernels take them."""
    __slots__ = ("x", "keep", "sizes", "kinds", "strides")

    def __init__(self, x, weight, bias, scale, shift, eps):
        _check_float_rows(x)
        if not (eps >= 0 and math.isfinite(eps)):
            raise ValueError("eps must be non-negative and finite")
        dev = x.device
        dims = x.dim()
        modulated = scale is not None or shift is not None
        if modulated and dims > 3:
            x = x.reshape(x.shape[0], math.prod(x.shape[1:-1]), x.shape[-1])
        x, batch, tokens, width, sb, sn = _two_strides(x)
        if width > _lib.NORM_MAX_WIDTH:
            raise NotImplementedError(f"rows of up to {_lib.NORM_MAX_WIDTH} elements are supported, got {width}")
        self.x = x
        w, wk = _term(weight, "weight", ((width,),), width, dev)
        b, bk = _term(bias, "bias", ((width,),), width, dev)
        # a modulation per entry of the first dimension; of rows without one, a single vector
        shapes = ((batch, width), (batch, 1, width)) if dims > 2 else ((width,), (1, width))
        s, sk = _term(scale, "scale", shapes, width, dev)
        t, tk = _term(shift, "shift", shapes, width, dev)
        self.keep = (w, b, s, t)
        self.sizes = (sb, sn, batch, tokens, width, _DTYPES[x.dtype])
        # the modulation's batch strides, the parameters' types and eps
        self.strides = tuple(0 if m is None or dims <= 2 else m.stride(0) for m in (s, t))
        self.kinds = (wk, bk, sk, tk, eps)

    @property
    def dense(self):
        """(batch, token) strides of dense rows."""
        return self.sizes[3] * self.sizes[4], self.sizes[4]


_plans = {}


def _meta(t):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


def _call(x, weight, bias, scale, shift, eps):
    """(x, parameters, sizes, strides, kinds, dense, lead, whole) of checked arguments, lead and whole being the shape and
    dense strides of a value per row and of rows.  What follows from their shapes, strides and
    types alone is kept for calls that repeat them: the checks cost more host time than the rest of a small call."""
    given = (weight, bias, scale, shift)
    try:
        key = (x.shape, x.stride(), x.dtype, x.device, _meta(weight), _meta(bias), _meta(scale), _meta(shift), eps)
        kept = _plans.get(key)
    except (AttributeError, TypeError):         # no tensors: the checks say so
        key = kept = None
    if kept is not None:
        return x, given, *kept
    c = _Call(x, weight, bias, scale, shift, eps)
    lead = tuple(x.shape[:-1])
    kept = (c.sizes, c.strides, c.kinds, c.dense, (lead, _dense(lead)), (tuple(x.shape), _dense(x.shape)))
    if key is not None and c.x.data_ptr() == x.data_ptr() and all(a is b for a, b in zip(c.keep, given)):
        if len(_plans) >= 1024:
            _plans.clear()
        _plans[key] = kept
    return c.x, c.keep, *kept


def _pointers(tensors):
    return [0 if t is None else t.data_ptr() for t in tensors]


def _like(x):
    """A dense tensor of x's shape and type."""
    return torch.empty_like(x) if x.is_contiguous() else torch.empty_like(x, memory_format=torch.contiguous_format)


_NO_BACK = (0,) * 13


def _forward(given, weight, bias, scale, shift, eps, stats):
    x, params, sizes, strides, kinds, dense, lead, whole = _call(given, weight, bias, scale, shift, eps)
    guard = _on(x.device)
    if guard is not None:
        with guard:
            return _forward(given, weight, bias, scale, shift, eps, stats)
    out = torch.empty_strided(*whole, dtype=x.dtype, device=x.device)
    mean = rstd = None
    mp = rp = 0
    if stats:
        mean = torch.empty_strided(*lead, dtype=torch.float32, device=x.device)
        rstd = torch.empty_like(mean)
        mp, rp = mean.data_ptr(), rstd.data_ptr()
    rc = lib().htrc_norm_forward(
        _lib.NORM_ARGS.pack(x.data_ptr(), *sizes, *_pointers(params), *strides, *kinds, out.data_ptr(), *dense, 0, 0, 0,
                            mp, rp, *_NO_BACK), _lib.raw_stream(x.device.index))
    if rc:
        check(rc, "htrc_norm_forward")
    return out, mean, rstd


_workspaces = {}


def _workspace_bytes(key, head):
    """What the backward asks for: it goes by sizes, strides and alignments alone (``key``)."""
    need = _workspaces.get(key)
    if need is None:
        size = ctypes.c_size_t()
        check(lib().htrc_norm_workspace_size(_lib.NORM_ARGS.pack(*head, 0, 0), size), "htrc_norm_workspace_size")
        if len(_workspaces) >= 1024:
            _workspaces.clear()
        need = _workspaces[key] = size.value
    return need


def _backward(dy, given, mean, rstd, weight, bias, scale, shift, wanted=(True,) * 4):
    """dx and the gradients of weight, bias, scale and shift: None for those that are none or not wanted."""
    x, params, sizes, strides, kinds, dense, _, whole = _call(given, weight, bias, scale, shift, 0.0)
    dev, shape = x.device, given.shape
    if not isinstance(dy, torch.Tensor) or dy.shape != shape or dy.dtype != x.dtype or dy.device != dev:
        raise ValueError(f"dy: {list(shape)} {x.dtype} on x's device expected")
    for t in (mean, rstd):
        if not isinstance(t, torch.Tensor) or t.shape != shape[:-1] or t.dtype is not torch.float32 or t.device != dev:
            raise ValueError(f"mean and rstd: {list(shape[:-1])} float32 on x's device expected")
    guard = _on(dev)
    if guard is not None:
        with guard:
            return _backward(dy, given, mean, rstd, weight, bias, scale, shift, wanted)
    mean, rstd = mean.contiguous(), rstd.contiguous()
    if dy.is_contiguous():
        gb, gn = dense
    else:
        dy, _, _, _, gb, gn = _two_strides(dy.reshape(sizes[2:5]))
    dx = torch.empty_strided(*whole, dtype=x.dtype, device=dev)
    grads, to = [], []
    for t, want in zip((weight, bias, scale, shift), wanted):
        g = _like(t) if want and t is not None else None
        grads.append(g)
        to.append(0 if g is None else g.data_ptr())
    status = _status_word(dev)
    xp, gp, terms = x.data_ptr(), dy.data_ptr(), _pointers(params)
    head = (xp, *sizes, *terms, *strides, *kinds, 0, 0, 0, 0, 0, 0, mean.data_ptr(), rstd.data_ptr(), gp, gb, gn,
            dx.data_ptr(), *dense, *to, 0 if status is None else status.data_ptr())
    ws, wp, need = None, 0, 0
    if any(to):
        need = _workspace_bytes((sizes, gb, gn, xp & 15, gp & 15, terms[0] != 0, terms[2] != 0, terms[3] != 0, dev.index), head)
        ws = torch.empty_strided((need,), (1,), dtype=torch.uint8, device=dev)
        wp = ws.data_ptr()
    rc = lib().htrc_norm_backward(_lib.NORM_ARGS.pack(*head, wp, need), _lib.raw_stream(dev.index))
    if rc:
        check(rc, "htrc_norm_backward")
    return (dx, *grads)


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, scale, shift, eps):
        y, mean, rstd = _forward(x, weight, bias, scale, shift, eps, True)
        ctx.save_for_backward(x, weight, bias, scale, shift, mean, rstd)
        ctx.mark_non_differentiable(mean, rstd)
        ctx.set_materialize_grads(False)
        return y, mean, rstd

    @staticmethod
    def backward(ctx, dy, *_):
        if dy is None:
            return (None,) * 6
        *given, mean, rstd = ctx.saved_tensors
        grads = _backward(dy, given[0], mean, rstd, *given[1:], ctx.needs_input_grad[1:5])
        return (*first_order("layer_norm", grads, (*given, dy)), None)


def layer_norm(x, *, weight=None, bias=None, scale=None, shift=None, eps=1e-6, return_stats=False):
    """x [.., width] normalised, in x's type, dense.  weight, bias: [width]; scale, shift: [batch, width] (or
    [batch, 1, width]), batch being x's first dimension, or [width] where x is [tokens, width].

    return_stats: also the rows' float32 mean and rstd [..], which ``layer_norm_backward`` takes and no gradient
    passes."""
    if recorded(x, weight, bias, scale, shift):
        y, mean, rstd = _Norm.apply(x, weight, bias, scale, shift, eps)
    else:
        y, mean, rstd = _forward(x, weight, bias, scale, shift, eps, return_stats)
    return (y, mean, rstd) if return_stats else y


def layer_norm_backward(dy, x, mean, rstd, *, weight=None, bias=None, scale=None, shift=None):
    """(dx, dweight, dbias, dscale, dshift) of ``layer_norm`` for its result's gradient dy and its statistics, each in
    its tensor's type, None for what is None."""
    return _backward(dy, x, mean, rstd, weight, bias, scale, shift)


def layer_norm_int8(x, *, weight=None, bias=None, scale=None, shift=None, eps=1e-6):
    """``layer_norm``'s float32 result as ``Int8Rows``, without its rows ever being written."""
    _refuse_gradients("layer_norm_int8", x, weight, bias, scale, shift)
    return _codes(x, weight, bias, scale, shift, eps)


def _codes(given, *terms):
    x, params, sizes, strides, kinds, _, lead, whole = _call(given, *terms)
    guard = _on(x.device)
    if guard is not None:
        with guard:
            return _codes(given, *terms)
    if sizes[4] % 16:
        codes, pitch = _new_codes(given.shape, given)
    else:
        codes, pitch = torch.empty_strided(*whole, dtype=torch.int8, device=x.device), sizes[4]
    scales = torch.empty_strided(*lead, dtype=torch.float32, device=x.device)
    rc = lib().htrc_norm_forward(
        _lib.NORM_ARGS.pack(x.data_ptr(), *sizes, *_pointers(params), *strides, *kinds, 0, 0, 0, codes.data_ptr(), pitch,
                            scales.data_ptr(), 0, 0, *_NO_BACK), _lib.raw_stream(x.device.index))
    if rc:
        check(rc, "htrc_norm_forward")
    return Int8Rows(codes, scales)
