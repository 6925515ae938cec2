"""Rotary positions over several axes (time, height, width) for the queries and keys of a video transformer's
attention, with the per-head RMS norm that precedes them and the change from a projection's token-major rows to the
head-major rows that ``flat_attention_heads`` takes, in one pass over the data (``csrc/rotary.cu``).

    q, k = rotary_qk(q, k, grid_positions((t, h, w)), axes=(44, 42, 42), q_weight=wq, k_weight=wk, heads_first=True)
    out = flat_attention_heads(q[0], k[0], v, **PROD, leaf=64)

A head's first ``sum(axes)`` elements are rotated, ``axes[a]`` of them by the token's position on axis ``a``: pair ``i``
of an axis of width ``w`` turns by ``position * theta ** (-2 i / w)`` (or ``position * freqs[...]``).  Pairs are
``(2 i, 2 i + 1)`` ("interleaved") or ``(i, i + R / 2)`` of the rotated width R ("half"); the rest of the head is left
as it is.  With a weight, the row is first normalised: ``x * rsqrt(mean(x ** 2) + eps) * weight``.

Inputs are float32, bfloat16 or float16 with any strides but a unit last one (slices of a joint projection are read in
place); arithmetic is float32, rounded once to the input's type.  The functions take part in autograd (first derivatives, reverse
mode); the backward passes can also be called by themselves.  There is no CPU path.
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import _lib
from ._autograd import first_order, recorded
from ._lib import check, lib

_DTYPES = {torch.float32: _lib.LAYER_F32, torch.bfloat16: _lib.LAYER_BF16, torch.float16: _lib.LAYER_F16}


def grid_positions(grid, *, start=None, device="cuda"):
    """int32 positions [prod(grid), len(grid)] of a latent grid's tokens in row-major order, from ``start`` on."""
    sizes = [int(g) for g in grid]
    if not sizes or min(sizes) < 0:
        raise ValueError("grid: one non-negative size per axis")
    first = [0] * len(sizes) if start is None else [int(x) for x in start]
    if len(first) != len(sizes):
        raise ValueError("start: one position per axis")
    at = [torch.arange(x, x + g, dtype=torch.int32, device=device) for x, g in zip(first, sizes)]
    return torch.stack([a.reshape(-1) for a in torch.meshgrid(*at, indexing="ij")], -1)


class _Spec:
    """The arguments that do not depend on the tensors, checked."""
    __slots__ = ("axes", "theta", "pairs", "eps", "freqs", "heads_first", "rotated", "table", "n_axes")

    def __init__(self, axes, theta, pairs, eps, freqs, heads_first):
        if not axes or min(axes) < 0 or any(w % 2 for w in axes):
            raise ValueError("axes: an even number of rotated elements per axis")
        if len(axes) > _lib.ROTARY_MAX_AXES:
            raise NotImplementedError(f"more than {_lib.ROTARY_MAX_AXES} axes")
        if pairs not in _lib.ROTARY_PAIRS:
            raise ValueError("pairs must be 'interleaved' or 'half'")
        if not (theta > 0 and math.isfinite(theta)):
            raise ValueError("theta must be positive and finite")
        if not (eps >= 0 and math.isfinite(eps)):
            raise ValueError("eps must be non-negative and finite")
        self.table = None
        if freqs is not None:
            if len(freqs) != sum(axes) // 2 or not all(math.isfinite(f) for f in freqs):
                raise ValueError("freqs: one finite frequency for each of the sum(axes) / 2 pairs")
            self.table = (ctypes.c_double * max(1, len(freqs)))(*freqs)
        self.rotated, self.n_axes = sum(axes), len(axes)
        self.axes = axes + (0,) * (_lib.ROTARY_MAX_AXES - len(axes))
        self.theta, self.pairs, self.eps = float(theta), _lib.ROTARY_PAIRS[pairs], float(eps)
        self.freqs = 0 if self.table is None else ctypes.addressof(self.table)
        self.heads_first = heads_first


_specs = functools.lru_cache(maxsize=64)(_Spec)


def _spec(axes, theta, pairs, eps, freqs, heads_first):
    if type(axes) is not tuple:
        axes = tuple(int(w) for w in axes)
    return _specs(axes, theta, pairs, eps, None if freqs is None else tuple(float(f) for f in freqs), bool(heads_first))


def _check_rows(x, name):
    if not isinstance(x, torch.Tensor) or x.dim() not in (3, 4):
        raise ValueError(f"{name}: [tokens, heads, dim] or [batch, tokens, heads, dim] expected")
    if x.dtype not in _DTYPES:
        raise ValueError(f"{name}: float32, bfloat16 or float16 expected, got {x.dtype}")
    if not x.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (there is no CPU path)")


def _check(spec, tensors, weights, positions):
    """Raises for what the kernels do not take; the positions as int32 or float32."""
    x = tensors[0]
    _check_rows(x, "x")
    shape, dtype, dev = x.shape, x.dtype, x.device
    dim = shape[-1]
    if not 2 <= dim <= _lib.ROTARY_MAX_DIM:
        raise NotImplementedError(f"heads of 2 to {_lib.ROTARY_MAX_DIM} elements are supported, got {dim}")
    if spec.rotated > dim:
        raise ValueError(f"axes rotate {spec.rotated} of {dim} elements")
    for t in tensors:
        if t is not x:
            _check_rows(t, "k")
            if t.dtype != dtype or t.device != dev or t.shape[:-2] != shape[:-2] or t.shape[-1] != dim:
                raise ValueError("k: q's type, device, batch, tokens and dim expected")
        if not 1 <= t.shape[-2] <= _lib.ROTARY_MAX_HEADS:
            raise NotImplementedError(f"1 to {_lib.ROTARY_MAX_HEADS} heads are supported")
    for w in weights:
        if w is not None and (w.dim() != 1 or w.shape[0] != dim or w.dtype not in _DTYPES or w.device != dev):
            raise ValueError(f"weight: [{dim}] float32, bfloat16 or float16 on the rows' device expected")
    at = positions.shape if isinstance(positions, torch.Tensor) and positions.device == dev else ()
    if len(at) not in (2, len(shape) - 1) or at[-2] != shape[-3] or (len(at) == 3 and at[0] not in (1, shape[0])):
        raise ValueError("positions: [tokens, axes] or [batch, tokens, axes] on the rows' device expected")
    if at[-1] != spec.n_axes:
        raise ValueError("positions: one for each of the axes expected")
    p = positions.dtype
    if p is torch.int32 or p is torch.float32:
        return positions
    if p is torch.bool or p.is_complex:
        raise ValueError("positions: integers or floats expected")
    return positions.to(torch.float32 if p.is_floating_point else torch.int32)


def _unit_rows(x):
    """x itself when its last dimension is dense, else a copy."""
    return x if x.stride(-1) == 1 else x.contiguous()


def _strides(x, heads_first=False):
    """(batch, token, head) element strides of rows [(batch,) tokens, heads, dim] (heads_first: heads, tokens)."""
    s = x.stride()
    b = s[0] if len(s) == 4 else 0
    return (b, s[-2], s[-3]) if heads_first else (b, s[-3], s[-2])


def _out_shape(shape, heads_first):
    return (*shape[:-3], shape[-2], shape[-3], shape[-1]) if heads_first else shape


_NO_TENSOR = (0,) * 16


def _pack(spec, x, positions, fields, count, ws=0, ws_bytes=0):
    shape = x.shape
    ps = positions.stride()
    batched = len(ps) == 3 and positions.shape[0] > 1
    return _lib.ROTARY_ARGS.pack(
        *fields, *(_NO_TENSOR if count == 1 else ()), count, _DTYPES[x.dtype], shape[0] if len(shape) == 4 else 1,
        shape[-3], shape[-1], positions.shape[-1], *spec.axes, spec.pairs, positions.data_ptr(),
        _lib.LAYER_F32 if positions.dtype is torch.float32 else _lib.LAYER_I32, ps[0] if batched else 0, ps[-2], ps[-1],
        spec.theta, spec.freqs, spec.eps, ws, ws_bytes)


def _empty(x, heads_first):
    """A contiguous output for rows x in either order."""
    return torch.empty_like(x.transpose(-3, -2) if heads_first else x, memory_format=torch.contiguous_format)


def _on(device):
    """A context with the tensors' device current (None where it is)."""
    return None if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _forward(spec, tensors, weights, positions):
    positions = _check(spec, tensors, weights, positions)
    x0 = tensors[0]
    dev, hf = x0.device, spec.heads_first
    guard = _on(dev)
    if guard is not None:
        with guard:
            return _forward(spec, tensors, weights, positions)
    outs, fields, keep = [], [], []
    for x, w in zip(tensors, weights):
        if x.stride(-1) != 1:
            x = x.contiguous()
        y = _empty(x, hf)
        wp = wd = 0
        if w is not None:
            w = w.contiguous()
            wp, wd = w.data_ptr(), _DTYPES[w.dtype]
        fields += (x.data_ptr(), *_strides(x), y.data_ptr(), *_strides(y, hf), 0, 0, 0, 0, wp, 0, wd, x.shape[-2])
        keep += (x, w)
        outs.append(y)
    rc = lib().htrc_rotary_forward(_pack(spec, x0, positions, fields, len(outs)), _lib.raw_stream(dev.index))
    if rc:
        check(rc, "htrc_rotary_forward")
    return outs


def _backward(spec, grads, tensors, weights, positions):
    positions = _check(spec, tensors, weights, positions)
    x0 = tensors[0]
    dtype, dev, hf = x0.dtype, x0.device, spec.heads_first
    for g, x in zip(grads, tensors):
        shape = _out_shape(x.shape, hf)
        if not isinstance(g, torch.Tensor) or g.shape != shape or g.dtype != dtype or g.device != dev:
            raise ValueError(f"the output's gradient: {list(shape)} {dtype} expected")
    guard = _on(dev)
    if guard is not None:
        with guard:
            return _backward(spec, grads, tensors, weights, positions)
    outs, dws, fields, keep = [], [], [], []
    for g, x, w in zip(grads, tensors, weights):
        g, x = _unit_rows(g), _unit_rows(x)
        dx = _empty(x, False)
        dw = None
        norm = (0, 0, 0, 0, 0, 0, 0)
        if w is not None:
            w = w.contiguous()
            dw = torch.empty_like(w)
            norm = (x.data_ptr(), *_strides(x), w.data_ptr(), dw.data_ptr(), _DTYPES[w.dtype])
        fields += (g.data_ptr(), *_strides(g, hf), dx.data_ptr(), *_strides(dx), *norm, x.shape[-2])
        keep += (g, x, w)
        outs.append(dx)
        dws.append(dw)
    ws, wp, need = None, 0, 0
    if any(w is not None for w in weights):
        size = ctypes.c_size_t()
        check(lib().htrc_rotary_workspace_size(_pack(spec, x0, positions, fields, len(outs)), size),
              "htrc_rotary_workspace_size")
        need = size.value
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        wp = ws.data_ptr()
    rc = lib().htrc_rotary_backward(_pack(spec, x0, positions, fields, len(outs), wp, need), _lib.raw_stream(dev.index))
    if rc:
        check(rc, "htrc_rotary_backward")
    return outs, dws


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, spec, positions, count, *args):
        tensors, weights = args[:count], args[count:]
        ctx.spec, ctx.count = spec, count
        ctx.save_for_backward(positions, *args)
        return tuple(_forward(spec, tensors, weights, positions))

    @staticmethod
    def backward(ctx, *grads):
        positions, *args = ctx.saved_tensors
        dx, dw = _backward(ctx.spec, grads, args[:ctx.count], args[ctx.count:], positions)
        return (None, None, None, *first_order("rotary_axes", (*dx, *dw), (*args, *grads)))


def _apply(spec, tensors, weights, positions):
    if recorded(*tensors, *weights):
        return _Rotary.apply(spec, positions, len(tensors), *tensors, *weights)
    return tuple(_forward(spec, tensors, weights, positions))


def rotary_axes(x, positions, *, axes, theta=10000.0, pairs="interleaved", weight=None, eps=1e-6, freqs=None,
                heads_first=False):
    """x [(batch,) tokens, heads, dim] normalised (with ``weight`` [dim]) and rotated, in x's type and order
    (heads_first: [(batch,) heads, tokens, dim], contiguous).

    positions [(batch,) tokens, len(axes)], integers (any int32 value, its angles exactly reduced) or floats (taken as
    float32); freqs:
    the ``sum(axes) / 2`` frequencies in radians per position instead of ``theta``'s."""
    return _apply(_spec(axes, theta, pairs, eps, freqs, heads_first), (x,), (weight,), positions)[0]


def rotary_axes_backward(dy, x, positions, *, axes, theta=10000.0, pairs="interleaved", weight=None, eps=1e-6,
                         freqs=None, heads_first=False):
    """(dx, dweight) of ``rotary_axes`` for the output's gradient dy (dweight None without a weight)."""
    dx, dw = _backward(_spec(axes, theta, pairs, eps, freqs, heads_first), (dy,), (x,), (weight,), positions)
    return dx[0], dw[0]


def rotary_qk(q, k, positions, *, axes, theta=10000.0, pairs="interleaved", q_weight=None, k_weight=None, eps=1e-6,
              freqs=None, heads_first=False):
    """``rotary_axes`` of q [(batch,) tokens, heads, dim] and k [(batch,) tokens, kv_heads, dim] in one launch."""
    return _apply(_spec(axes, theta, pairs, eps, freqs, heads_first), (q, k), (q_weight, k_weight), positions)


def rotary_qk_backward(dq, dk, q, k, positions, *, axes, theta=10000.0, pairs="interleaved", q_weight=None,
                       k_weight=None, eps=1e-6, freqs=None, heads_first=False):
    """(dq, dk, dq_weight, dk_weight) of ``rotary_qk`` for its outputs' gradients."""
    dx, dw = _backward(_spec(axes, theta, pairs, eps, freqs, heads_first), (dq, dk), (q, k), (q_weight, k_weight),
                       positions)
    return (*dx, *dw)
