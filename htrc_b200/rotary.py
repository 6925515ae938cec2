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
place); arithmetic is float32, rounded once to the input's type.  The functions take part in autograd; the backward
passes can also be called by themselves.  There is no CPU path.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from ._lib import check, lib, ptr, stream_ptr

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


def _unit_rows(x):
    """x itself when its last dimension is dense, else a copy."""
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


class _Spec:
    """The arguments that every call shares, checked."""
    __slots__ = ("axes", "theta", "pairs", "eps", "freqs", "heads_first")

    def __init__(self, axes, theta, pairs, eps, freqs, heads_first):
        axes = tuple(int(w) for w in axes)
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
        if freqs is not None:
            freqs = tuple(float(f) for f in freqs)
            if len(freqs) != sum(axes) // 2 or not all(math.isfinite(f) for f in freqs):
                raise ValueError("freqs: one finite frequency for each of the sum(axes) / 2 pairs")
        self.axes, self.theta, self.pairs, self.eps = axes, float(theta), pairs, float(eps)
        self.freqs, self.heads_first = freqs, bool(heads_first)


def _check_rows(x, name, like=None):
    if not isinstance(x, torch.Tensor) or x.dim() not in (3, 4):
        raise ValueError(f"{name}: [tokens, heads, dim] or [batch, tokens, heads, dim] expected")
    if x.dtype not in _DTYPES:
        raise ValueError(f"{name}: float32, bfloat16 or float16 expected, got {x.dtype}")
    if not x.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (there is no CPU path)")
    if like is not None and (x.dtype != like.dtype or x.device != like.device or x.dim() != like.dim() or
                             x.shape[:-2] != like.shape[:-2] or x.shape[-1] != like.shape[-1]):
        raise ValueError(f"{name}: the other tensor's type, device, batch, tokens and dim expected")


def _check(spec, tensors, weights, positions):
    x = tensors[0]
    _check_rows(x, "x")
    for t in tensors[1:]:
        _check_rows(t, "k", x)
    dim = int(x.shape[-1])
    if dim > _lib.ROTARY_MAX_DIM or dim < 2:
        raise NotImplementedError(f"heads of 2 to {_lib.ROTARY_MAX_DIM} elements are supported, got {dim}")
    if sum(spec.axes) > dim:
        raise ValueError(f"axes rotate {sum(spec.axes)} of {dim} elements")
    for t in tensors:
        if not 1 <= int(t.shape[-2]) <= _lib.ROTARY_MAX_HEADS:
            raise NotImplementedError(f"1 to {_lib.ROTARY_MAX_HEADS} heads are supported")
    for w in weights:
        if w is not None and (w.shape != (dim,) or w.dtype not in _DTYPES or w.device != x.device):
            raise ValueError(f"weight: [{dim}] float32, bfloat16 or float16 on the rows' device expected")
    lead = x.shape[:-2]
    if not isinstance(positions, torch.Tensor) or positions.device != x.device or \
            positions.dim() not in (2, x.dim() - 1) or positions.shape[-1] != len(spec.axes) or \
            positions.shape[-2] != lead[-1] or (positions.dim() == 3 and positions.shape[0] not in (1, lead[0])):
        raise ValueError("positions: [tokens, axes] or [batch, tokens, axes] on the rows' device expected")
    if positions.is_floating_point():
        return positions if positions.dtype == torch.float32 else positions.float()
    if positions.dtype == torch.bool or positions.is_complex():
        raise ValueError("positions: integers or floats expected")
    return positions if positions.dtype == torch.int32 else positions.to(torch.int32)


def _strides(x, heads_first=False):
    """(batch, token, head) element strides of rows [(batch,) tokens, heads, dim] (heads_first: heads, tokens)."""
    s = x.stride()
    b = s[0] if x.dim() == 4 else 0
    return (b, s[-2], s[-3]) if heads_first else (b, s[-3], s[-2])


def _args(spec, like, positions):
    a = _lib.HtrcRotaryArgs()
    a.dtype = _DTYPES[like.dtype]
    a.batch = int(like.shape[0]) if like.dim() == 4 else 1
    a.tokens, a.dim = int(like.shape[-3]), int(like.shape[-1])
    a.n_axes = len(spec.axes)
    for i, w in enumerate(spec.axes):
        a.axis_width[i] = w
    a.pairs = _lib.ROTARY_PAIRS[spec.pairs]
    a.positions = ptr(positions)
    a.position_dtype = _lib.LAYER_F32 if positions.dtype == torch.float32 else _lib.LAYER_I32
    batched = positions.dim() == 3 and positions.shape[0] > 1
    a.position_stride[:] = (positions.stride(0) if batched else 0, positions.stride(-2), positions.stride(-1))
    a.theta, a.eps = spec.theta, spec.eps
    if spec.freqs is not None:
        a._freqs = (ctypes.c_double * len(spec.freqs))(*spec.freqs)
        a.freqs = ctypes.cast(a._freqs, ctypes.POINTER(ctypes.c_double))
    return a


def _out_shape(x, heads_first):
    return (*x.shape[:-3], x.shape[-2], x.shape[-3], x.shape[-1]) if heads_first else x.shape


def _forward(spec, tensors, weights, positions):
    positions = _check(spec, tensors, weights, positions)
    a = _args(spec, tensors[0], positions)
    a.n_tensors = len(tensors)
    outs = []
    keep = []
    with torch.cuda.device(tensors[0].device):
        for i, (x, w) in enumerate(zip(tensors, weights)):
            x = _unit_rows(x)
            w = None if w is None else w.contiguous()
            y = torch.empty(_out_shape(x, spec.heads_first), dtype=x.dtype, device=x.device)
            t = a.tensor[i]
            t.in_, t.in_stride[:], t.out, t.out_stride[:] = ptr(x), _strides(x), ptr(y), _strides(y, spec.heads_first)
            t.heads = int(x.shape[-2])
            if w is not None:
                t.weight, t.weight_dtype = ptr(w), _DTYPES[w.dtype]
            keep += [x, w]
            outs.append(y)
        check(lib().htrc_rotary_forward(a, stream_ptr()), "htrc_rotary_forward")
    return outs


def _backward(spec, grads, tensors, weights, positions):
    positions = _check(spec, tensors, weights, positions)
    a = _args(spec, tensors[0], positions)
    a.n_tensors = len(tensors)
    outs, dws, keep = [], [], []
    dev = tensors[0].device
    with torch.cuda.device(dev):
        for i, (g, x, w) in enumerate(zip(grads, tensors, weights)):
            if not isinstance(g, torch.Tensor) or g.shape != _out_shape(x, spec.heads_first) or g.dtype != x.dtype or \
                    g.device != dev:
                raise ValueError(f"the output's gradient: {list(_out_shape(x, spec.heads_first))} {x.dtype} expected")
            g, x = _unit_rows(g), _unit_rows(x)
            w = None if w is None else w.contiguous()
            dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
            dw = None if w is None else torch.empty_like(w)
            t = a.tensor[i]
            t.in_, t.in_stride[:], t.out, t.out_stride[:] = ptr(g), _strides(g, spec.heads_first), ptr(dx), _strides(dx)
            t.heads = int(x.shape[-2])
            if w is not None:
                t.x, t.x_stride[:] = ptr(x), _strides(x)
                t.weight, t.weight_dtype, t.dweight = ptr(w), _DTYPES[w.dtype], ptr(dw)
            keep += [g, x, w]
            outs.append(dx)
            dws.append(dw)
        ws = None
        if any(w is not None for w in weights):
            need = ctypes.c_size_t()
            check(lib().htrc_rotary_workspace_size(a, need), "htrc_rotary_workspace_size")
            ws = torch.empty(need.value, dtype=torch.uint8, device=dev)
            a.workspace, a.workspace_bytes = ptr(ws), need.value
        check(lib().htrc_rotary_backward(a, stream_ptr()), "htrc_rotary_backward")
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
        return (None, None, None, *dx, *dw)


def _apply(spec, tensors, weights, positions):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (*tensors, *weights)):
        return _Rotary.apply(spec, positions, len(tensors), *tensors, *weights)
    return tuple(_forward(spec, tensors, weights, positions))


def rotary_axes(x, positions, *, axes, theta=10000.0, pairs="interleaved", weight=None, eps=1e-6, freqs=None,
                heads_first=False):
    """x [(batch,) tokens, heads, dim] normalised (with ``weight`` [dim]) and rotated, in x's type and order
    (heads_first: [(batch,) heads, tokens, dim], contiguous).

    positions [(batch,) tokens, len(axes)], integers (any int32 value, its angles exactly reduced) or floats; freqs:
    the ``sum(axes) / 2`` frequencies in radians per position instead of ``theta``'s."""
    return _apply(_Spec(axes, theta, pairs, eps, freqs, heads_first), (x,), (weight,), positions)[0]


def rotary_axes_backward(dy, x, positions, *, axes, theta=10000.0, pairs="interleaved", weight=None, eps=1e-6,
                         freqs=None, heads_first=False):
    """(dx, dweight) of ``rotary_axes`` for the output's gradient dy (dweight None without a weight)."""
    dx, dw = _backward(_Spec(axes, theta, pairs, eps, freqs, heads_first), (dy,), (x,), (weight,), positions)
    return dx[0], dw[0]


def rotary_qk(q, k, positions, *, axes, theta=10000.0, pairs="interleaved", q_weight=None, k_weight=None, eps=1e-6,
              freqs=None, heads_first=False):
    """``rotary_axes`` of q [(batch,) tokens, heads, dim] and k [(batch,) tokens, kv_heads, dim] in one launch."""
    return _apply(_Spec(axes, theta, pairs, eps, freqs, heads_first), (q, k), (q_weight, k_weight), positions)


def rotary_qk_backward(dq, dk, q, k, positions, *, axes, theta=10000.0, pairs="interleaved", q_weight=None,
                       k_weight=None, eps=1e-6, freqs=None, heads_first=False):
    """(dq, dk, dq_weight, dk_weight) of ``rotary_qk`` for its outputs' gradients."""
    dx, dw = _backward(_Spec(axes, theta, pairs, eps, freqs, heads_first), (dq, dk), (q, k), (q_weight, k_weight),
                       positions)
    return (*dx, *dw)
