"""Cross attention of a video transformer's tokens to an encoder's states of another length (a prompt, a reference
clip), forward and backward, on tcgen05 kernels (``csrc/cross_fwd.cu``, ``csrc/cross_bwd.cu``).

    out = cross_attention(q, k, v, key_lengths=lengths)            # [batch, tokens, heads, dim]
    out = cross_attention(q, k, v, mask=mask, heads_first=True)    # [batch, heads, tokens, dim]

Query head ``h`` reads key head ``h // (heads // kv_heads)``.  ``key_lengths`` [batch] ends each entry's keys; ``mask``
broadcasts to [batch, heads, queries, keys]: bool (False excludes) or float (added to the logits, -inf excludes).  A
query with no key left gives 0, its log-sum-exp -inf.  Keys that the lengths or a mask without a query dimension
exclude are never computed with, whatever their rows hold; a mask with one expects finite keys and values.

q, k, v: bfloat16 or float16, dim a multiple of 8 up to 128, any strides that keep rows 16-byte aligned (others are
copied).  Logits, softmax and sums are float32; the softmax weights enter the second product in the operands' type.
The functions take part in autograd (first derivatives, reverse mode); the backward can also be called by itself.  There is
no CPU path.
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import _lib
from ._autograd import first_order, recorded
from ._lib import check, lib

_DTYPES = {torch.bfloat16: _lib.LAYER_BF16, torch.float16: _lib.LAYER_F16}
_MASKS = {torch.bool: _lib.LAYER_U8, torch.float32: _lib.LAYER_F32, torch.bfloat16: _lib.LAYER_BF16,
          torch.float16: _lib.LAYER_F16}
_LENGTHS = (torch.int32, torch.int64, torch.int16, torch.int8, torch.uint8)
_NO_BACK = (0,) * 17
_status = {}


def _status_word(device):
    """The device word that the kernels' guards write (one per device, zeroed before any stream sees it).  None while a
    graph is captured before the first call: its zero fill would become part of the graph."""
    w = _status.get(device)
    if w is None and not torch.cuda.is_current_stream_capturing():
        w = torch.zeros(64, dtype=torch.int32, device=device)
        torch.cuda.current_stream(device).synchronize()
        _status[device] = w
    return w


def cross_status(device=None):
    """Raise if a cross-attention kernel on the device reported a failed guard since the last check (synchronises).  The
    calls of a graph report where the device had a call before the capture."""
    from .flat import device_status
    dev = torch.device("cuda" if device is None else device)
    if dev.index is None:                 # the words are kept by index
        dev = torch.device(dev.type, torch.cuda.current_device())
    with torch.cuda.device(dev):
        return device_status(_status_word(dev))


def _rows(x):
    """x where its rows are dense, 16-byte aligned and their own, else a contiguous copy."""
    s0, s1, s2, s3 = x.stride()
    if s3 == 1 and s1 > 0 and s2 > 0 and not (s0 | s1 | s2) & 7 and not x.data_ptr() & 15:
        return x
    x = x.contiguous()
    if x.data_ptr() & 15:
        x = x.clone()
    # a dense tensor may still hold any stride for a dimension of one
    _, n1, n2, n3 = x.shape
    return x.as_strided(x.shape, (n1 * n2 * n3, n2 * n3, n3, 1))


def _strides(x, heads_first):
    """(batch, token, head) strides of a 4-d tensor."""
    s0, s1, s2, _ = x.stride()
    return (s0, s2, s1) if heads_first else (s0, s1, s2)


def _mask_strides(mask, want):
    """The mask's strides over [batch, heads, queries, keys], 0 where it broadcasts."""
    shape, stride = mask.shape, mask.stride()
    if len(shape) > 4 or any(n != w and n != 1 for n, w in zip(reversed(shape), reversed(want))):
        raise ValueError(f"mask {list(shape)} does not broadcast to {list(want)}")
    strides = tuple(0 if n == 1 else t for n, t in zip(shape, stride))
    return (0,) * (4 - len(strides)) + strides


class _Call:
    """The checked arguments of one call: 4-d operands, shapes and the mask."""
    __slots__ = ("q", "k", "v", "heads_first", "lengths", "mask", "squeeze", "lse_shape", "shape_args", "mask_args",
                 "device")

    def __init__(self, q, k, v, key_lengths, mask, scale, heads_first):
        for name, x in (("q", q), ("k", k), ("v", v)):
            if not isinstance(x, torch.Tensor) or x.dim() not in (3, 4) or x.dim() != q.dim():
                raise ValueError(f"{name}: [batch, tokens, heads, dim] or [tokens, heads, dim] expected "
                                 "(heads_first: [batch, heads, tokens, dim] or [heads, tokens, dim])")
            if x.dtype not in _DTYPES or x.dtype != q.dtype:
                raise NotImplementedError(f"{name}: q, k and v in one of bfloat16 and float16 expected, got {x.dtype}")
            if not x.is_cuda or x.device != q.device:
                raise ValueError("q, k, v must be on one CUDA device (there is no CPU path)")
        self.squeeze = q.dim() == 3
        if self.squeeze:
            q, k, v = q[None], k[None], v[None]
        dev = self.device = q.device
        if heads_first:
            self.heads_first = True
            batch, heads, queries, dim = q.shape
            kb, kv_heads, keys, kd = k.shape
        else:
            self.heads_first = False
            batch, queries, heads, dim = q.shape
            kb, keys, kv_heads, kd = k.shape
        if k.shape != v.shape or kb != batch or kd != dim:
            raise ValueError("k and v: q's batch and dim, and one shape, expected")
        if kv_heads < 1 or heads < 1 or heads % kv_heads:
            raise ValueError(f"{heads} query heads do not share {kv_heads} key heads evenly")
        if dim % 8 or not 8 <= dim <= _lib.CROSS_MAX_DIM:
            raise NotImplementedError(f"dim: a multiple of 8 up to {_lib.CROSS_MAX_DIM} is supported, got {dim}")
        scale = dim ** -0.5 if scale is None else float(scale)
        if not (scale > 0 and math.isfinite(scale)):
            raise ValueError("scale must be positive and finite")
        if key_lengths is not None:
            if not isinstance(key_lengths, torch.Tensor) or key_lengths.dim() != 1 or key_lengths.shape[0] != batch or \
                    key_lengths.dtype not in _LENGTHS or key_lengths.device != dev:
                raise ValueError("key_lengths: [batch] integers on q's device expected")
            if key_lengths.dtype is not torch.int32 or not key_lengths.is_contiguous():
                # more keys than there are is all of them, whatever a wider type held (a narrower one may not hold `keys`)
                key_lengths = key_lengths.long().clamp(0, keys).to(torch.int32).contiguous()
        self.lengths = key_lengths
        self.mask = mask
        self.mask_args = (0, 0, 0, 0, 0, 0)
        if mask is not None:
            if not isinstance(mask, torch.Tensor) or mask.dtype not in _MASKS or mask.device != dev:
                raise ValueError("mask: a bool, float32, bfloat16 or float16 tensor on q's device expected")
            self.mask_args = (mask.data_ptr(), _MASKS[mask.dtype], *_mask_strides(mask, (batch, heads, queries, keys)))
        self.q, self.k, self.v = _rows(q), _rows(k), _rows(v)
        self.lse_shape = (batch, heads, queries)
        self.shape_args = (batch, queries, keys, heads, kv_heads, dim, _DTYPES[q.dtype], scale,
                           0 if key_lengths is None else key_lengths.data_ptr())

    def pack(self, out, lse, back):
        hf, q, k, v = self.heads_first, self.q, self.k, self.v
        status = _status_word(self.device)
        return _lib.CROSS_ARGS.pack(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), *_strides(q, hf), *_strides(k, hf), *_strides(v, hf),
            out.data_ptr(), *_strides(out, hf), 0 if lse is None else lse.data_ptr(), *self.shape_args, *self.mask_args,
            0 if status is None else status.data_ptr(), *back)


@functools.lru_cache(maxsize=256)
def _workspace_bytes(entry, device_index, args):
    """What ``entry`` asks for with these packed arguments, whose pointers are blanked: it goes by shapes alone."""
    need = ctypes.c_size_t()
    check(getattr(lib(), entry)(args, need), entry)
    return need.value


def _workspace(c, entry):
    """A fresh workspace for the call (or None): (tensor, pointer, bytes)."""
    blank = _lib.CROSS_ARGS.pack(*(0,) * 17, *c.shape_args[:-1], 0, c.mask_args[0] and 1, *c.mask_args[1:], 0, *(0,) * 19)
    need = _workspace_bytes(entry, c.device.index, blank)
    if need == 0:
        return None, 0, 0
    ws = torch.empty(need, dtype=torch.uint8, device=c.device)
    return ws, ws.data_ptr(), need


def _on(device):
    """A context with the tensors' device current (None where it is)."""
    return None if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _forward(c, want_lse):
    guard = _on(c.device)
    if guard is not None:
        with guard:
            return _forward(c, want_lse)
    out = torch.empty_like(c.q, memory_format=torch.contiguous_format)
    lse = c.q.new_empty(c.lse_shape, dtype=torch.float32) if want_lse else None
    ws, ptr, need = _workspace(c, "htrc_cross_forward_workspace_size")
    args = c.pack(out, lse, (*_NO_BACK, ptr, need))
    rc = lib().htrc_cross_forward(args, _lib.raw_stream(c.device.index))
    if rc:
        check(rc, "htrc_cross_forward")
    return (out[0], None if lse is None else lse[0]) if c.squeeze else (out, lse)


def _backward(c, dout, out, lse, dlse):
    hf, q = c.heads_first, c.q
    if c.squeeze:
        dout, out, lse = dout[None], out[None], lse[None]
        dlse = None if dlse is None else dlse[None]
    for name, x in (("dout", dout), ("out", out)):
        if x.shape != q.shape or x.dtype != q.dtype or x.device != c.device:
            raise ValueError(f"{name}: q's shape, type and device expected")
    for name, x in (("lse", lse), ("dlse", dlse)):
        if x is not None and (x.shape != c.lse_shape or x.dtype != torch.float32 or x.device != c.device):
            raise ValueError(f"{name}: [batch, heads, queries] float32 on q's device expected")
    guard = _on(c.device)
    if guard is not None:
        with guard:
            return _launch_backward(c, dout, out, lse, dlse)
    return _launch_backward(c, dout, out, lse, dlse)


def _launch_backward(c, dout, out, lse, dlse):
    hf = c.heads_first
    do, o, z = _rows(dout), _rows(out), lse.contiguous()
    dz = None if dlse is None else dlse.contiguous()
    dq, dk, dv = (torch.empty_like(x, memory_format=torch.contiguous_format) for x in (c.q, c.k, c.v))
    ws, ptr, need = _workspace(c, "htrc_cross_backward_workspace_size")
    args = c.pack(o, z, (do.data_ptr(), *_strides(do, hf), 0 if dz is None else dz.data_ptr(), dq.data_ptr(), dk.data_ptr(),
                         dv.data_ptr(), *_strides(dq, hf), *_strides(dk, hf), *_strides(dv, hf), ptr, need))
    rc = lib().htrc_cross_backward(args, _lib.raw_stream(c.device.index))
    if rc:
        check(rc, "htrc_cross_backward")
    return (dq[0], dk[0], dv[0]) if c.squeeze else (dq, dk, dv)


class _Cross(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, key_lengths, mask, scale, heads_first):
        c = _Call(q, k, v, key_lengths, mask, scale, heads_first)
        out, lse = _forward(c, True)
        ctx.save_for_backward(q, k, v, key_lengths, mask, out, lse)
        ctx.more = (scale, heads_first)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    def backward(ctx, dout, dlse):
        q, k, v, key_lengths, mask, out, lse = ctx.saved_tensors
        if dout is None and dlse is None:
            return (None,) * 7
        dout = torch.zeros_like(out) if dout is None else dout
        grads = _backward(_Call(q, k, v, key_lengths, mask, *ctx.more), dout, out, lse, dlse)
        return (*first_order("cross_attention", grads, (q, k, v, dout, dlse)), None, None, None, None)


def cross_attention(q, k, v, *, key_lengths=None, mask=None, scale=None, heads_first=False, return_lse=False):
    """q [batch, queries, heads, dim], k / v [batch, keys, kv_heads, dim] (heads_first: heads before tokens; batch may
    be left out) -> out in q's shape, type and order, and with return_lse the float32 log-sum-exp of the logits
    [batch, heads, queries].  scale: of the logits, 1 / sqrt(dim) by default; a mask gets no gradient."""
    if recorded(q, k, v):
        out, lse = _Cross.apply(q, k, v, key_lengths, mask, scale, heads_first)
    else:
        out, lse = _forward(_Call(q, k, v, key_lengths, mask, scale, heads_first), return_lse)
    return (out, lse) if return_lse else out


def cross_attention_backward(dout, q, k, v, out, lse, *, dlse=None, key_lengths=None, mask=None, scale=None,
                             heads_first=False):
    """(dq, dk, dv) of ``cross_attention`` from its inputs, its outputs and their gradients (dlse: None or the
    gradient of lse).  The gradients of shared key heads are summed over their query heads."""
    return _backward(_Call(q, k, v, key_lengths, mask, scale, heads_first), dout, out, lse, dlse)
