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
The functions take part in autograd; the backward can also be called by itself.  There is no CPU path.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from ._lib import check, lib, ptr, stream_ptr

_DTYPES = {torch.bfloat16: _lib.LAYER_BF16, torch.float16: _lib.LAYER_F16}
_MASKS = {torch.bool: _lib.LAYER_U8, torch.float32: _lib.LAYER_F32, torch.bfloat16: _lib.LAYER_BF16,
          torch.float16: _lib.LAYER_F16}
_status = {}


def _status_word(device):
    """The device word that the kernels' guards write (one per device, zeroed when it is made)."""
    w = _status.get(device)
    if w is None:
        w = _status[device] = torch.zeros(64, dtype=torch.int32, device=device)
    return w


def cross_status(device=None):
    """Raise if a cross-attention kernel on the device reported a failed guard since the last check (synchronises)."""
    from .flat import device_status
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    with torch.cuda.device(dev):
        return device_status(_status_word(dev))


def _rows(x):
    """x where its rows are dense, 16-byte aligned and its own, else a contiguous copy."""
    s = x.stride()
    fine = (s[-1] == 1 or x.shape[-1] == 1) and x.data_ptr() % 16 == 0 and all(
        n == 1 or (t % 8 == 0 and (t > 0 or i == 0)) for i, (n, t) in enumerate(zip(x.shape[:-1], s[:-1])))
    return x if fine else x.contiguous()


def _strides(x, heads_first):
    """(batch, token, head) strides of a 4-d tensor."""
    s = x.stride()
    return (s[0], s[2], s[1]) if heads_first else (s[0], s[1], s[2])


class _Call:
    """The checked arguments of one call: 4-d operands, shapes and the mask."""
    __slots__ = ("q", "k", "v", "heads_first", "scale", "lengths", "mask", "batch", "queries", "keys", "heads",
                 "kv_heads", "dim", "squeeze")

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
        self.heads_first = bool(heads_first)
        t, h = (2, 1) if heads_first else (1, 2)
        self.batch, self.queries, self.heads, self.dim = (int(q.shape[i]) for i in (0, t, h, 3))
        self.keys, self.kv_heads = int(k.shape[t]), int(k.shape[h])
        if k.shape != v.shape or int(k.shape[0]) != self.batch or int(k.shape[3]) != self.dim:
            raise ValueError("k and v: q's batch and dim, and one shape, expected")
        if self.kv_heads < 1 or self.heads < 1 or self.heads % self.kv_heads:
            raise ValueError(f"{self.heads} query heads do not share {self.kv_heads} key heads evenly")
        if self.dim % 8 or not 8 <= self.dim <= _lib.CROSS_MAX_DIM:
            raise NotImplementedError(f"dim: a multiple of 8 up to {_lib.CROSS_MAX_DIM} is supported, got {self.dim}")
        self.scale = 1.0 / math.sqrt(self.dim) if scale is None else float(scale)
        if not (self.scale > 0 and math.isfinite(self.scale)):
            raise ValueError("scale must be positive and finite")
        if key_lengths is not None:
            if not isinstance(key_lengths, torch.Tensor) or key_lengths.shape != (self.batch,) or \
                    key_lengths.is_floating_point() or key_lengths.device != q.device:
                raise ValueError("key_lengths: [batch] integers on q's device expected")
            key_lengths = key_lengths.to(torch.int32).contiguous()
        self.lengths = key_lengths
        if mask is not None:
            if not isinstance(mask, torch.Tensor) or mask.dtype not in _MASKS or mask.device != q.device:
                raise ValueError("mask: a bool, float32, bfloat16 or float16 tensor on q's device expected")
            try:
                mask = mask.expand(self.batch, self.heads, self.queries, self.keys)
            except RuntimeError as e:
                raise ValueError(f"mask {list(mask.shape)} does not broadcast to "
                                 f"{[self.batch, self.heads, self.queries, self.keys]}") from e
        self.mask = mask
        self.q, self.k, self.v = _rows(q), _rows(k), _rows(v)

    def args(self):
        a = _lib.HtrcCrossArgs()
        hf = self.heads_first
        a.q, a.k, a.v = ptr(self.q), ptr(self.k), ptr(self.v)
        a.q_stride[:], a.k_stride[:], a.v_stride[:] = (_strides(x, hf) for x in (self.q, self.k, self.v))
        a.batch, a.queries, a.keys = self.batch, self.queries, self.keys
        a.heads, a.kv_heads, a.dim, a.dtype = self.heads, self.kv_heads, self.dim, _DTYPES[self.q.dtype]
        a.scale = self.scale
        a.key_lengths = ptr(self.lengths)
        if self.mask is not None:
            a.mask, a.mask_dtype = ptr(self.mask), _MASKS[self.mask.dtype]
            a.mask_stride[:] = self.mask.stride()
        a.status = ptr(_status_word(self.q.device))
        return a


def _forward(c):
    q = c.q
    with torch.cuda.device(q.device):
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        lse = torch.empty((c.batch, c.heads, c.queries), dtype=torch.float32, device=q.device)
        a = c.args()
        a.out, a.out_stride[:], a.lse = ptr(out), _strides(out, c.heads_first), ptr(lse)
        check(lib().htrc_cross_forward(a, stream_ptr()), "htrc_cross_forward")
    return out, lse


def _backward(c, dout, out, lse, dlse):
    hf, q = c.heads_first, c.q
    if c.squeeze:
        dout, out, lse = dout[None], out[None], lse.reshape(1, *lse.shape[-2:])
        dlse = None if dlse is None else dlse.reshape(1, *dlse.shape[-2:])
    for name, x in (("dout", dout), ("out", out)):
        if x.shape != q.shape or x.dtype != q.dtype or x.device != q.device:
            raise ValueError(f"{name}: q's shape, type and device expected")
    for name, x in (("lse", lse), ("dlse", dlse)):
        if x is not None and (x.shape != (c.batch, c.heads, c.queries) or x.dtype != torch.float32 or
                              x.device != q.device):
            raise ValueError(f"{name}: [batch, heads, queries] float32 on q's device expected")
    with torch.cuda.device(q.device):
        dout, out = _rows(dout), _rows(out)
        lse = lse.contiguous()
        dlse = None if dlse is None else dlse.contiguous()
        dq, dk, dv = (torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, c.k, c.v))
        a = c.args()
        a.out, a.out_stride[:], a.lse = ptr(out), _strides(out, hf), ptr(lse)
        a.dout, a.dout_stride[:], a.dlse = ptr(dout), _strides(dout, hf), ptr(dlse)
        a.dq, a.dk, a.dv = ptr(dq), ptr(dk), ptr(dv)
        a.dq_stride[:], a.dk_stride[:], a.dv_stride[:] = (_strides(x, hf) for x in (dq, dk, dv))
        need = ctypes.c_size_t()
        check(lib().htrc_cross_workspace_size(a, need), "htrc_cross_workspace_size")
        ws = torch.empty(max(need.value, 256), dtype=torch.uint8, device=q.device)
        a.workspace, a.workspace_bytes = ptr(ws), int(ws.numel())
        check(lib().htrc_cross_backward(a, stream_ptr()), "htrc_cross_backward")
    return (dq[0], dk[0], dv[0]) if c.squeeze else (dq, dk, dv)


class _Cross(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, key_lengths, mask, scale, heads_first):
        c = _Call(q, k, v, key_lengths, mask, scale, heads_first)
        out, lse = _forward(c)
        if c.squeeze:
            out, lse = out[0], lse[0]
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
        return (*grads, None, None, None, None)


def cross_attention(q, k, v, *, key_lengths=None, mask=None, scale=None, heads_first=False, return_lse=False):
    """q [batch, queries, heads, dim], k / v [batch, keys, kv_heads, dim] (heads_first: heads before tokens; batch may
    be left out) -> out in q's shape, type and order, and with return_lse the float32 log-sum-exp of the logits
    [batch, heads, queries].  scale: of the logits, 1 / sqrt(dim) by default; a mask gets no gradient."""
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out, lse = _Cross.apply(q, k, v, key_lengths, mask, scale, heads_first)
    else:
        c = _Call(q, k, v, key_lengths, mask, scale, heads_first)
        out, lse = _forward(c)
        if c.squeeze:
            out, lse = out[0], lse[0]
    return (out, lse) if return_lse else out


def cross_attention_backward(dout, q, k, v, out, lse, *, dlse=None, key_lengths=None, mask=None, scale=None,
                             heads_first=False):
    """(dq, dk, dv) of ``cross_attention`` from its inputs, its outputs and their gradients (dlse: None or the
    gradient of lse).  The gradients of shared key heads are summed over their query heads."""
    return _backward(_Call(q, k, v, key_lengths, mask, scale, heads_first), dout, out, lse, dlse)
