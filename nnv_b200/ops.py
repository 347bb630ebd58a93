"""Operators of transformer networks on CUDA tensors: layer normalisation and attention over an encoder's states,
with their gradients.

``NN.evaluate`` runs the same kernels in double for the layers ``nn.LayerNormalizationLayer`` and
``nn.AttentionLayer``; this module is for hosts that keep their tensors on the GPU (torch).  Every function
checks its arguments (``ValueError`` / ``TypeError`` before anything is launched), allocates its outputs,
enqueues its kernels on torch's current stream of the tensors' device and returns without waiting.  Gradients are
explicit calls: the forward functions do not record for autograd.

Element types: float64, float32, bfloat16, float16, one type per call.  Statistics (mean, rstd, log-sum-exp) are
float32, or float64 with float64 tensors; sums are held in that type and a result is rounded once when stored.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib as L

__all__ = ["layer_norm", "layer_norm_backward", "cross_attention", "cross_attention_backward"]

_DTYPES = {torch.float64: L.F64, torch.float32: L.F32, torch.bfloat16: L.BF16, torch.float16: L.F16}


def _tensor(name, t, like=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch tensor" % name)
    if t.dtype not in _DTYPES:
        raise TypeError("%s has element type %s (float64, float32, bfloat16 or float16 expected)" % (name, t.dtype))
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise ValueError("%s (%s on %s) does not match the input (%s on %s)"
                         % (name, t.dtype, t.device, like.dtype, like.device))
    if t.device.type != "cuda":
        raise ValueError("%s is on %s; these operators have no CPU path" % (name, t.device))
    return t


def _stat_type(t):
    return torch.float64 if t.dtype is torch.float64 else torch.float32


def _stat(name, t, shape, like):
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch tensor" % name)
    if t.dtype != _stat_type(like) or t.device != like.device or tuple(t.shape) != tuple(shape):
        raise ValueError("%s must be a %s tensor of shape %s on %s" % (name, _stat_type(like), tuple(shape), like.device))
    return t.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


class _on:
    """The tensors' device made current for a call (the library works on the current device)."""

    __slots__ = ("want", "prev")

    def __init__(self, device):
        self.want = device.index

    def __enter__(self):
        self.prev = torch.cuda.current_device()
        if self.prev != self.want:
            torch.cuda.set_device(self.want)
        return torch.cuda.current_stream(self.want).cuda_stream

    def __exit__(self, *exc):
        if self.prev != self.want:
            torch.cuda.set_device(self.prev)


def _rows(t, cols):
    """(tensor, rows, elements from row to row) of t[..., cols] seen as rows; copies what has no single row stride."""
    rows = t.numel() // cols
    if t.is_contiguous():
        return t, rows, cols
    if t.dim() == 2 and t.stride(1) == 1 and (rows <= 1 or t.stride(0) >= cols):
        return t, rows, (t.stride(0) if rows > 1 else cols)
    return t.contiguous(), rows, cols


def _ln_input(x):
    _tensor("x", x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must have at least one dimension, the normalised one, and at least one column")
    return x.shape[-1]


def _weight(name, w, cols, x):
    if w is None:
        return None
    _tensor(name, w, x)
    if w.dim() != 1 or w.shape[0] != cols:
        raise ValueError("%s must have one entry per column (%d), got shape %s" % (name, cols, tuple(w.shape)))
    return w.contiguous()


def layer_norm(x, scale=None, offset=None, eps=1e-5, return_stats=False):
    """(x - mean) / sqrt(var + eps) * scale + offset over the last dimension of ``x``.

    ``scale`` and ``offset`` (one entry per column) may be None.  With ``return_stats`` the rows' mean and
    1/sqrt(var + eps) come back too, shaped like ``x`` without its last dimension: what the backward call takes."""
    cols = _ln_input(x)
    scale, offset = _weight("scale", scale, cols, x), _weight("offset", offset, cols, x)
    eps = float(eps)
    if not (eps >= 0 and math.isfinite(eps)):
        raise ValueError("eps must be finite and not negative")
    xr, rows, ldx = _rows(x, cols)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    mean = rstd = None
    if return_stats:
        mean = torch.empty(x.shape[:-1], dtype=_stat_type(x), device=x.device)
        rstd = torch.empty_like(mean)
    with _on(x.device) as stream:
        L.check(L.load().nnvb_layer_norm_forward(stream, _DTYPES[x.dtype], rows, cols, xr.data_ptr(), ldx, _ptr(scale),
                                                 _ptr(offset), eps, y.data_ptr(), cols, _ptr(mean), _ptr(rstd)),
                "nnvb_layer_norm_forward")
    return (y, mean, rstd) if return_stats else y


def layer_norm_backward(dy, x, scale, mean, rstd):
    """Gradients (dx, dscale, doffset) of ``layer_norm``: ``dy`` the gradient of its output, ``mean`` and ``rstd``
    its statistics.  The weights' gradients are sums over all rows, in a fixed order; with ``scale`` None they
    are those of a scale of ones."""
    cols = _ln_input(x)
    _tensor("dy", dy, x)
    if dy.shape != x.shape:
        raise ValueError("dy has shape %s, x %s" % (tuple(dy.shape), tuple(x.shape)))
    scale = _weight("scale", scale, cols, x)
    mean, rstd = _stat("mean", mean, x.shape[:-1], x), _stat("rstd", rstd, x.shape[:-1], x)
    xr, rows, ldx = _rows(x, cols)
    gr, _, ldg = _rows(dy, cols)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dscale = torch.empty(cols, dtype=x.dtype, device=x.device)
    doffset = torch.empty_like(dscale)
    lib = L.load()
    dt = _DTYPES[x.dtype]
    nbytes = lib.nnvb_layer_norm_workspace(dt, rows, cols)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    with _on(x.device) as stream:
        L.check(lib.nnvb_layer_norm_backward(stream, dt, rows, cols, gr.data_ptr(), ldg, xr.data_ptr(), ldx, _ptr(scale),
                                             mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), cols, dscale.data_ptr(),
                                             doffset.data_ptr(), ws.data_ptr(), nbytes),
                "nnvb_layer_norm_backward")
    return dx, dscale, doffset


def _heads(name, t, like=None):
    _tensor(name, t, like)
    if t.dim() != 4:
        raise ValueError("%s must be [batch, tokens, heads, head size], got shape %s" % (name, tuple(t.shape)))
    # the kernels take any strides but need a head's elements side by side
    return t if t.shape[3] <= 1 or t.stride(3) == 1 else t.contiguous()


def _attn(q, k, v, lengths, scale):
    q = _heads("q", q)
    k, v = _heads("k", k, q), _heads("v", v, q)
    B, Lq, Hq, D = q.shape
    if k.shape != v.shape:
        raise ValueError("k and v differ in shape: %s, %s" % (tuple(k.shape), tuple(v.shape)))
    Lk, Hkv = k.shape[1], k.shape[2]
    if k.shape[0] != B or k.shape[3] != D:
        raise ValueError("q %s and k %s differ in batch or head size" % (tuple(q.shape), tuple(k.shape)))
    if Hq < 1 or Hkv < 1 or Hq % Hkv:
        raise ValueError("%d query heads cannot share %d state heads evenly" % (Hq, Hkv))
    if not 1 <= D <= 256:
        raise ValueError("head size %d is outside 1..256" % D)
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    scale = float(scale)
    if not (math.isfinite(scale) and scale > 0):
        raise ValueError("scale must be finite and positive")
    if lengths is not None:
        if not isinstance(lengths, torch.Tensor) or lengths.dtype != torch.int32 or lengths.device != q.device \
                or tuple(lengths.shape) != (B,):
            raise ValueError("lengths must be an int32 tensor with one entry per batch entry on %s" % q.device)
        lengths = lengths.contiguous()
    d = L.AttentionDesc(_DTYPES[q.dtype], 0, B, Lq, Lk, Hq, Hkv, D, scale, q.stride()[:3], k.stride()[:3], v.stride()[:3])
    return q, k, v, lengths, d


def cross_attention(q, k, v, lengths=None, scale=None, return_lse=False):
    """softmax(scale * q k^T) v of the positions q [B, Lq, Hq, D] over an encoder's states k, v [B, Lk, Hkv, D].

    Hq is a multiple of Hkv: query head h reads state head h // (Hq / Hkv).  ``lengths`` (int32 [B], on the device)
    gives the valid states of each batch entry, clipped to 0..Lk; what the others hold has no effect.  Rows
    without a valid state are zero.  ``scale`` defaults to 1/sqrt(D).  Tensors may be strided views.  With
    ``return_lse`` the log-sum-exp [B, Hq, Lq] of each row's scores comes back too (-inf without states)."""
    q, k, v, lengths, d = _attn(q, k, v, lengths, scale)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    d.out_stride = out.stride()[:3]
    lse = torch.empty((q.shape[0], q.shape[2], q.shape[1]), dtype=_stat_type(q), device=q.device) if return_lse else None
    with _on(q.device) as stream:
        L.check(L.load().nnvb_cross_attention_forward(stream, C.byref(d), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                                      _ptr(lengths), out.data_ptr(), _ptr(lse)),
                "nnvb_cross_attention_forward")
    return (out, lse) if return_lse else out


def cross_attention_backward(dout, q, k, v, out, lse, lengths=None, scale=None):
    """Gradients (dq, dk, dv) of ``cross_attention``: ``dout`` the gradient of its output, ``out`` and ``lse`` what it
    returned (``return_lse=True``).  dk and dv are summed, in a fixed order, over the query heads that share a state
    head, and are zero for states behind ``lengths``."""
    q, k, v, lengths, d = _attn(q, k, v, lengths, scale)
    dout, out = _heads("dout", dout, q), _heads("out", out, q)
    if dout.shape != q.shape or out.shape != q.shape:
        raise ValueError("dout %s and out %s must be shaped like q %s" % (tuple(dout.shape), tuple(out.shape), tuple(q.shape)))
    lse = _stat("lse", lse, (q.shape[0], q.shape[2], q.shape[1]), q)
    d.out_stride, d.dout_stride = out.stride()[:3], dout.stride()[:3]
    dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dk = torch.empty(k.shape, dtype=q.dtype, device=q.device)
    dv = torch.empty(k.shape, dtype=q.dtype, device=q.device)
    lib = L.load()
    nbytes = lib.nnvb_cross_attention_workspace(C.byref(d))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    with _on(q.device) as stream:
        L.check(lib.nnvb_cross_attention_backward(stream, C.byref(d), dout.data_ptr(), q.data_ptr(), k.data_ptr(),
                                                  v.data_ptr(), out.data_ptr(), lse.data_ptr(), _ptr(lengths),
                                                  dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), nbytes),
                "nnvb_cross_attention_backward")
    return dq, dk, dv
