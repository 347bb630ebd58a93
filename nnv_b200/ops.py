"""Operators of transformer networks on CUDA tensors: layer normalisation and attention over an encoder's states,
with their gradients.

``NN.evaluate`` runs the same kernels in double for the layers ``nn.LayerNormalizationLayer`` and
``nn.AttentionLayer``; this module is for hosts that keep their tensors on the GPU (torch).  Every function
checks its arguments (``ValueError`` / ``TypeError`` before anything is launched), allocates its outputs,
enqueues its kernels on torch's current stream of the tensors' device and returns without waiting.  Gradients are
explicit calls: the forward functions do not record for autograd, and refuse tensors that require a gradient while
it records (call them under ``torch.no_grad()``), because that gradient would be lost.

Element types: float64, float32, bfloat16, float16, one type per call.  Statistics (mean, rstd, log-sum-exp) are
float32, or float64 with float64 tensors; sums are held in that type and a result is rounded once when stored.
16-bit attention of more than a few rows also rounds the softmax weights once, before they meet v, or dout in the
gradient dv.  A row whose valid scores are all -inf is NaN; float16 takes scores up to 2^25 in magnitude.
"""
from __future__ import annotations

import math
import struct

import torch

from . import _lib as L

__all__ = ["layer_norm", "layer_norm_backward", "cross_attention", "cross_attention_backward"]

_DTYPES = {torch.float64: L.F64, torch.float32: L.F32, torch.bfloat16: L.BF16, torch.float16: L.F16}
_entries = {}
_DESC = struct.Struct("ii6qd15q")              # nnvb_attention_desc
# the current stream as an address, without a Stream object per call (a fifth of a small call's host time)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _explicit(*tensors):
    """Refuses what autograd would record: its backward pass would silently stop here."""
    if torch.is_grad_enabled() and any(getattr(t, "requires_grad", False) for t in tensors):
        raise ValueError("a tensor requires a gradient, which these operators do not record for autograd: call them under "
                         "torch.no_grad() and take the gradients from the _backward function")


def _kind(name, t):
    """The nnvb_dtype of a CUDA tensor."""
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch tensor" % name)
    kind = _DTYPES.get(t.dtype)
    if kind is None:
        raise TypeError("%s has element type %s (float64, float32, bfloat16 or float16 expected)" % (name, t.dtype))
    if not t.is_cuda:
        raise ValueError("%s is on %s; these operators have no CPU path" % (name, t.device))
    return kind


def _match(name, t, like):
    """A second tensor of a call: the first one's type and device."""
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch tensor" % name)
    if t.dtype is not like.dtype or t.get_device() != like.get_device():
        raise ValueError("%s (%s on %s) does not match the input (%s on %s)"
                         % (name, t.dtype, t.device, like.dtype, like.device))
    return t


def _stat_type(t):
    return torch.float64 if t.dtype is torch.float64 else torch.float32


def _stat(name, t, shape, like):
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch tensor" % name)
    if t.dtype is not _stat_type(like) or t.get_device() != like.get_device() or t.shape != shape:
        raise ValueError("%s must be a %s tensor of shape %s on %s" % (name, _stat_type(like), tuple(shape), like.device))
    return t.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _like(t):
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _launch(dev, name, *args):
    """Call a library entry on torch's current stream of device ``dev``, with that device current."""
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(L.load(), name)
    if torch.cuda.current_device() == dev:
        status = fn(_raw_stream(dev), *args)
    else:
        with torch.cuda.device(dev):
            status = fn(_raw_stream(dev), *args)
    if status:
        L.check(status, name)


def _rows(t, cols):
    """(tensor, rows, elements from row to row) of t[..., cols] seen as rows; copies what has no single row stride."""
    rows = t.numel() // cols
    if t.is_contiguous():
        return t, rows, cols
    if t.dim() == 2 and t.stride(1) == 1 and (rows <= 1 or t.stride(0) >= cols):
        return t, rows, (t.stride(0) if rows > 1 else cols)
    return t.contiguous(), rows, cols


def _ln_input(x):
    kind = _kind("x", x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must have at least one dimension, the normalised one, and at least one column")
    return kind, x.shape[-1]


def _weight(name, w, cols, x):
    if w is None:
        return None
    _match(name, w, x)
    if w.shape != (cols,):
        raise ValueError("%s must have one entry per column (%d), got shape %s" % (name, cols, tuple(w.shape)))
    return w.contiguous()


def layer_norm(x, scale=None, offset=None, eps=1e-5, return_stats=False):
    """(x - mean) / sqrt(var + eps) * scale + offset over the last dimension of ``x``.

    ``scale`` and ``offset`` (one entry per column) may be None.  With ``return_stats`` the rows' mean and
    1/sqrt(var + eps) come back too, shaped like ``x`` without its last dimension: what the backward call takes."""
    _explicit(x, scale, offset)
    kind, cols = _ln_input(x)
    scale, offset = _weight("scale", scale, cols, x), _weight("offset", offset, cols, x)
    eps = float(eps)
    if not (eps >= 0 and math.isfinite(eps)):
        raise ValueError("eps must be finite and not negative")
    xr, rows, ldx = _rows(x, cols)
    y = _like(x)
    mean = rstd = None
    if return_stats:
        mean = torch.empty(x.shape[:-1], dtype=_stat_type(x), device=x.device)
        rstd = torch.empty_like(mean)
    _launch(x.get_device(), "nnvb_layer_norm_forward", kind, rows, cols, xr.data_ptr(), ldx, _ptr(scale), _ptr(offset),
            eps, y.data_ptr(), cols, _ptr(mean), _ptr(rstd))
    return (y, mean, rstd) if return_stats else y


def layer_norm_backward(dy, x, scale, mean, rstd):
    """Gradients (dx, dscale, doffset) of ``layer_norm``: ``dy`` the gradient of its output, ``mean`` and ``rstd``
    its statistics.  The weights' gradients are sums over all rows, in a fixed order; with ``scale`` None they
    are those of a scale of ones."""
    kind, cols = _ln_input(x)
    _match("dy", dy, x)
    if dy.shape != x.shape:
        raise ValueError("dy has shape %s, x %s" % (tuple(dy.shape), tuple(x.shape)))
    scale = _weight("scale", scale, cols, x)
    mean, rstd = _stat("mean", mean, x.shape[:-1], x), _stat("rstd", rstd, x.shape[:-1], x)
    xr, rows, ldx = _rows(x, cols)
    gr, _, ldg = _rows(dy, cols)
    dx = _like(x)
    dscale = x.new_empty(cols) if scale is None else torch.empty_like(scale)
    doffset = torch.empty_like(dscale)
    nbytes = L.load().nnvb_layer_norm_workspace(kind, rows, cols)
    ws = mean.new_empty(nbytes // mean.element_size()) if nbytes else None
    _launch(x.get_device(), "nnvb_layer_norm_backward", kind, rows, cols, gr.data_ptr(), ldg, xr.data_ptr(), ldx,
            _ptr(scale), mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), cols, dscale.data_ptr(), doffset.data_ptr(),
            _ptr(ws), nbytes)
    return dx, dscale, doffset


def _heads(name, t):
    if t.dim() != 4:
        raise ValueError("%s must be [batch, tokens, heads, head size], got shape %s" % (name, tuple(t.shape)))
    # the kernels take any strides but need a head's elements side by side
    return t if t.stride(3) == 1 or t.shape[3] <= 1 else t.contiguous()


def _attn(q, k, v, lengths, scale):
    """Checked (q, k, v, lengths) and the fields of their nnvb_attention_desc up to the output's strides."""
    kind = _kind("q", q)
    q, k, v = _heads("q", q), _heads("k", _match("k", k, q)), _heads("v", _match("v", v, q))
    B, Lq, Hq, D = q.shape
    if k.shape != v.shape:
        raise ValueError("k and v differ in shape: %s, %s" % (tuple(k.shape), tuple(v.shape)))
    Bk, Lk, Hkv, Dk = k.shape
    if Bk != B or Dk != D:
        raise ValueError("q %s and k %s differ in batch or head size" % (tuple(q.shape), tuple(k.shape)))
    if Hq < 1 or Hkv < 1 or Hq % Hkv:
        raise ValueError("%d query heads cannot share %d state heads evenly" % (Hq, Hkv))
    if not 1 <= D <= 256:
        raise ValueError("head size %d is outside 1..256" % D)
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    else:
        scale = float(scale)
        if not (math.isfinite(scale) and scale > 0):
            raise ValueError("scale must be finite and positive")
    if lengths is not None:
        if not isinstance(lengths, torch.Tensor) or lengths.dtype is not torch.int32 \
                or lengths.get_device() != q.get_device() or lengths.shape != (B,):
            raise ValueError("lengths must be an int32 tensor with one entry per batch entry on %s" % q.device)
        lengths = lengths.contiguous()
    sq, sk, sv = q.stride(), k.stride(), v.stride()
    return q, k, v, lengths, (kind, 0, B, Lq, Lk, Hq, Hkv, D, scale, sq[0], sq[1], sq[2], sk[0], sk[1], sk[2],
                              sv[0], sv[1], sv[2])


def cross_attention(q, k, v, lengths=None, scale=None, return_lse=False):
    """softmax(scale * q k^T) v of the positions q [B, Lq, Hq, D] over an encoder's states k, v [B, Lk, Hkv, D].

    Hq is a multiple of Hkv: query head h reads state head h // (Hq / Hkv).  ``lengths`` (int32 [B], on the device)
    gives the valid states of each batch entry, clipped to 0..Lk; what the others hold has no effect.  Rows
    without a valid state are zero.  ``scale`` defaults to 1/sqrt(D).  Tensors may be strided views.  With
    ``return_lse`` the log-sum-exp [B, Hq, Lq] of each row's scores comes back too (-inf without states)."""
    _explicit(q, k, v)
    q, k, v, lengths, head = _attn(q, k, v, lengths, scale)
    out = _like(q)
    so = out.stride()
    lse = torch.empty((q.shape[0], q.shape[2], q.shape[1]), dtype=_stat_type(q), device=q.device) if return_lse else None
    _launch(q.get_device(), "nnvb_cross_attention_forward", _DESC.pack(*head, so[0], so[1], so[2], 0, 0, 0), q.data_ptr(),
            k.data_ptr(), v.data_ptr(), _ptr(lengths), out.data_ptr(), _ptr(lse))
    return (out, lse) if return_lse else out


def cross_attention_backward(dout, q, k, v, out, lse, lengths=None, scale=None):
    """Gradients (dq, dk, dv) of ``cross_attention``: ``dout`` the gradient of its output, ``out`` and ``lse`` what it
    returned (``return_lse=True``).  dk and dv are summed, in a fixed order, over the query heads that share a state
    head, and are zero for states behind ``lengths``."""
    q, k, v, lengths, head = _attn(q, k, v, lengths, scale)
    dout, out = _heads("dout", _match("dout", dout, q)), _heads("out", _match("out", out, q))
    if dout.shape != q.shape or out.shape != q.shape:
        raise ValueError("dout %s and out %s must be shaped like q %s" % (tuple(dout.shape), tuple(out.shape), tuple(q.shape)))
    lse = _stat("lse", lse, (q.shape[0], q.shape[2], q.shape[1]), q)
    so, sd = out.stride(), dout.stride()
    desc = _DESC.pack(*head, so[0], so[1], so[2], sd[0], sd[1], sd[2])
    dq, dk = _like(q), _like(k)
    dv = torch.empty_like(dk)
    nbytes = L.load().nnvb_cross_attention_workspace(desc)
    ws = lse.new_empty(nbytes // lse.element_size())
    _launch(q.get_device(), "nnvb_cross_attention_backward", desc, dout.data_ptr(), q.data_ptr(), k.data_ptr(),
            v.data_ptr(), out.data_ptr(), lse.data_ptr(), _ptr(lengths), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
            ws.data_ptr(), nbytes)
    return dq, dk, dv
