"""What the transformer operators refuse, checked without a GPU: nothing below launches a kernel."""
import ctypes as C

import pytest
import torch

from nnv_b200 import _lib, ops

FAKE = 1 << 20          # never dereferenced: every call below is refused first


def _desc(**kw):
    d = _lib.AttentionDesc(_lib.BF16, 0, 2, 3, 4, 8, 2, 16, 0.25, (384, 128, 16), (128, 32, 16), (128, 32, 16),
                           (384, 128, 16), (384, 128, 16))
    for k, v in kw.items():
        setattr(d, k, v if not isinstance(v, tuple) else (C.c_int64 * 3)(*v))
    return d


def test_descriptor_layout():
    assert C.sizeof(_lib.AttentionDesc) == 8 + 6 * 8 + 8 + 5 * 24
    assert _lib.AttentionDesc.scale.offset == 56 and _lib.AttentionDesc.q_stride.offset == 64
    d = _desc()
    packed = ops._DESC.pack(_lib.BF16, 0, 2, 3, 4, 8, 2, 16, 0.25, *d.q_stride, *d.k_stride, *d.v_stride, *d.out_stride,
                            *d.dout_stride)
    assert packed == bytes(d)


@pytest.mark.parametrize("change,word", [
    ({"dtype": 7}, "element type"), ({"batch": -1}, "bad sizes"), ({"kv_len": 1 << 31}, "bad sizes"),
    ({"q_len": 1 << 30}, "bad sizes"),
    ({"q_heads": 7}, "heads"), ({"kv_heads": 0}, "heads"), ({"head_dim": 0}, "head size"), ({"head_dim": 257}, "head size"),
    ({"scale": 0.0}, "factor"), ({"scale": float("nan")}, "factor"), ({"scale": 1e300}, "factor"),
    ({"scale": 1e-60}, "factor"), ({"k_stride": (-1, 0, 0)}, "negative stride"),
    ({"out_stride": (384, 128, 8)}, "overlap"), ({"out_stride": (0, 128, 16)}, "overlap")])
def test_attention_forward_refuses(change, word):
    lib = _lib.load()
    s = lib.nnvb_cross_attention_forward(None, C.byref(_desc(**change)), FAKE, FAKE, FAKE, None, FAKE, None)
    assert s == _lib.NNVB_E_ARG and word in lib.nnvb_last_error().decode()


def test_attention_null_pointers_and_workspace():
    lib = _lib.load()
    d = _desc()
    assert lib.nnvb_cross_attention_forward(None, None, FAKE, FAKE, FAKE, None, FAKE, None) == _lib.NNVB_E_ARG
    assert lib.nnvb_cross_attention_forward(None, C.byref(d), FAKE, None, FAKE, None, FAKE, None) == _lib.NNVB_E_ARG
    assert lib.nnvb_cross_attention_forward(None, C.byref(d), FAKE, FAKE, FAKE, None, None, None) == _lib.NNVB_E_ARG
    need = lib.nnvb_cross_attention_workspace(C.byref(d))
    assert need >= 2 * 3 * 8 * 4
    args = [FAKE] * 6 + [None] + [FAKE] * 3
    assert lib.nnvb_cross_attention_backward(None, C.byref(d), *args, FAKE, need - 1) == _lib.NNVB_E_ARG
    assert b"workspace" in lib.nnvb_last_error()
    assert lib.nnvb_cross_attention_backward(None, C.byref(d), *args, FAKE + 8, need) == _lib.NNVB_E_ARG
    assert lib.nnvb_cross_attention_backward(None, C.byref(d), *args, None, need) == _lib.NNVB_E_ARG
    args[5] = None                                                     # the log-sum-exp
    assert lib.nnvb_cross_attention_backward(None, C.byref(d), *args, FAKE, need) == _lib.NNVB_E_ARG
    # nothing to do is not an error and needs no memory
    assert lib.nnvb_cross_attention_forward(None, C.byref(_desc(batch=0)), None, None, None, None, None, None) == 0
    assert lib.nnvb_cross_attention_forward(None, C.byref(_desc(q_len=0)), None, None, None, None, None, None) == 0


def test_layer_norm_refuses():
    lib = _lib.load()
    fwd = lib.nnvb_layer_norm_forward
    assert fwd(None, 9, 2, 8, FAKE, 8, FAKE, FAKE, 1e-5, FAKE, 8, None, None) == _lib.NNVB_E_ARG
    assert fwd(None, _lib.F32, -1, 8, FAKE, 8, FAKE, FAKE, 1e-5, FAKE, 8, None, None) == _lib.NNVB_E_ARG
    assert fwd(None, _lib.F32, 2, 0, FAKE, 8, FAKE, FAKE, 1e-5, FAKE, 8, None, None) == _lib.NNVB_E_ARG
    assert fwd(None, _lib.F32, 2, 8, FAKE, 7, FAKE, FAKE, 1e-5, FAKE, 8, None, None) == _lib.NNVB_E_ARG
    assert b"overlap" in lib.nnvb_last_error()
    assert fwd(None, _lib.F32, 2, 8, FAKE, 8, FAKE, FAKE, -1.0, FAKE, 8, None, None) == _lib.NNVB_E_ARG
    assert fwd(None, _lib.F32, 2, 8, FAKE, 8, FAKE, FAKE, float("nan"), FAKE, 8, None, None) == _lib.NNVB_E_ARG
    assert fwd(None, _lib.F32, 2, 8, None, 8, FAKE, FAKE, 1e-5, FAKE, 8, None, None) == _lib.NNVB_E_ARG
    assert fwd(None, _lib.F32, 0, 8, None, 8, None, None, 1e-5, None, 8, None, None) == _lib.NNVB_OK
    bwd = lib.nnvb_layer_norm_backward
    need = lib.nnvb_layer_norm_workspace(_lib.F32, 1000, 1024)
    assert need >= 2 * 1024 * 4
    for ws, n in ((FAKE, need - 1), (FAKE + 4, need), (None, need)):
        assert bwd(None, _lib.F32, 1000, 1024, FAKE, 1024, FAKE, 1024, FAKE, FAKE, FAKE, FAKE, 1024, FAKE, FAKE, ws, n) == _lib.NNVB_E_ARG
        assert b"workspace" in lib.nnvb_last_error()
    assert lib.nnvb_layer_norm_workspace(_lib.F32, 2, 8) == 0                  # small tensors need none
    need = 0
    assert bwd(None, _lib.F32, 2, 8, FAKE, 8, FAKE, 8, FAKE, None, FAKE, FAKE, 8, FAKE, FAKE, FAKE, need) == _lib.NNVB_E_ARG
    assert bwd(None, _lib.F32, 2, 8, FAKE, 6, FAKE, 8, FAKE, FAKE, FAKE, FAKE, 8, FAKE, FAKE, FAKE, need) == _lib.NNVB_E_ARG


def test_python_refuses_before_anything_runs():
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="no CPU path"):
        ops.layer_norm(x)
    with pytest.raises(TypeError):
        ops.layer_norm(x.to(torch.int32))
    with pytest.raises(TypeError):
        ops.layer_norm([1.0])
    q = torch.zeros(2, 3, 4, 8)
    with pytest.raises(ValueError, match="no CPU path"):
        ops.cross_attention(q, q, q)
    with pytest.raises(TypeError):
        ops.cross_attention(q.to(torch.complex64), q, q)
