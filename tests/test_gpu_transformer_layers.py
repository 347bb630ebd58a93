"""Networks with layer normalisation and attention layers through NN.evaluate and NN.falsify, and the same run of
operators on device tensors: layer norm, attention over an encoder's states, their gradients."""
import math

import numpy as np
import pytest

from nnv_b200 import _lib
from nnv_b200 import nn


def _ln(x, s, o, eps):
    z = (x - x.mean(0)) / np.sqrt(x.var(0) + eps)
    return z * s[:, None] + o[:, None]


def _attend(q, K, V, heads, scale):
    c, hk, _ = K.shape
    out = np.zeros_like(q)
    for h in range(heads):
        k, v = K[:, h // (heads // hk)], V[:, h // (heads // hk)]
        s = scale * (q[h * c:(h + 1) * c].T @ k)
        p = np.exp(s - s.max(1, keepdims=True))
        out[h * c:(h + 1) * c] = v @ (p / p.sum(1, keepdims=True)).T
    return out


# float64 sums of a few hundred terms of order one: 1e-12 is a few thousand roundings of 2^-53
TOL = 1e-12


@pytest.mark.gpu
@pytest.mark.parametrize("D,T,n", [(24, 5, 7), (16, 4, 3), (48, 1, 200), (8, 50, 2), (7, 3, 4), (7, 3, 2)])
def test_layer_norm_layer(ctx, D, T, n):
    rng = np.random.default_rng(D + T)
    s, o = 1 + 0.1 * rng.standard_normal(D), rng.standard_normal(D)
    net = nn.NN([nn.LayerNormalizationLayer(D, s, o, 1e-6)])
    xs = [rng.standard_normal((D, T, 1)) for _ in range(n)]
    for x, y in zip(xs, net.evaluate(xs)):
        assert np.abs(y.reshape(D, T, order="F") - _ln(x[:, :, 0], s, o, 1e-6)).max() < TOL * 10
    plain = nn.NN([nn.LayerNormalizationLayer(D)])
    y = plain.evaluate(xs[0])
    assert np.abs(y.reshape(D, T, order="F") - _ln(xs[0][:, :, 0], np.ones(D), np.zeros(D), 1e-5)).max() < TOL * 10


@pytest.mark.gpu
@pytest.mark.parametrize("c,heads,hk,T,S,n", [(8, 4, 2, 5, 33, 6), (16, 2, 2, 1, 70, 130), (5, 3, 1, 3, 9, 4), (64, 2, 1, 2, 200, 3)])
def test_attention_layer(ctx, c, heads, hk, T, S, n):
    rng = np.random.default_rng(c)
    K, V = rng.standard_normal((c, hk, S)), rng.standard_normal((c, hk, S))
    xs = [rng.standard_normal((c * heads, T, 1)) for _ in range(n)]
    ys = nn.NN([nn.AttentionLayer(heads, K, V)]).evaluate(xs)
    flat = nn.NN([nn.AttentionLayer(heads, K.reshape(c * hk, S, order="F"), V.reshape(c * hk, S, order="F"), hk, 0.2)]).evaluate(xs)
    for x, y, z in zip(xs, ys, flat):
        assert np.abs(y.reshape(c * heads, T, order="F") - _attend(x[:, :, 0], K, V, heads, 1 / math.sqrt(c))).max() < TOL
        assert np.abs(z.reshape(c * heads, T, order="F") - _attend(x[:, :, 0], K, V, heads, 0.2)).max() < TOL


@pytest.mark.gpu
def test_decoder_block_evaluated_and_falsified(ctx):
    """FC -> layer norm -> FC -> attention over fixed states -> FC -> ReLU -> layer norm -> FC, as a network."""
    rng = np.random.default_rng(3)
    D, c, heads, S, out = 20, 8, 4, 50, 5
    W = [rng.standard_normal(s) / math.sqrt(s[1]) for s in ((D, 12), (c * heads, D), (D, c * heads), (out, D))]
    b = [0.1 * rng.standard_normal(w.shape[0]) for w in W]
    s, o = 1 + 0.1 * rng.standard_normal(D), 0.1 * rng.standard_normal(D)
    K, V = rng.standard_normal((c, 2, S)), rng.standard_normal((c, 2, S))
    net = nn.NN([nn.FullyConnectedLayer(W[0], b[0]), nn.LayerNormalizationLayer(D, s, o), nn.FullyConnectedLayer(W[1], b[1]),
                 nn.AttentionLayer(heads, K, V), nn.FullyConnectedLayer(W[2], b[2]), nn.ReluLayer(),
                 nn.LayerNormalizationLayer(D, s, o), nn.FullyConnectedLayer(W[3], b[3])])

    def ref(x):
        x = x.reshape(-1, 1)
        x = _ln(W[0] @ x + b[0][:, None], s, o, 1e-5)
        x = _attend(W[1] @ x + b[1][:, None], K, V, heads, 1 / math.sqrt(c))
        x = _ln(np.maximum(W[2] @ x + b[2][:, None], 0), s, o, 1e-5)
        return (W[3] @ x + b[3][:, None])[:, 0]
    xs = [rng.standard_normal(12) for _ in range(77)]
    for x, y in zip(xs, net.evaluate(xs)):
        assert np.abs(y - ref(x)).max() < 100 * TOL
    I = nn.Star(-np.ones(12), np.ones(12))
    centre = net.evaluate(np.zeros(12))
    U = nn.HalfSpace(np.eye(out)[:1], [centre[0]])
    found = net.falsify(I, U, 200, np.random.default_rng(1))
    assert found and all(ref(p)[0] <= centre[0] + 1e-9 for p in found)
    with pytest.raises(_lib.NNVError) as e:
        net.reach(I, {"reachMethod": "approx-star"})
    assert e.value.status == _lib.NNVB_E_UNSUPPORTED and "evaluated" in str(e.value)


@pytest.mark.gpu
def test_layers_that_do_not_fit_the_input(ctx):
    for layer, x in ((nn.LayerNormalizationLayer(8), np.zeros((4, 4, 1))), (nn.AttentionLayer(2, np.ones((4, 2, 3)), np.ones((4, 2, 3))), np.zeros(9)),
                     (nn.LayerNormalizationLayer(4), np.zeros((4, 4, 2)))):
        with pytest.raises(_lib.NNVError) as e:
            nn.NN([layer]).evaluate(x)
        assert e.value.status == _lib.NNVB_E_ARG


def test_layer_arguments():
    with pytest.raises(ValueError):
        nn.LayerNormalizationLayer(4, np.ones(3))
    with pytest.raises(ValueError):
        nn.LayerNormalizationLayer(4, Epsilon=-1)
    K = np.ones((4, 2, 3))
    for bad in ((3, K, K), (2, K, K[:, :1]), (2, K, K, 3), (2, K, K, 2, 0.0), (2, np.ones((7, 3)), np.ones((7, 3))),
                (1, np.ones((257, 1, 2)), np.ones((257, 1, 2))), (2, K[..., :0], K[..., :0])):
        with pytest.raises(ValueError):
            nn.AttentionLayer(*bad)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["float64", "bfloat16"])
def test_operators_in_a_row_with_gradients(name):
    """A pre-norm attention block on device tensors, its gradients against autograd of the formulas in 64 bits on
    the CPU.  bf16: every stage rounds to 2^-8 relative, a dozen roundings of values that stay of order one, so the
    relative 2-norm error is below 12 * 2^-8; float64: below 1e-11."""
    import torch
    from nnv_b200 import ops
    t = getattr(torch, name)
    g = torch.Generator().manual_seed(2)
    B, Lq, Lk, Hq, Hkv, c = 2, 70, 150, 4, 2, 64
    D = Hq * c

    def r(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64).to(t)
    x, s, o, k, v, dy = r(B, Lq, D), 1 + 0.1 * r(D), 0.1 * r(D), r(B, Lk, Hkv, c), r(B, Lk, Hkv, c), r(B, Lq, D)
    lengths = torch.tensor([150, 61], dtype=torch.int32)
    dev = [a.cuda() for a in (x, s, o, k, v, dy)]
    X, S, O, K, V, DY = dev
    q, mean, rstd = ops.layer_norm(X, S, O, return_stats=True)
    q4 = q.view(B, Lq, Hq, c)
    att, lse = ops.cross_attention(q4, K, V, lengths.cuda(), return_lse=True)
    y = X + att.view(B, Lq, D)
    dq, dk, dv = ops.cross_attention_backward(DY.view(B, Lq, Hq, c), q4, K, V, att, lse, lengths.cuda())
    dx, ds, do = ops.layer_norm_backward(dq.view(B, Lq, D), X, S, mean, rstd)
    dx = dx + DY
    leaves = [a.double().requires_grad_() for a in (x, s, o, k, v)]
    xx, ss, oo, kk, vv = leaves
    qq = torch.nn.functional.layer_norm(xx, (D,), ss, oo, 1e-5).view(B, Lq, Hkv, Hq // Hkv, c)
    sc = torch.einsum("bqhgd,bkhd->bhgqk", qq, kk) / math.sqrt(c)
    sc = sc.masked_fill((torch.arange(Lk)[None, :] >= lengths[:, None])[:, None, None, None, :], -math.inf)
    yy = xx + torch.einsum("bhgqk,bkhd->bqhgd", sc.softmax(-1), vv).reshape(B, Lq, D)
    yy.backward(dy.double())
    tol = 1e-11 if name == "float64" else 12 * 2.0 ** -8
    for got, want in zip((y, dx, ds, do, dk, dv), (yy.detach(), xx.grad, ss.grad, oo.grad, kk.grad, vv.grad)):
        err = (got.double().cpu() - want).norm() / want.norm()
        assert err < tol, err
