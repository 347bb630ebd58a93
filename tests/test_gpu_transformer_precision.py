"""What 16-bit attention must not lose: gradients over the whole range of their type, gradients of peaked rows, weights
of states that an outweighing one leaves small, and scores of -inf.

The gradients' measure is the error's relative 2-norm, row by row where no row is peaked, beside the same measure of the
exact gradient rounded once to its type.  (A row whose weight lies on one state has a dq around 1 - P; sums in 32 bits
leave 2^-24 of delta there, so its own relative error has no bound.)  dq and dk are sums of dS = P (dP - delta) times 16-bit inputs in 32 bits, so
that rounding is the only one of 2^-9 (bf16) or 2^-12 (fp16) root mean square.  All others are of 32-bit values, of
random sign, and together at most half of it: sqrt(1 + 1/4) = 1.12 times the storage rounding.  One rounding of dS to
16 bits, or of the output that delta is taken from, adds as much as the storage itself: 1.41 times.
"""
import math

import pytest
import torch

import transformer_reference as R

pytestmark = pytest.mark.gpu
F16 = [torch.bfloat16, torch.float16]
LIMIT = 1.12


def _data(t, B, Lq, Lk, Hq, Hkv, D, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)

    def r(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64)
    return (spread * r(B, Lq, Hq, D)).to(t), r(B, Lk, Hkv, D).to(t), r(B, Lk, Hkv, D).to(t), r(B, Lq, Hq, D)


def _formula(q, k, v, dout):
    """(dq, dk) in 64 bits on the CPU."""
    q, k, v, dout = (x.double() for x in (q, k, v, dout))
    B, Lq, Hq, D = q.shape
    Hkv = k.shape[2]
    qg, dg = (x.view(B, Lq, Hkv, Hq // Hkv, D) for x in (q, dout))
    p = (torch.einsum("bqhgd,bkhd->bhgqk", qg, k) / math.sqrt(D)).softmax(-1)
    dp = torch.einsum("bqhgd,bkhd->bhgqk", dg, v)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(D)
    return torch.einsum("bhgqk,bkhd->bqhgd", ds, k).reshape(q.shape), torch.einsum("bhgqk,bqhgd->bkhd", ds, qg)


def _row_error(x, want):
    e = (x.double() - want).norm(dim=-1) / want.norm(dim=-1).clamp_min(1e-300)
    return float(e.square().mean().sqrt())


def _error(x, want):
    return float((x.double() - want).norm() / want.norm())


def _check_gradients(q, k, v, dout, measure=_row_error):
    from nnv_b200 import ops
    t = q.dtype
    want = _formula(q, k, v, dout)
    dev = [x.cuda() for x in (q, k, v, dout)]
    out, lse = ops.cross_attention(*dev[:3], return_lse=True)
    got = ops.cross_attention_backward(dev[3], *dev[:3], out, lse)
    for name, a, b in zip(("dq", "dk"), got, want):
        a = a.cpu()
        assert a.isfinite().all(), name
        err, store = measure(a, b), measure(b.to(t), b)
        assert err <= LIMIT * store, "%s: %.3g, storage rounding %.3g" % (name, err, store)


@pytest.mark.parametrize("size", [1e-4, 1e-3, 1e-2, 1.0, 1e3])
@pytest.mark.parametrize("Lq,Lk,D", [(200, 100, 64), (200, 4000, 64), (130, 1500, 128)])
def test_half_precision_gradients_of_any_size(size, Lq, Lk, D):
    q, k, v, dout = _data(torch.float16, 1, Lq, Lk, 2, 1, D, spread=1.5)
    _check_gradients(q, k, v, (size * dout).half())


def test_half_precision_gradients_behind_the_type():
    """dS up to 99675, beyond fp16, where dq and dk stay below 60000."""
    q, k, v, dout = _data(torch.float16, 1, 64, 16, 1, 1, 64, seed=8, spread=1.5)
    _check_gradients(q, k, v, (12000 * dout).clamp(-46560, 46560).half())


def test_half_precision_gradients_of_uneven_rows():
    """Positions whose gradients differ by 2^20, none at all among them, and states whose values differ by 2^10."""
    q, k, v, dout = _data(torch.float16, 2, 150, 700, 4, 2, 64, spread=1.5)
    dout *= torch.logspace(-10, 10, 150, base=2.0)[None, :, None, None]
    v = (v.double() * torch.logspace(5, -5, 700, base=2.0)[None, :, None, None]).half()
    dout[:, 7] = 0
    _check_gradients(q, k, v, dout.half())


@pytest.mark.parametrize("t", F16)
@pytest.mark.parametrize("spread", [1.0, 4.0, 16.0])
@pytest.mark.parametrize("Lq,Lk,H", [(150, 128, 2), (150, 129, 2), (100, 4096, 1), (600, 300, 16)])
def test_gradients_of_peaked_rows(t, spread, Lq, Lk, H):
    q, k, v, dout = _data(t, 1, Lq, Lk, H, 1, 64, spread=spread)
    _check_gradients(q, k, v, dout.to(t), _error)


@pytest.mark.parametrize("t", F16)
@pytest.mark.parametrize("spread", [4.0, 16.0])
@pytest.mark.parametrize("Lq,Lk,H,D", [(60, 400, 6, 136), (300, 70, 2, 256), (20, 3000, 1, 66)])
def test_gradients_of_peaked_rows_in_other_layouts(t, spread, Lq, Lk, H, D):
    """Heads that the tensor cores do not take: more than 128 channels, rows that are not whole 16-byte pieces."""
    q, k, v, dout = _data(t, 1, Lq, Lk, H, 1, D, spread=spread)
    _check_gradients(q, k, v, dout.to(t), _error)


@pytest.mark.parametrize("t", F16)
@pytest.mark.parametrize("Lq,Lk,D", [(130, 300, 64), (300, 1000, 128), (50, 5000, 64), (2, 300, 64)])
def test_scores_of_minus_infinity_weigh_nothing(t, Lq, Lk, D):
    from nnv_b200 import ops
    q, k, v, _ = _data(t, 1, Lq, Lk, 2, 2, D)
    q = q.abs()
    keep = torch.ones(Lk, dtype=torch.bool)
    keep[100::3] = False
    k[:, ~keep] = -math.inf
    big = torch.finfo(t).max
    v[:, ~keep] = big
    out, lse = ops.cross_attention(q.cuda(), k.cuda(), v.cuda(), return_lse=True)
    ref = R.attention(q, k[:, keep], v[:, keep], None, 1 / math.sqrt(D))
    R.check("out", out, *ref["out"])
    R.check("lse", lse, *ref["lse"])
    k[:] = -math.inf                           # softmax of nothing but -inf: 0 / 0
    v[:] = 1
    out, lse = ops.cross_attention(q.cuda(), k.cuda(), v.cuda(), return_lse=True)
    assert out.isnan().all() and (lse == -math.inf).all()


@pytest.mark.parametrize("Lq", [1, 4, 100])
def test_half_precision_keeps_small_weights_beside_an_outweighing_state(Lq):
    """One state holds nearly all weight and no value: the others' weights, around 2^-26 of it, make the output."""
    from nnv_b200 import ops
    t, Lk, D = torch.float16, 3000, 64
    q, k, v, _ = _data(t, 1, Lq, Lk, 1, 1, D)
    q[..., 0], k[..., 0] = 8.0, 0.0            # scores: 8 k_0 / 8 plus sigma 1 of the other channels
    k[:, 0] = 0
    k[:, 0, :, 0] = 18.0                       # e^18 = 2^26 times the others
    v[:, 1:] = 1000 * v[:, 1:].abs()
    v[:, 0] = 0
    out = ops.cross_attention(q.cuda(), k.cuda(), v.cuda()).cpu().double()
    p = (torch.einsum("bqhd,bkhd->bhqk", q.double(), k.double()) / 8).softmax(-1)
    want = torch.einsum("bhqk,bkhd->bqhd", p, v.double())
    # half a step of fp16 for each weight and for the output, fp32 arithmetic a 16th of that
    tol = 2.0 ** -11 * (2 + 1 / 16) * want
    R.check("out", out, want.numpy(), tol.numpy())


@pytest.mark.parametrize("t,size", [(torch.bfloat16, 300.0), (torch.bfloat16, 3000.0), (torch.bfloat16, 10000.0),
                                    (torch.float16, 300.0), (torch.float16, 3000.0)])
@pytest.mark.parametrize("Lq,Lk", [(2, 500), (200, 500), (100, 4000)])
def test_scores_of_millions_pick_a_state(t, size, Lq, Lk):
    """Scores of 1e5 to 1e9 whose rounding in 32 bits is up to dozens of powers of two, and gaps far wider than that: each
    row is the value of its largest score, to the roundings of a weight and of the output."""
    from nnv_b200 import ops
    q, k, v, _ = _data(t, 1, Lq, Lk, 2, 2, 64, spread=size)
    k = (size * k.double()).to(t)
    assert q.isfinite().all() and k.isfinite().all()
    s = torch.einsum("bqhd,bkhd->bhqk", q.double(), k.double()) / 8
    two = s.topk(2, -1).values
    clear = (two[..., 0] - two[..., 1]) > 64 * 2.0 ** -24 * torch.einsum("bqhd,bkhd->bhqk", q.double().abs(), k.double().abs()).amax(-1) / 8 + 40
    assert clear.double().mean() > 0.8
    out = ops.cross_attention(q.cuda(), k.cuda(), v.cuda()).cpu()
    assert out.isfinite().all()
    want = torch.stack([v[0, s[0, h].argmax(-1), h] for h in range(2)], 1)[None]
    # m c is rounded, so the weight is not quite 1: its own rounding to 16 bits is a half step, the output's another
    near = (out.double() - want.double()).abs() <= 2.02 * R.half_step(t) * want.double().abs()
    assert (near.all(-1) | ~clear.transpose(1, 2)).all()


@pytest.mark.parametrize("t", F16)
@pytest.mark.parametrize("Lq,G,Lk,D", [(1, 1, 900, 64), (1, 8, 4097, 128), (4, 4, 300, 64), (3, 5, 2000, 96)])
def test_few_rows_round_only_what_they_store(t, Lq, G, Lk, D):
    """Weights as two 16-bit terms: one would add as much as the storage rounding (1.41 times it)."""
    from nnv_b200 import ops
    q, k, v, _ = _data(t, 4, Lq, Lk, 2 * G, 2, D, spread=1.5)
    out = ops.cross_attention(q.cuda(), k.cuda(), v.cuda()).cpu()
    p = (torch.einsum("bqhgd,bkhd->bhgqk", q.double().view(4, Lq, 2, G, D), k.double()) / math.sqrt(D)).softmax(-1)
    want = torch.einsum("bhgqk,bkhd->bqhgd", p, v.double()).reshape(out.shape)
    assert _error(out, want) <= LIMIT * _error(want.to(t), want)


def test_half_precision_backward_captured_twice():
    """Two graphs with a workspace each, replayed in turn on inputs whose size changes between replays."""
    from nnv_b200 import ops
    q, k, v, dout = _data(torch.float16, 2, 200, 400, 4, 2, 64, spread=2.0)
    q, k, v, dout = q.cuda(), k.cuda(), v.cuda(), dout.half().cuda()
    graphs = []
    for i in range(2):
        q_, d_ = q.clone(), dout.clone()
        ops.cross_attention(q_, k, v)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, lse = ops.cross_attention(q_, k, v, return_lse=True)
            grads = ops.cross_attention_backward(d_, q_, k, v, out, lse)
        graphs.append((graph, q_, d_, grads))
    for size in (1.0, 2.0 ** -12, 2.0 ** 9):
        for i, (graph, q_, d_, grads) in enumerate(graphs):
            d_.copy_(dout * size * (i + 1))
            graph.replay()
        torch.cuda.synchronize()
        for graph, q_, d_, grads in graphs:
            out, lse = ops.cross_attention(q_, k, v, return_lse=True)
            assert all(torch.equal(a, b) for a, b in zip(grads, ops.cross_attention_backward(d_, q_, k, v, out, lse)))
            assert all(g.isfinite().all() and g.any() for g in grads)
