"""Attention over an encoder's states on device tensors against 64 bits, with bounds derived from the roundings made."""
import math

import numpy as np
import pytest
import torch

import transformer_reference as R

pytestmark = pytest.mark.gpu
TYPES = [torch.float64, torch.float32, torch.bfloat16, torch.float16]
F16 = [torch.bfloat16, torch.float16]


def _data(t, B, Lq, Lk, Hq, Hkv, D, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)

    def r(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64)
    q, k = (spread * r(B, Lq, Hq, D)).to(t).cuda(), r(B, Lk, Hkv, D).to(t).cuda()
    return q, k, r(B, Lk, Hkv, D).to(t).cuda(), r(B, Lq, Hq, D).to(t).cuda()


def _lens(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32).cuda()


def _check(t, q, k, v, dout, lengths, scale=None, backward=True):
    from nnv_b200 import ops
    out, lse = ops.cross_attention(q, k, v, lengths, scale, return_lse=True)
    ref = R.attention(q, k, v, lengths, scale or 1 / math.sqrt(q.shape[3]), dout if backward else None)
    R.check("out", out, *ref["out"])
    R.check("lse", lse, *ref["lse"])
    if backward:
        got = ops.cross_attention_backward(dout, q, k, v, out, lse, lengths, scale)
        for name, x in zip(("dq", "dk", "dv"), got):
            R.check(name, x, *ref[name])
        again = ops.cross_attention_backward(dout, q, k, v, out, lse, lengths, scale)
        assert all(torch.equal(a, b) for a, b in zip(got, again))      # a fixed order of additions
    return out, lse


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("Lq,Lk", [(1, 1), (1, 129), (2, 64), (5, 128), (64, 65), (127, 63), (128, 128), (129, 257), (300, 40)])
def test_lengths_around_the_tiles(t, Lq, Lk):
    _check(t, *_data(t, 2, Lq, Lk, 2, 2, 64), None)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("D", [1, 8, 20, 32, 33, 64, 72, 80, 96, 120, 128, 136, 200, 256])
def test_head_sizes(t, D):
    _check(t, *_data(t, 1, 70, 90, 2, 1, D), None)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("Hq,Hkv", [(6, 2), (8, 1), (3, 3)])
def test_shared_heads_and_ragged_lengths(t, Hq, Hkv):
    q, k, v, dout = _data(t, 5, 37, 200, Hq, Hkv, 64)
    lengths = _lens([200, 0, 1, 131, 64])
    out, lse = _check(t, q, k, v, dout, lengths)
    assert torch.equal(out[1], torch.zeros_like(out[1])) and (lse[1] == -math.inf).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("D", [64, 128, 80])
def test_what_lies_behind_the_lengths_has_no_effect(t, D):
    from nnv_b200 import ops
    q, k, v, dout = _data(t, 4, 150, 300, 4, 2, D)
    lengths = _lens([300, 0, 77, 256])
    out, lse = ops.cross_attention(q, k, v, lengths, return_lse=True)
    grads = ops.cross_attention_backward(dout, q, k, v, out, lse, lengths)
    for b, n in enumerate([300, 0, 77, 256]):
        k[b, n:] = math.nan
        v[b, n:] = math.inf if b % 2 else math.nan
    out2, lse2 = ops.cross_attention(q, k, v, lengths, return_lse=True)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    grads2 = ops.cross_attention_backward(dout, q, k, v, out, lse, lengths)
    assert all(torch.equal(a, b) for a, b in zip(grads, grads2))
    for b, n in enumerate([300, 0, 77, 256]):
        assert not grads[1][b, n:].any() and not grads[2][b, n:].any()
    assert not grads[0][1].any()
    # one step with few positions takes other kernels
    o1 = ops.cross_attention(q[:, :1], k, v, lengths)
    assert o1.isfinite().all() and not o1[1].any()


def test_lengths_are_clipped():
    from nnv_b200 import ops
    q, k, v, _ = _data(torch.bfloat16, 3, 20, 50, 2, 2, 64)
    a = ops.cross_attention(q, k, v, _lens([50, 0, 50]))
    b = ops.cross_attention(q, k, v, _lens([51, -3, 1 << 30]))
    assert torch.equal(a, b)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("Lq", [1, 2, 3, 4, 7])
@pytest.mark.parametrize("Lk,G", [(1, 1), (31, 4), (1000, 8), (4097, 2), (300, 3)])
def test_few_positions_over_many_states(t, Lq, Lk, G):
    q, k, v, dout = _data(t, 3, Lq, Lk, 2 * G, 2, 128)
    _check(t, q, k, v, dout, _lens([Lk, Lk // 2, 0]), backward=False)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,Lq,Lk,H", [(1, 100, 5000, 1), (1, 300, 2000, 2), (2, 20, 3000, 1), (1, 2000, 300, 1)])
def test_few_rows_over_a_long_axis(t, B, Lq, Lk, H, D):
    """Few tiles over many: clusters of blocks share one."""
    q, k, v, dout = _data(t, B, Lq, Lk, H, H, D)
    _check(t, q, k, v, dout, _lens([Lk - 70] * B))


@pytest.mark.parametrize("t", [torch.float64, torch.float32])
@pytest.mark.parametrize("D", [64, 80, 128])
def test_many_tiles_in_single_and_double(t, D):
    """Enough tiles on both sides for the large problems' kernels; grouped heads, ragged lengths, odd sizes."""
    q, k, v, dout = _data(t, 10, 99, 70, 16, 8, D)
    _check(t, q, k, v, dout, _lens([70, 0, 1, 64, 65, 33, 70, 12, 69, 3]))


@pytest.mark.parametrize("t", F16)
@pytest.mark.parametrize("D", [64, 128])
def test_clusters_with_ragged_lengths(t, D):
    """Entries whose states do not reach every block of the cluster, 128 and fewer states among them, and none."""
    q, k, v, dout = _data(t, 5, 40, 3000, 2, 1, D)
    lengths = _lens([3000, 0, 100, 129, 1000])
    for b, n in enumerate([3000, 0, 100, 129, 1000]):
        k[b, n:] = math.nan
        v[b, n:] = math.nan
    ref_k, ref_v = k.nan_to_num(), v.nan_to_num()
    from nnv_b200 import ops
    out, lse = ops.cross_attention(q, k, v, lengths, return_lse=True)
    ref = R.attention(q, ref_k, ref_v, lengths, 1 / math.sqrt(D), dout)
    R.check("out", out, *ref["out"])
    R.check("lse", lse, *ref["lse"])
    for name, x in zip(("dq", "dk", "dv"), ops.cross_attention_backward(dout, q, k, v, out, lse, lengths)):
        R.check(name, x, *ref[name])


@pytest.mark.parametrize("t", TYPES)
def test_large_scores_and_a_rising_maximum(t):
    """Scores that grow along the states: the running maximum moves at every tile."""
    q, k, v, dout = _data(t, 1, 130, 700, 2, 2, 64)
    q.copy_(q.abs())
    k.copy_((k.abs().double() * torch.linspace(0.1, 6, 700, device="cuda")[None, :, None, None]).to(t))
    _check(t, q, k, v, dout, None)


@pytest.mark.parametrize("Lq,Lk", [(2, 3000), (200, 4000)])
def test_small_weights_keep_their_bits_in_half_precision(Lq, Lk):
    """Weights around 1/Lk, many below the smallest normal fp16: dv to the rounding of its terms and of its own, without
    the absolute error that subnormal weights would add (2^-25 each, the allowance of the other tests)."""
    from nnv_b200 import ops
    q, k, v, dout = _data(torch.float16, 1, Lq, Lk, 2, 2, 64, spread=2.0)
    out, lse = ops.cross_attention(q, k, v, return_lse=True)
    dv = ops.cross_attention_backward(dout, q, k, v, out, lse)[2]
    want, _ = R.attention(q, k, v, None, 0.125, dout)["dv"]
    s = torch.einsum("bqhd,bkhd->bhqk", q.double(), k.double()) * 0.125
    spread = torch.einsum("bhqk,bqhd->bkhd", s.softmax(-1), dout.double().abs()).cpu().numpy()
    # rounding of each weight (half a step, 2^-11) and fp32 arithmetic (a 16th of it at most), then dv's own rounding,
    # which is absolute (2^-25) where dv itself is below the smallest normal number
    R.check("dv", dv, want, 2.0 ** -11 * (1 + 1 / 16) * spread + 2.0 ** -11 * abs(want) + 2.0 ** -25)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("Hq,Hkv,Lq", [(8, 2, 9), (12, 2, 50), (64, 1, 3), (128, 1, 5), (4, 2, 200)])
def test_grouped_heads_share_tiles(t, Hq, Hkv, Lq):
    """Groups of 4, 6, 64, 128 and 2 heads: positions of a group's heads are rows of one tile."""
    q, k, v, dout = _data(t, 2, Lq, 150, Hq, Hkv, 64)
    _check(t, q, k, v, dout, _lens([150, 61]))
    one = q[:, :, :1].expand(-1, -1, Hq, -1)                   # a broadcast query head is not packed
    out, lse = _check(t, one, k, v, dout, _lens([150, 61]))


@pytest.mark.parametrize("t", TYPES)
def test_scale_and_strided_views(t):
    from nnv_b200 import ops
    B, Lq, Lk, H, D = 2, 140, 150, 4, 64
    q, k, v, dout = _data(t, B, Lq, Lk, H, H, D)
    kv = torch.cat([k, v], -1)                                 # interleaved: strides over both
    kk, vv = kv[..., :D], kv[..., D:]
    qt = q.transpose(1, 2).contiguous().transpose(1, 2)        # heads before tokens
    dt = dout.transpose(1, 2).contiguous().transpose(1, 2)
    a, la = ops.cross_attention(q, k, v, None, 0.3, return_lse=True)
    b, lb = ops.cross_attention(qt, kk, vv, None, 0.3, return_lse=True)
    assert torch.equal(a, b) and torch.equal(la, lb)
    ga = ops.cross_attention_backward(dout, q, k, v, a, la, None, 0.3)
    gb = ops.cross_attention_backward(dt, qt, kk, vv, b.transpose(1, 2).contiguous().transpose(1, 2), lb, None, 0.3)
    assert all(torch.equal(x, y) for x, y in zip(ga, gb))
    _check(t, qt, kk, vv, dt, None, 0.3)
    one = k[:1].expand(B, -1, -1, -1)                          # the same states for every batch entry
    a = ops.cross_attention(q, one, one)
    b = ops.cross_attention(q, one.contiguous(), one.contiguous())
    R.check("broadcast", a, b.double().cpu().numpy(), R.attention(q, one, one, None, 1 / 8.0)["out"][1] * 2)
    odd = torch.empty(B, Lk, H, D + 1, dtype=t, device="cuda")[..., 1:]
    odd.copy_(k)                                               # rows that are not 16-byte aligned
    _check(t, q, odd, v, dout, None)
    last = q.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2)      # head elements apart: copied
    assert torch.equal(ops.cross_attention(last, k, v), ops.cross_attention(q, k, v))


def test_infinite_scores_follow_the_formula():
    from nnv_b200 import ops
    q, k, v, _ = _data(torch.float32, 1, 3, 70, 1, 1, 32)
    q.abs_()
    k[0, 5] = -math.inf                       # weight 0: as if the state were not there
    v[0, 5] = 0
    out = ops.cross_attention(q, k, v)
    keep = [i for i in range(70) if i != 5]
    ref = R.attention(q, k[:, keep], v[:, keep], None, 1 / math.sqrt(32))
    R.check("out", out, *ref["out"])


@pytest.mark.parametrize("t", TYPES)
def test_empty_sides(t):
    from nnv_b200 import ops
    q, k, v, dout = _data(t, 2, 3, 4, 2, 2, 16)
    out, lse = ops.cross_attention(q, k[:, :0], v[:, :0], return_lse=True)
    assert not out.any() and (lse == -math.inf).all()
    dq, dk, dv = ops.cross_attention_backward(dout, q, k[:, :0], v[:, :0], out, lse)
    assert not dq.any() and dk.shape == dv.shape == (2, 0, 2, 16)
    out, lse = ops.cross_attention(q[:, :0], k, v, return_lse=True)
    dq, dk, dv = ops.cross_attention_backward(dout[:, :0], q[:, :0], k, v, out, lse)
    assert out.shape == dq.shape == (2, 0, 2, 16) and not dk.any() and not dv.any()
    assert ops.cross_attention(q[:0], k[:0], v[:0]).shape == (0, 3, 2, 16)


def test_gradient_against_differences():
    from nnv_b200 import ops
    q, k, v, dout = _data(torch.float64, 2, 3, 5, 4, 2, 4)
    lengths = _lens([5, 3])
    out, lse = ops.cross_attention(q, k, v, lengths, return_lse=True)
    grads = ops.cross_attention_backward(dout, q, k, v, out, lse, lengths)
    step = 1e-5              # central differences: error step^2 / 6 * third derivative, plus 1e-16 / step
    for arg, grad in zip((q, k, v), grads):
        flat, gflat = arg.view(-1), grad.reshape(-1)
        for i in range(flat.numel()):
            keep = flat[i].item()
            flat[i] = keep + step
            up = (ops.cross_attention(q, k, v, lengths) * dout).sum().item()
            flat[i] = keep - step
            down = (ops.cross_attention(q, k, v, lengths) * dout).sum().item()
            flat[i] = keep
            assert abs((up - down) / (2 * step) - gflat[i].item()) < 1e-7


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_on_another_stream_and_captured(t):
    from nnv_b200 import ops
    q, k, v, dout = _data(t, 2, 200, 400, 4, 2, 64)
    out, lse = ops.cross_attention(q, k, v, return_lse=True)
    step = ops.cross_attention(q[:, :1], k, v)
    ref = ops.cross_attention_backward(dout, q, k, v, out, lse)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        o2 = ops.cross_attention(q, k, v)
        s2 = ops.cross_attention(q[:, :1], k, v)
    side.synchronize()
    assert torch.equal(out, o2) and torch.equal(step, s2)
    graphs, got = [], []
    for _ in range(2):                        # two graphs: each holds its own workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o, l = ops.cross_attention(q, k, v, return_lse=True)
            got.append((o, ops.cross_attention(q[:, :1], k, v), *ops.cross_attention_backward(dout, q, k, v, o, l)))
        graphs.append(graph)
    for _ in range(2):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for o, s, *g in got:
        assert torch.equal(o, out) and torch.equal(s, step) and all(torch.equal(a, b) for a, b in zip(g, ref))


@pytest.mark.parametrize("t", [torch.float64, torch.float32])
@pytest.mark.parametrize("D", [40, 64, 96, 128])
@pytest.mark.parametrize("Lq,Lk", [(300, 8), (300, 16), (150, 17), (150, 32), (150, 33), (10, 700), (17, 700), (33, 700)])
def test_one_short_side_in_single_and_double(t, D, Lq, Lk):
    q, k, v, dout = _data(t, 3, Lq, Lk, 2, 1, D)
    _check(t, q, k, v, dout, _lens([Lk, Lk // 2, 0]))


@pytest.mark.parametrize("t", [torch.float64, torch.float32])
@pytest.mark.parametrize("Lq,Lk", [(40, 600), (600, 40)])
def test_tiles_split_where_blocks_do_not_come_out_even(t, Lq, Lk):
    q, k, v, dout = _data(t, 10, Lq, Lk, 16, 16, 64)
    _check(t, q, k, v, dout, _lens([Lk, 0, 1, Lk - 1, 65, 64, 63, 17, Lk, 5]) if Lk > 64 else None)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("Lq,Lk,D", [(1, 40, 64), (24, 40, 64), (24, 40, 136)])
def test_offsets_past_32_bits(t, Lq, Lk, D):
    """Tokens so far apart that the last one begins more than 2^31 elements behind the first, in every operand."""
    q, k, v, dout = _data(t, 1, Lq, Lk, 2, 2, D)
    step = (1 << 31) // (Lk - 4) // 64 * 64
    far = torch.empty(step * Lk, dtype=t, device="cuda")
    views = [far.as_strided((1, n, 2, D), (step * Lk, step, D, 1), i * 1024) for i, n in enumerate((Lk, Lk, Lq, Lq))]
    for a, b in zip(views, (k, v, q, dout)):
        a.copy_(b)
    assert step * (Lk - 1) > 1 << 31
    _check(t, views[2], views[0], views[1], views[3], None)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("B,Lk", [(70, 1150), (128, 2100), (129, 300)])
def test_large_batches_of_single_positions(t, B, Lk):
    q, k, v, dout = _data(t, B, 1, Lk, 8, 8, 16)
    g = torch.Generator().manual_seed(5)
    lengths = torch.randint(0, Lk + 1, (B,), generator=g).tolist()
    lengths[:6] = [0, 0, Lk, Lk, 77, 77]
    out, _ = _check(t, q, k, v, dout, _lens(lengths), backward=False)
    assert torch.equal(out[:2], torch.zeros_like(out[:2]))


def test_two_streams_at_once():
    from nnv_b200 import ops
    sets = [_data(torch.bfloat16, 1, 300, 2000, 2, 2, 128), _data(torch.float16, 1, 500, 1500, 4, 1, 64),
            _data(torch.float32, 1, 100, 900, 2, 2, 64)]

    def work(q, k, v, dout):
        out, lse = ops.cross_attention(q, k, v, return_lse=True)
        return (out, ops.cross_attention(q[:, :1], k, v), *ops.cross_attention_backward(dout, q, k, v, out, lse))
    want = [work(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(5):
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(work(*s))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % len(sets)]))


def test_shapes_that_do_not_fit_are_refused():
    from nnv_b200 import ops
    q, k, v, dout = _data(torch.bfloat16, 2, 3, 4, 4, 2, 16)
    out, lse = ops.cross_attention(q, k, v, return_lse=True)
    for bad in (lambda: ops.cross_attention(q, k[:1], v[:1]), lambda: ops.cross_attention(q, k, v[:, :3]),
                lambda: ops.cross_attention(q[:, :, :3], k, v), lambda: ops.cross_attention(q[0], k, v),
                lambda: ops.cross_attention(q, k.float(), v), lambda: ops.cross_attention(q, k, v, _lens([1, 2, 3])),
                lambda: ops.cross_attention(q, k, v, torch.tensor([1, 2]).cuda()),
                lambda: ops.cross_attention(q, k, v, torch.tensor([1, 2], dtype=torch.int32)),
                lambda: ops.cross_attention(q, k, v, None, 0.0), lambda: ops.cross_attention(q, k, v, None, math.inf),
                lambda: ops.cross_attention_backward(dout[:, :2], q, k, v, out, lse),
                lambda: ops.cross_attention_backward(dout, q, k, v, out, lse.double()),
                lambda: ops.cross_attention_backward(dout, q, k, v, out, lse[:, :2])):
        with pytest.raises(ValueError):
            bad()
    assert np.isfinite(out.float().cpu().numpy()).all()
