"""Layer normalisation and attention over an encoder's states in 64 bits on the CPU, each result with a bound on how
far a kernel that follows the formulas may be from it.

A rounding to type t is off by at most u_t = finfo(t).eps / 2 relative to the value.  Sums are held in 32 bits (64 for
double): u is half that type's eps.  A sum of n terms in a fixed order is off by at most (additions on the longest
path) * u * (sum of magnitudes).
"""
import numpy as np
import torch


def half_step(t):
    return torch.finfo(t).eps / 2


def acc_half_step(t):
    return 2.0 ** -53 if t is torch.float64 else 2.0 ** -24


# additions on the longest path of a row sum: 16 terms per thread in order, 5 shuffle steps, 16 warps, and the few
# operations each term takes; rows read by the wide form add cols / 1024 terms per thread (up to 64 in these tests)
LN_PATH = 128
# the same for the sums over rows: up to 40 rows per thread in these tests, 32 groups of a block, 128 partial rows per
# warp, 8 warps
LN_ROWS_PATH = 256


def layer_norm(x, scale, offset, eps, t):
    """y, mean, rstd and the bound on y's error."""
    u, ut = acc_half_step(t), half_step(t)
    x = x.double().cpu().numpy()
    s = np.ones(x.shape[1]) if scale is None else scale.double().cpu().numpy()
    o = np.zeros(x.shape[1]) if offset is None else offset.double().cpu().numpy()
    mean = x.mean(1, keepdims=True)
    rstd = 1.0 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + eps)
    z = (x - mean) * rstd
    y = z * s + o
    # z: the mean's error is LN_PATH u mean|x|, the subtraction's u |x - mean|, both times rstd; rstd's own relative
    # error comes from a sum of squares of deviations (LN_PATH u, halved by the root, plus the mean's error)
    big = np.abs(x).mean(1, keepdims=True) * rstd
    ez = LN_PATH * u * (big + np.abs(z) * (2 + big * big * LN_PATH * u))
    tol = ut * np.abs(y) + (1 + ut) * (ez * np.abs(s) + 3 * u * (np.abs(z * s) + np.abs(o)))
    return y, mean[:, 0], rstd[:, 0], tol


def layer_norm_backward(dy, x, scale, eps, t):
    """(dx, dscale, doffset) and their bounds."""
    u, ut = acc_half_step(t), half_step(t)
    x, dy = x.double().cpu().numpy(), dy.double().cpu().numpy()
    s = np.ones(x.shape[1]) if scale is None else scale.double().cpu().numpy()
    mean = x.mean(1, keepdims=True)
    rstd = 1.0 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + eps)
    z = (x - mean) * rstd
    g = dy * s
    m1, m2 = g.mean(1, keepdims=True), (g * z).mean(1, keepdims=True)
    dx = rstd * (g - m1 - z * m2)
    big = np.abs(x).mean(1, keepdims=True) * rstd
    ez = LN_PATH * u * (big + 2 * np.abs(z))
    e1 = LN_PATH * u * np.abs(g).mean(1, keepdims=True)
    e2 = LN_PATH * u * np.abs(g * z).mean(1, keepdims=True) + (np.abs(g) * ez).mean(1, keepdims=True)
    tdx = rstd * (e1 + np.abs(z) * e2 + ez * np.abs(m2) + 8 * u * (np.abs(g) + np.abs(m1) + np.abs(z * m2)))
    tdx = ut * np.abs(dx) + (1 + ut) * (tdx + LN_PATH * u * np.abs(dx))
    ds, do = (dy * z).sum(0), dy.sum(0)
    tds = ut * np.abs(ds) + (1 + ut) * (LN_ROWS_PATH * u * np.abs(dy * z).sum(0) + (np.abs(dy) * ez).sum(0))
    tdo = ut * np.abs(do) + (1 + ut) * LN_ROWS_PATH * u * np.abs(dy).sum(0)
    return (dx, ds, do), (tdx, tds, tdo)


def attention(q, k, v, lengths, scale, dout=None):
    """out and lse with their bounds, and with ``dout`` the gradients with theirs:
    {"out": (value, bound), "lse": ..., "dq": ..., "dk": ..., "dv": ...} as float64 arrays."""
    t = q.dtype
    u, ut = acc_half_step(t), half_step(t)
    # the 16-bit kernels round the weights P, and dS, once to the tensors' type before they meet V, K, Q and dO
    up = ut if t in (torch.bfloat16, torch.float16) else 0.0
    # fp16 weights below its smallest normal number are off by half the smallest subnormal instead
    tiny = 2.0 ** -25 if t is torch.float16 else 0.0
    Q, K, V = (x.double().cpu().numpy() for x in (q, k, v))
    G = None if dout is None else dout.double().cpu().numpy()
    B, Lq, Hq, D = Q.shape
    Lk, Hkv = K.shape[1:3]
    n = [Lk] * B if lengths is None else [min(max(int(x), 0), Lk) for x in lengths.cpu()]
    out, tout = np.zeros(Q.shape), np.zeros(Q.shape)
    lse, tlse = np.full((B, Hq, Lq), -np.inf), np.zeros((B, Hq, Lq))
    r = {"dq": np.zeros(Q.shape), "dk": np.zeros(K.shape), "dv": np.zeros(K.shape)}
    e = {x: np.zeros(r[x].shape) for x in r}
    for b in range(B):
        if n[b] == 0:
            continue
        for h in range(Hq):
            g = h // (Hq // Hkv)
            kk, vv, qq = K[b, :n[b], g], V[b, :n[b], g], Q[b, :, h]
            s = scale * (qq @ kk.T)
            m = s.max(1, keepdims=True)
            p = np.exp(s - m)
            l = p.sum(1, keepdims=True)
            p /= l
            lse[b, h], out[b, :, h] = (m + np.log(l))[:, 0], p @ vv
            # a score: D products added in some order, the factor (folded with log2 e), the subtraction of the
            # maximum; an error d of the exponent is a relative error d of the weight; exp2 itself 2 u; the sum
            # of the weights: n additions at most
            es = (D + 4) * u * scale * (np.abs(qq) @ np.abs(kk).T) + 4 * u * (np.abs(s) + np.abs(m))
            ep = es + 4 * u
            el = (p * ep).sum(1, keepdims=True) + (n[b] + 8) * u
            pv = p @ np.abs(vv)
            # tiny is relative to the row's running maximum, at least 2^-8 of the true one after a lazy rescale
            eo = (p * ep) @ np.abs(vv) + (el + (n[b] + 8) * u + up) * pv + (tiny / l) * np.abs(vv).sum(0)
            tout[b, :, h] = ut * np.abs(out[b, :, h]) + (1 + ut) * eo + (tiny if t is torch.float16 else 0)
            tlse[b, h] = (el[:, 0] + es.max(1) + 4 * u * (np.abs(lse[b, h]) + 1))
            if dout is None:
                continue
            do = G[b, :, h]
            dp = do @ vv.T
            de = (do * out[b, :, h]).sum(1, keepdims=True)
            ds = p * (dp - de)
            # P from the stored log-sum-exp; delta from the stored (rounded) output
            epb = ep + tlse[b, h][:, None]
            ede = (np.abs(do) * tout[b, :, h]).sum(1, keepdims=True) + (D + 2) * u * (np.abs(do) * np.abs(out[b, :, h])).sum(1, keepdims=True)
            edp = (D + 2) * u * (np.abs(do) @ np.abs(vv).T)
            eds = p * (epb * np.abs(dp - de) + edp + ede + 4 * u * (np.abs(dp) + np.abs(de))) + up * np.abs(ds) * (1 + epb) + tiny
            N = n[b] + 8
            r["dq"][b, :, h] = scale * (ds @ kk)
            e["dq"][b, :, h] = scale * (eds @ np.abs(kk) + N * u * (np.abs(ds) @ np.abs(kk)))
            N = Lq * (Hq // Hkv) + 8
            r["dk"][b, :n[b], g] += scale * (ds.T @ qq)
            e["dk"][b, :n[b], g] += scale * (eds.T @ np.abs(qq) + N * u * (np.abs(ds).T @ np.abs(qq)))
            r["dv"][b, :n[b], g] += p.T @ do
            e["dv"][b, :n[b], g] += (p * (epb + up) + tiny).T @ np.abs(do) + N * u * (p.T @ np.abs(do))
    res = {"out": (out, tout), "lse": (lse, tlse)}
    if dout is not None:
        for x in r:
            res[x] = (r[x], ut * np.abs(r[x]) + (1 + ut) * e[x] + (tiny if t is torch.float16 else 0))
    return res


def check(name, got, want, tol):
    got = got.double().cpu().numpy()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    both_inf = np.isinf(want) & (got == want)
    with np.errstate(invalid="ignore"):
        bad = ~(np.abs(got - want) <= tol) & ~both_inf
    assert not bad.any(), "%s: %d of %d outside the bound, worst %.3g times it" % (
        name, bad.sum(), bad.size, np.nanmax(np.abs(got - want)[bad] / np.maximum(tol[bad], 1e-300)))
