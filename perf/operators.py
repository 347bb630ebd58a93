"""What is measured of the transformer operators: layer normalisation and attention over an encoder's states.

``run`` computes a case in its plain form (elementary torch operations, ``own = False``) or through
``nnv_b200.ops`` (``own = True``).  Both get the same inputs from ``prepare``.

Layouts: layer norm works on rows, x[rows, cols].  Attention takes q[B, Lq, Hq, D] and the states' keys and
values k, v[B, Lk, Hkv, D] (Hq a multiple of Hkv; query head h reads state head h // (Hq / Hkv)); ``lengths[b]``
of the Lk states of batch entry b are valid, and an entry without states gives zero rows.  A backward case is
the backward call alone: what its forward call saved (statistics; output and log-sum-exp) is in hand before.
"""
import math
import random

import torch

own = False

TYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f64": 8, "f32": 4, "bf16": 2, "f16": 2}

# the largest drawn work: that of the largest listed case of each kind
LN_ELEMENTS = 16384 * 8192
ATT_PAIRS = {"bf16": 8 * 16 * 2048 * 4096 * 128, "f16": 8 * 16 * 2048 * 4096 * 128,
             "f32": 4 * 12 * 448 * 1500 * 64, "f64": 64 * 8 * 50 * 197 * 64}
STEP_STATES = 64 * 8 * 4096 * 128


def listed():
    return [
        # one decoder step of 8 sequences of width 768, normalised: all latency
        {"name": "ln_fwd_step", "op": "ln_fwd", "dtype": "bf16", "rows": 8, "cols": 768},
        # concrete evaluation of 1000 sampled inputs (falsification), 197 tokens each of width 192, in double
        {"name": "ln_fwd_samples_f64", "op": "ln_fwd", "dtype": "f64", "rows": 197000, "cols": 192},
        # a training batch of 16 384 tokens, width 8192
        {"name": "ln_fwd_train", "op": "ln_fwd", "dtype": "bf16", "rows": 16384, "cols": 8192},
        # its gradients
        {"name": "ln_bwd_train", "op": "ln_bwd", "dtype": "bf16", "rows": 16384, "cols": 8192},
        # a ragged small batch with an odd width, single precision
        {"name": "ln_bwd_odd_f32", "op": "ln_bwd", "dtype": "f32", "rows": 3001, "cols": 777},
        # decoder positions attending to long encoder states: the compute-bound case
        {"name": "ca_fwd_long", "op": "ca_fwd", "dtype": "bf16", "B": 8, "Lq": 2048, "Lk": 4096, "Hq": 16, "Hkv": 16,
         "D": 128, "ragged": False},
        # padded batch of short targets over 1500 states, grouped heads, one entry without states
        {"name": "ca_fwd_ragged", "op": "ca_fwd", "dtype": "f16", "B": 6, "Lq": 333, "Lk": 1500, "Hq": 12, "Hkv": 4,
         "D": 64, "ragged": True},
        # single precision evaluation of a mid-sized decoder
        {"name": "ca_fwd_f32", "op": "ca_fwd", "dtype": "f32", "B": 4, "Lq": 448, "Lk": 1500, "Hq": 12, "Hkv": 12,
         "D": 64, "ragged": False},
        # sampled inputs evaluated in double: 50 query tokens over 197 fixed states
        {"name": "ca_fwd_samples_f64", "op": "ca_fwd", "dtype": "f64", "B": 64, "Lq": 50, "Lk": 197, "Hq": 8, "Hkv": 8,
         "D": 64, "ragged": False},
        # one decoder step of a serving batch over its encoder states: bandwidth
        {"name": "ca_step_batch", "op": "ca_fwd", "dtype": "bf16", "B": 64, "Lq": 1, "Lk": 4096, "Hq": 32, "Hkv": 8,
         "D": 128, "ragged": True},
        # the gradients of a training step, padded states
        {"name": "ca_bwd_train", "op": "ca_bwd", "dtype": "bf16", "B": 4, "Lq": 2048, "Lk": 2048, "Hq": 16, "Hkv": 16,
         "D": 128, "ragged": False},
        # gradients with shared heads, ragged lengths and an odd number of positions
        {"name": "ca_bwd_ragged", "op": "ca_bwd", "dtype": "bf16", "B": 6, "Lq": 333, "Lk": 777, "Hq": 12, "Hkv": 4,
         "D": 64, "ragged": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["ln_fwd", "ln_bwd", "ca_fwd", "ca_step", "ca_bwd"])
    if op in ("ln_fwd", "ln_bwd"):
        dtype = rng.choice(["f64", "f32", "bf16", "f16"])
        cols = _log(rng, 8, 16384)
        rows = _log(rng, 1, 262144)
        return {"op": op, "dtype": dtype, "rows": max(1, min(rows, LN_ELEMENTS * 2 // (BYTES[dtype] * cols))), "cols": cols}
    if op == "ca_step":
        c = {"op": "ca_fwd", "dtype": rng.choice(["bf16", "f16"]), "B": _log(rng, 1, 128), "Lq": 1, "Lk": _log(rng, 1, 32768),
             "Hkv": rng.choice([1, 2, 4, 8, 12, 16]), "D": rng.choice([64, 80, 96, 128]), "ragged": rng.random() < 0.5}
        c["Hq"] = c["Hkv"] * rng.choice([1, 1, 2, 4, 8])
        c["Lk"] = max(1, min(c["Lk"], STEP_STATES // (c["B"] * c["Hkv"] * c["D"])))
        return c
    dtype = rng.choice(["bf16", "bf16", "f16", "f32", "f64"])
    c = {"op": op, "dtype": dtype, "B": _log(rng, 1, 32), "Lq": _log(rng, 2, 4096), "Lk": _log(rng, 1, 8192),
         "Hkv": rng.choice([1, 2, 4, 8, 12, 16]), "D": rng.choice([32, 64, 80, 96, 128]), "ragged": rng.random() < 0.5}
    c["Hq"] = c["Hkv"] * rng.choice([1, 1, 1, 2, 4])
    # a backward pass costs 2.5 times its forward pass; the largest listed case stays the largest.  The gradients of
    # a softmax over one state vanish, so a backward case has a few states at least
    most = ATT_PAIRS[dtype] / (2.5 if op == "ca_bwd" else 1.0)
    least = 8 if op == "ca_bwd" else 1
    c["Lk"] = max(least, min(c["Lk"], int(most // (c["B"] * c["Lq"] * c["Hq"] * c["D"]))))
    c["Lq"] = max(2, min(c["Lq"], int(most // (c["B"] * c["Lk"] * c["Hq"] * c["D"]))))
    return c


def _lengths(c):
    """Valid states per batch entry: all of them, or (ragged) spread over 1..Lk with an empty entry in larger batches."""
    if not c["ragged"]:
        return None
    r = random.Random(c["B"] * 1000003 + c["Lk"])
    n = [r.randint(1, c["Lk"]) for _ in range(c["B"])]
    n[0] = c["Lk"]
    if c["B"] >= 4:
        n[2] = 0
    return n


def _inputs(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 17)
    t = TYPES[c["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float64 if t is torch.float64 else torch.float32)

    if c["op"].startswith("ln"):
        rows, cols = c["rows"], c["cols"]
        # activations: a row has its own mean and spread
        s = {"x": (normal(rows, cols) * (0.5 + normal(rows, 1).abs()) + 0.3 * normal(rows, 1)).to(t),
             "scale": (1.0 + 0.1 * normal(cols)).to(t), "offset": (0.1 * normal(cols)).to(t)}
        if c["op"] == "ln_bwd":
            s["dy"] = normal(rows, cols).to(t)
        return s
    B, Lq, Lk, Hq, Hkv, D = (c[n] for n in ("B", "Lq", "Lk", "Hq", "Hkv", "D"))
    s = {"q": (1.5 * normal(B, Lq, Hq, D)).to(t), "k": normal(B, Lk, Hkv, D).to(t), "v": normal(B, Lk, Hkv, D).to(t)}
    if c["op"] == "ca_bwd":
        s["dout"] = normal(B, Lq, Hq, D).to(t)
    return s


def prepare(case, seed):
    s = {"case": case, "eps": 1e-5, **_inputs(case, seed)}
    if case["op"] == "ln_bwd":
        x = s["x"].double()
        mean = x.mean(1)
        st = torch.float64 if case["dtype"] == "f64" else torch.float32
        s["mean"] = mean.to(st)
        s["rstd"] = ((x - mean[:, None]).square().mean(1) + s["eps"]).rsqrt().to(st)
    if case["op"].startswith("ca"):
        n = _lengths(case)
        s["lengths"] = None if n is None else torch.tensor(n, dtype=torch.int32, device="cuda")
        if case["op"] == "ca_bwd":
            s["out"], s["lse"] = _plain_attention(s)
    return s


def _wide(x):
    return x if x.dtype is torch.float64 else x.float()


def _plain_ln(s):
    x = _wide(s["x"])
    mean = x.mean(1, keepdim=True)
    xc = x - mean
    rstd = 1.0 / torch.sqrt((xc * xc).mean(1, keepdim=True) + s["eps"])
    return xc * rstd, rstd


def _plain_weights(s):
    """Softmax weights [B, Hkv, G, Lq, Lk] and log-sum-exp [B, Hkv, G, Lq] in 32 (64) bits."""
    q, k = _wide(s["q"]), _wide(s["k"])
    B, Lq, Hq, D = q.shape
    Lk, Hkv = k.shape[1], k.shape[2]
    qg = q.reshape(B, Lq, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4)
    sc = torch.matmul(qg, k.permute(0, 2, 3, 1)[:, :, None]) * (1.0 / math.sqrt(D))
    if s["lengths"] is not None:
        off = torch.arange(Lk, device=q.device)[None, :] >= s["lengths"][:, None]
        sc.masked_fill_(off[:, None, None, None, :], float("-inf"))
    m = sc.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    p = torch.exp(sc.sub_(m))
    l = p.sum(-1, keepdim=True)
    lse = torch.where(l > 0, m + torch.log(l), torch.full_like(l, float("-inf")))[..., 0]
    p = p.div_(torch.where(l > 0, l, torch.ones_like(l)))
    return p, lse


def _plain_attention(s):
    p, lse = _plain_weights(s)
    v = _wide(s["v"]).permute(0, 2, 1, 3)[:, :, None]
    o = torch.matmul(p, v).permute(0, 3, 1, 2, 4)
    return o.reshape(s["q"].shape).to(s["q"].dtype), lse.reshape(lse.shape[0], -1, lse.shape[-1]).contiguous()


def _plain_attention_backward(s):
    p, _ = _plain_weights(s)
    q, k, v, do = _wide(s["q"]), _wide(s["k"]), _wide(s["v"]), _wide(s["dout"])
    B, Lq, Hq, D = q.shape
    Hkv = k.shape[2]
    G = Hq // Hkv
    qg = q.reshape(B, Lq, Hkv, G, D).permute(0, 2, 3, 1, 4)
    dog = do.reshape(B, Lq, Hkv, G, D).permute(0, 2, 3, 1, 4)
    dv = torch.matmul(p.transpose(-1, -2), dog).sum(2)
    dp = torch.matmul(dog, v.permute(0, 2, 3, 1)[:, :, None])
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * (1.0 / math.sqrt(D))
    dq = torch.matmul(ds, k.permute(0, 2, 1, 3)[:, :, None]).permute(0, 3, 1, 2, 4).reshape(q.shape)
    dk = torch.matmul(ds.transpose(-1, -2), qg).sum(2)
    t = s["q"].dtype
    return dq.to(t), dk.permute(0, 2, 1, 3).contiguous().to(t), dv.permute(0, 2, 1, 3).contiguous().to(t)


def run(s):
    op = s["case"]["op"]
    if own:
        from nnv_b200 import ops
        if op == "ln_fwd":
            return ops.layer_norm(s["x"], s["scale"], s["offset"], s["eps"])
        if op == "ln_bwd":
            return ops.layer_norm_backward(s["dy"], s["x"], s["scale"], s["mean"], s["rstd"])
        if op == "ca_fwd":
            return ops.cross_attention(s["q"], s["k"], s["v"], s["lengths"])
        return ops.cross_attention_backward(s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"], s["lengths"])
    if op == "ln_fwd":
        xh, _ = _plain_ln(s)
        return (xh * _wide(s["scale"]) + _wide(s["offset"])).to(s["x"].dtype)
    if op == "ln_bwd":
        xh, rstd = _plain_ln(s)
        dy, t = _wide(s["dy"]), s["x"].dtype
        gdy = dy * _wide(s["scale"])
        dx = rstd * (gdy - gdy.mean(1, keepdim=True) - xh * (gdy * xh).mean(1, keepdim=True))
        return dx.to(t), (dy * xh).sum(0).to(t), dy.sum(0).to(t)
    if op == "ca_fwd":
        return _plain_attention(s)[0]
    return _plain_attention_backward(s)


def _pairs(c):
    n = _lengths(c)
    return c["Lq"] * c["Hq"] * (c["B"] * c["Lk"] if n is None else sum(n)), (c["B"] * c["Lk"] if n is None else sum(n))


def work(c):
    e = BYTES[c["dtype"]]
    if c["op"] == "ln_fwd":
        n = c["rows"] * c["cols"]
        return {"bytes": e * (2 * n + 2 * c["cols"]), "flops": 7 * n}
    if c["op"] == "ln_bwd":
        n = c["rows"] * c["cols"]
        return {"bytes": e * (3 * n + 3 * c["cols"]) + 2 * c["rows"] * (8 if e == 8 else 4), "flops": 14 * n}
    pairs, states = _pairs(c)
    nq, nk = c["B"] * c["Lq"] * c["Hq"] * c["D"], c["B"] * c["Lk"] * c["Hkv"] * c["D"]
    read = states * c["Hkv"] * c["D"]
    if c["op"] == "ca_fwd":
        return {"bytes": e * (2 * nq + 2 * read), "flops": 4 * pairs * c["D"]}
    # reads q, k, v, out, dout and the log-sum-exp, writes dq, dk, dv; five products a pair
    return {"bytes": e * (4 * nq + 2 * read + 2 * nk) + 4 * c["B"] * c["Lq"] * c["Hq"], "flops": 10 * pairs * c["D"]}


def exact(case, seed):
    """The definitions in 64 bits, one batch entry and head at a time, written apart from the plain form."""
    s = prepare(case, seed)
    op = case["op"]
    if op.startswith("ln"):
        x, w = s["x"].double(), s["scale"].double()
        n = x.shape[1]
        var, mu = torch.var_mean(x, 1, unbiased=False, keepdim=True)
        sd = torch.sqrt(var + s["eps"])
        z = (x - mu) / sd
        if op == "ln_fwd":
            return z * w + s["offset"].double()
        dz = s["dy"].double() * w
        dx = (n * dz - dz.sum(1, keepdim=True) - z * (dz * z).sum(1, keepdim=True)) / (n * sd)
        return dx, (s["dy"].double() * z).sum(0), s["dy"].double().sum(0)
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    B, Lq, Hq, D = q.shape
    Hkv = k.shape[2]
    n = _lengths(case) or [case["Lk"]] * B
    outs = [torch.zeros_like(q)] if op == "ca_fwd" else [torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)]
    for b in range(B):
        for h in range(Hq if n[b] else 0):
            g = h // (Hq // Hkv)
            kk, vv, qq = k[b, :n[b], g], v[b, :n[b], g], q[b, :, h]
            p = torch.softmax(qq @ kk.T / math.sqrt(D), 1)
            if op == "ca_fwd":
                outs[0][b, :, h] = p @ vv
                continue
            do = s["dout"][b, :, h].double()
            dp = do @ vv.T
            ds = p * (dp - (p * dp).sum(1, keepdim=True)) / math.sqrt(D)
            outs[0][b, :, h] = ds @ kk
            outs[1][b, :n[b], g] += ds.T @ qq
            outs[2][b, :n[b], g] += p.T @ do
    return outs[0] if op == "ca_fwd" else tuple(outs)
