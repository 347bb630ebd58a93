"""Reference-shaped host API over the CUDA engine.

Class and method names, argument meaning and error behaviour follow the
reference's MATLAB classes for the approx-star path, so that a script written
against ``NN.reach(inputSet, reachOptions)`` / ``NN.verify_robustness`` reads
the same here:

    NN                         code/nnv/engine/nn/NN.m
    ImageStar / Star           code/nnv/engine/set/ImageStar.m, Star.m
    HalfSpace                  code/nnv/engine/set/HalfSpace.m
    Conv2DLayer, FullyConnectedLayer, BatchNormalizationLayer,
    AveragePooling2DLayer, ReluLayer
                               code/nnv/engine/nn/layers/*.m
    verify_specification       code/nnv/engine/utils/verify_specification.m

All set arithmetic runs on the GPU through libnnvb200.so.  The one step that
stays on the host is the feasibility LP of Star.isEmptySet for halfspaces the
device tests leave undecided; the reference hands that LP to linprog/glpk
(lpsolver.m), this module hands it to HiGHS.
"""
from __future__ import annotations

import os
import time
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import scipy.sparse as sp
from scipy.optimize import linprog

from . import _lib as L
from .engine import Batch, Context, Network

__all__ = ["NN", "ImageStar", "Star", "HalfSpace", "ImageInputLayer", "FlattenLayer", "Conv2DLayer", "FullyConnectedLayer",
           "BatchNormalizationLayer", "AveragePooling2DLayer", "ReluLayer", "LayerNormalizationLayer", "AttentionLayer",
           "verify_specification",
           "default_context"]

_ctx = None


def default_context(device=0, arena_bytes=0):
    """Process-wide engine context (created on first use)."""
    global _ctx
    if _ctx is None:
        _ctx = Context(device, arena_bytes)
    return _ctx


# --------------------------------------------------------------------------- sets


class ImageStar:
    """ImageStar.m:47-94.  ``ImageStar(lb, ub)`` (ImageStar.m:302-343) or
    ``ImageStar(V, C, d, pred_lb, pred_ub)`` (ImageStar.m:172-227)."""

    def __init__(self, *args):
        self.im_lb = self.im_ub = None
        self._lazy = None
        if len(args) == 2:
            lb = np.asarray(args[0], dtype=np.float64)
            ub = np.asarray(args[1], dtype=np.float64)
            if lb.size == 0:
                raise ValueError("Invalid lower bound image")
            if ub.size == 0:
                raise ValueError("Invalid upper bound image")
            if lb.shape != ub.shape:
                raise ValueError("Inconsistency between lower bound image and upper bound image")
            if lb.ndim == 2:
                lb, ub = lb[:, :, None], ub[:, :, None]
            self.im_lb, self.im_ub = lb, ub
            self.height, self.width, self.numChannel = lb.shape
            n = lb.size
            lbv, ubv = lb.reshape(n, order="F"), ub.reshape(n, order="F")
            nz = np.nonzero(0.5 * (ubv - lbv) != 0)[0] if n > 1 else np.arange(1)
            self.numPred = len(nz)
            self._V = None                      # built on demand: centre + diag of half widths
            self._C = np.zeros((1, self.numPred))
            self.d = np.zeros(1)
            self.pred_lb = -np.ones(self.numPred)
            self.pred_ub = np.ones(self.numPred)
        elif len(args) == 5:
            V, Cm, d, pl, pu = args
            V = np.asfortranarray(np.asarray(V, dtype=np.float64))
            if V.ndim == 3:
                V = V[:, :, :, None]
            if V.ndim != 4:
                raise ValueError("Invalid basis matrix")
            Cm = np.atleast_2d(np.asarray(Cm, dtype=np.float64))
            d = np.asarray(d, dtype=np.float64).ravel()
            pl = np.asarray(pl, dtype=np.float64).ravel()
            pu = np.asarray(pu, dtype=np.float64).ravel()
            if Cm.size and Cm.shape[0] != d.size:
                raise ValueError("Inconsistent dimension between constraint matrix and constraint vector")
            if Cm.size and Cm.shape[1] != V.shape[3] - 1:
                raise ValueError("Inconsistent dimension between the basis matrix and the constraint matrix")
            if pl.size != pu.size or pl.size != V.shape[3] - 1:
                raise ValueError("Number of predicates is different from the size of the lower bound or upper bound predicate vector")
            self.height, self.width, self.numChannel = V.shape[:3]
            self.numPred = V.shape[3] - 1
            self._V, self._C, self.d, self.pred_lb, self.pred_ub = V, Cm, d, pl, pu
        else:
            raise ValueError("Invalid number of input arguments, (2 or 5)")

    # V and C may live on the device until somebody asks for them
    @property
    def V(self):
        if self._V is None:
            if self._lazy is not None:
                self._V = self._lazy[0].get_V(self._lazy[1])
            else:
                n = self.height * self.width * self.numChannel
                lbv = self.im_lb.reshape(n, order="F")
                ubv = self.im_ub.reshape(n, order="F")
                vec = 0.5 * (ubv - lbv)
                nz = np.nonzero(vec != 0)[0] if n > 1 else np.arange(1)
                M = np.zeros((n, len(nz) + 1), order="F")
                M[:, 0] = 0.5 * (lbv + ubv)
                M[nz, np.arange(1, len(nz) + 1)] = vec[nz]
                self._V = M.reshape(self.height, self.width, self.numChannel, -1, order="F")
        return self._V

    @property
    def C(self):
        if self._C is None and self._lazy is not None:
            self._C, self.d = self._lazy[0].get_constraints(self._lazy[1])
        return self._C

    def affineMap(self, scale=None, offset=None, ctx=None):
        """ImageStar.affineMap (ImageStar.m:431-460): every slice of V times ``scale`` (a scalar or one factor
        per channel), ``offset`` (scalar, per channel or a whole image) added to the centre.  The scaling runs on
        the GPU as a per-channel affine layer; an offset image, which has no per-channel form, is added to the
        centre slice on the host."""
        C = self.numChannel
        sc = np.ones(C)
        if scale is not None and np.size(scale):
            a = np.asarray(scale, dtype=np.float64)
            if a.size != 1 and (a.ndim < 3 or a.shape[2] != C or a.size != C):
                raise ValueError("Inconsistent number of channels between scale array and the ImageStar")
            sc = np.full(C, float(a.reshape(-1)[0])) if a.size == 1 else a.reshape(-1)
        off = np.zeros(C)
        off_image = None
        if offset is not None and np.size(offset):
            o = np.asarray(offset, dtype=np.float64)
            if o.size == 1:
                off = np.full(C, float(o.reshape(-1)[0]))
            elif o.size == C and (o.ndim < 3 or o.shape[:2] == (1, 1)):
                off = o.reshape(-1)
            else:
                off_image = o.reshape(self.height, self.width, C)
        layer = {"type": "bn", "mean": np.zeros(C), "var": np.ones(C), "scale": sc, "offset": off, "eps": 0.0}
        newV = (ctx or default_context()).layer_apply(layer, self.V)
        if off_image is not None:
            newV[..., 0] = newV[..., 0] + off_image
        return ImageStar(newV, self.C, self.d, self.pred_lb, self.pred_ub)

    def toStar(self):
        """ImageStar.m:569-592."""
        n = self.height * self.width * self.numChannel
        S = Star(self.V.reshape(n, -1, order="F"), self.C, self.d, self.pred_lb, self.pred_ub)
        return S

    def estimateRanges(self, ctx=None):
        """ImageStar.estimateRanges (ImageStar.m:836-885); returns images lb, ub."""
        lb, ub = self.toStar().estimateRanges(ctx)
        shp = (self.height, self.width, self.numChannel)
        return lb.reshape(shp, order="F"), ub.reshape(shp, order="F")

    def evaluate(self, pred_val):
        """ImageStar.evaluate (ImageStar.m:396-425): the image at a value of the predicate vector."""
        pred_val = np.asarray(pred_val, dtype=np.float64).reshape(-1)
        if pred_val.size != self.numPred:
            raise ValueError("Inconsistency between the size of the predicate vector and the number of predicates in the imagestar")
        if self._V is None and self.im_lb is not None:
            n = self.height * self.width * self.numChannel
            lbv, ubv = self.im_lb.reshape(n, order="F"), self.im_ub.reshape(n, order="F")
            x = 0.5 * (lbv + ubv)
            vec = 0.5 * (ubv - lbv)
            nz = np.nonzero(vec != 0)[0] if n > 1 else np.arange(1)
            x[nz] += vec[nz] * pred_val
            return x.reshape(self.height, self.width, self.numChannel, order="F")
        return self.V[..., 0] + self.V[..., 1:] @ pred_val

    def sample(self, N, rng=None):
        """ImageStar.sample (ImageStar.m:369-394): predicate vectors sampled from the star
        (0 | I, C, d, pred_lb, pred_ub) by Star.sample, each evaluated to an image.  Returns a list."""
        if N < 1:
            raise ValueError("Invalid number of samples")
        rng = rng or np.random.default_rng()
        P = self.numPred
        C = self.C
        if not np.size(C) or not np.any(C):                  # predicate box only: no rejection needed
            A = (self.pred_ub - self.pred_lb)[:, None] * rng.random((P, 2 * N)) + self.pred_lb[:, None]
            A = A[:, :N]
        else:
            S = Star(np.hstack([np.zeros((P, 1)), np.eye(P)]), C, self.d, self.pred_lb, self.pred_ub)
            A = S.sample(N, rng)
        return [self.evaluate(A[:, i]) for i in range(A.shape[1])]

    def _query(self):
        if self._V is None and self.im_lb is not None and self._lazy is None:
            return {"lb": self.im_lb, "ub": self.im_ub}
        return {"V": self.V, "C": self.C, "d": self.d, "pl": self.pred_lb, "pu": self.pred_ub}


class Star:
    """Star.m:13-24.  ``Star(lb, ub)`` (Star.m:220-237) or ``Star(V, C, d, pred_lb, pred_ub)``
    (Star.m:151-191)."""

    def __init__(self, *args):
        if len(args) == 2:
            lb = np.asarray(args[0], dtype=np.float64).ravel()
            ub = np.asarray(args[1], dtype=np.float64).ravel()
            if lb.size != ub.size:
                raise ValueError("Inconsistent dimensions between lb and ub")
            I = ImageStar(lb.reshape(-1, 1, 1), ub.reshape(-1, 1, 1))
            self.V = I.V.reshape(lb.size, -1, order="F")
            self.C, self.d = I.C, I.d
            self.predicate_lb, self.predicate_ub = I.pred_lb, I.pred_ub
            self.state_lb, self.state_ub = lb, ub
        elif len(args) in (3, 5):
            V = np.asfortranarray(np.atleast_2d(np.asarray(args[0], dtype=np.float64)))
            Cm = np.atleast_2d(np.asarray(args[1], dtype=np.float64))
            d = np.asarray(args[2], dtype=np.float64).ravel()
            if Cm.size and V.shape[1] != Cm.shape[1] + 1:
                raise ValueError("Inconsistency between basic matrix and constraint matrix")
            if Cm.size and Cm.shape[0] != d.size:
                raise ValueError("Inconsistency between constraint matrix and constraint vector")
            self.V, self.C, self.d = V, Cm, d
            if len(args) == 5:
                self.predicate_lb = np.asarray(args[3], dtype=np.float64).ravel()
                self.predicate_ub = np.asarray(args[4], dtype=np.float64).ravel()
                if self.predicate_lb.size != V.shape[1] - 1 or self.predicate_ub.size != V.shape[1] - 1:
                    raise ValueError("Inconsistency between number of predicate variables and predicate lower- or upper-bounds vector")
            else:
                self.predicate_lb = np.zeros(0)
                self.predicate_ub = np.zeros(0)
            self.state_lb = self.state_ub = None
        else:
            raise ValueError("Invalid number of input arguments (should be 2, 3 or 5)")
        self.dim = self.V.shape[0]
        self.nVar = self.V.shape[1] - 1

    def toImageStar(self, height, width, numChannel):
        """Star.m:1398-1418."""
        if self.dim != height * width * numChannel:
            raise ValueError("Inconsistent dimension in the ImageStar and the original Star set")
        pl, pu = self._pred_bounds()
        return ImageStar(self.V.reshape(height, width, numChannel, -1, order="F"), self.C, self.d, pl, pu)

    def _pred_bounds(self):
        if self.predicate_lb.size == 0 and self.nVar > 0:      # Star.m:1091-1096
            return -np.ones(self.nVar), np.ones(self.nVar)
        return self.predicate_lb, self.predicate_ub

    def estimateRanges(self, ctx=None):
        """Star.estimateRanges, Star.m:1078-1106 (on the GPU)."""
        ctx = ctx or default_context()
        pl, pu = self._pred_bounds()
        return ctx.estimate_ranges(self.V, pl, pu)

    def affineMap(self, W, b=None):
        """Star.affineMap, Star.m:313-343 (on the GPU as a one-layer network)."""
        W = np.atleast_2d(np.asarray(W, dtype=np.float64))
        if W.shape[1] != self.dim:
            raise ValueError("Inconsistency between the affine mapping matrix and dimension of the star set")
        b = np.zeros(W.shape[0]) if b is None else np.asarray(b, dtype=np.float64).ravel()
        if b.size != W.shape[0]:
            raise ValueError("Inconsistency between the mapping vec and mapping matrix")
        out = default_context().layer_apply({"type": "fc", "W": W, "b": b}, self.V.reshape(self.dim, 1, 1, -1, order="F"))
        return Star(out.reshape(W.shape[0], -1, order="F"), self.C, self.d, self.predicate_lb, self.predicate_ub)

    def intersectHalfSpace(self, H, g):
        """Star.intersectHalfSpace, Star.m:555-589; returns None when empty."""
        H = np.atleast_2d(np.asarray(H, dtype=np.float64))
        g = np.asarray(g, dtype=np.float64).reshape(-1)
        if H.shape[0] != g.size:
            raise ValueError("Inconsistent dimension between Halfspace matrix and halfspace vector")
        if H.shape[1] != self.dim:
            raise ValueError("Inconsistent dimension between halfspace and star set")
        C1 = H @ self.V[:, 1:]
        d1 = g - H @ self.V[:, 0]
        Cn = np.vstack([self.C, C1]) if np.size(self.C) else C1
        dn = np.concatenate([self.d, d1]) if np.size(self.C) else d1
        S = Star(self.V, Cn, dn, self.predicate_lb, self.predicate_ub)
        return None if S.isEmptySet() else S

    def isEmptySet(self):
        """Star.isEmptySet, Star.m:1216-1232."""
        return _lp_is_empty(sp.csr_matrix(self.C), self.d, self.predicate_lb, self.predicate_ub)

    def contains(self, x):
        """Star.contains (Star.m:1189-1213): is there a predicate vector with x = c + V alpha, C alpha <= d,
        pred_lb <= alpha <= pred_ub (a feasibility LP with equality rows)."""
        x = np.asarray(x, dtype=np.float64).reshape(-1)
        if x.size != self.dim:
            raise ValueError("Dimension mismatch")
        pl, pu = self._pred_bounds()
        A = self.C if np.size(self.C) else None
        res = linprog(np.zeros(self.nVar), A_ub=A, b_ub=self.d if A is not None else None, A_eq=self.V[:, 1:],
                      b_eq=x - self.V[:, 0], bounds=list(zip(pl, pu)), method="highs")
        return res.status == 0

    def sample(self, N, rng=None):
        """Star.sample (Star.m:278-308): 2N points uniform in the set's bounding box, those inside the set
        kept, at most N returned (columns).  ``rng``: a numpy Generator standing in for MATLAB's rand."""
        if N < 1:
            raise ValueError("Invalid number of samples")
        rng = rng or np.random.default_rng()
        lb, ub = self.estimateRanges()
        X = (ub - lb)[:, None] * rng.random((self.dim, 2 * N)) + lb[:, None]
        pl, pu = self._pred_bounds()
        box_only = not np.size(self.C) or not np.any(self.C)
        diag = self.nVar == self.dim and np.count_nonzero(self.V[:, 1:] - np.diag(np.diag(self.V[:, 1:]))) == 0
        if box_only and diag and np.all(np.asarray(self.d) >= 0):
            return X[:, :N]                 # a box: every point of its bounding box is a point of the set
        keep = [i for i in range(2 * N) if self.contains(X[:, i])]
        return X[:, keep[:N]]

    def _query(self):
        pl, pu = self._pred_bounds()
        return {"V": self.V.reshape(self.dim, 1, 1, -1, order="F"), "C": self.C, "d": self.d, "pl": pl, "pu": pu}


class HalfSpace:
    """HalfSpace.m:14-32: the set G x <= g."""

    def __init__(self, G, g):
        G = np.atleast_2d(np.asarray(G, dtype=np.float64))
        g = np.asarray(g, dtype=np.float64).reshape(-1)
        if G.shape[0] != g.size:
            raise ValueError("Inconsistent dimension between half-space matrix and half-space vector")
        self.G, self.g, self.dim = G, g, G.shape[1]

    def contains(self, x):
        """HalfSpace.contains (HalfSpace.m:35-55): no row of g - G x is negative."""
        x = np.asarray(x, dtype=np.float64).reshape(-1)
        if x.size != self.dim:
            raise ValueError("Inconsistent dimension between the vector x and the half-space object")
        return not np.any(self.g - self.G @ x < 0)


_LP_POOL = None


def _lp_map(fn, items):
    """Independent host LPs on all host cores: HiGHS releases the interpreter lock while it solves, so a thread
    pool scales (the reference spreads its LP work over ``numCores`` workers with ``parfor``, NN.m:651-667).
    Results come back in the order of ``items``."""
    global _LP_POOL
    items = list(items)
    if len(items) < 2:
        return [fn(x) for x in items]
    if _LP_POOL is None:
        _LP_POOL = ThreadPoolExecutor(max_workers=max(1, os.cpu_count() or 1), thread_name_prefix="nnvb-lp")
    return list(_LP_POOL.map(fn, items))


def _lp_is_empty(Cs, d, pl, pu):
    """lpsolver(f=0, C, d, [], [], pl, pu, 'linprog', 'emptySet') (lpsolver.m): the
    box-only closed form (:34-49), else a feasibility LP.  Exit mapping of
    Star.m:1224-1230: feasible -> not empty, infeasible -> empty, else error."""
    d = np.asarray(d, dtype=np.float64).ravel()
    P = Cs.shape[1]
    if Cs.nnz == 0 and pl.size and np.all(np.isfinite(pl)) and np.all(np.isfinite(pu)) and np.all(d >= 0):
        return False
    bounds = list(zip(pl, pu)) if pl.size else [(None, None)] * P
    res = linprog(np.zeros(P), A_ub=Cs, b_ub=d, bounds=bounds, method="highs")
    if res.status == 0:
        return False
    if res.status == 2:
        return True
    raise RuntimeError("Error, exitflag = %d (%s)" % (res.status, res.message))


LP_FEAS_TOL = 1e-7          # the primal feasibility tolerance the feasibility form of the same test works to


def _row_meets_star(S, G, g):
    """Is the intersection of the star S with the halfspace G x <= g (one row) non-empty?  The reference asks
    through a feasibility LP with zero objective (Star.intersectHalfSpace + isEmptySet, Star.m:555-589,
    1216-1232); the same question as an optimisation — is the minimum of G x over the star at most g — has the
    same answer and takes the simplex a sixth of the iterations on the output sets of the benchmark networks
    (about 100 instead of 900: the objective steers it, where the zero-objective form wanders through phase 1)."""
    G = np.asarray(G, dtype=np.float64).reshape(-1)
    g0 = float(np.ravel(g)[0])
    f = G @ S.V[:, 1:]
    c0 = float(G @ S.V[:, 0])
    pl, pu = S._pred_bounds()
    Cs = sp.csr_matrix(S.C) if np.size(S.C) else sp.csr_matrix((0, S.nVar))
    box_only = (Cs.shape[0] == 0 or Cs.nnz == 0) and np.all(np.isfinite(pl)) and np.all(np.isfinite(pu)) \
        and np.all(np.asarray(S.d) >= 0)
    lo = _lp_extreme(f, c0, Cs, S.d, list(zip(pl, pu)), box_only, pl, pu, False)
    return lo <= g0 + LP_FEAS_TOL * max(1.0, abs(g0))


def _lp_extreme(f, c0, Cs, d, bounds, box_only, pl, pu, maximize):
    """Star.getMax / Star.getMin (Star.m:859-895, :745-781) through lpsolver.m: all-zero objective -> the
    centre value; all-zero constraint matrix -> the closed-form box optimum (lpsolver.m:34-49); else an LP."""
    if not np.any(f):
        return c0
    sgn = -1.0 if maximize else 1.0
    if box_only:
        ff = sgn * f
        return sgn * float(np.sum(np.minimum(ff * pl, ff * pu))) + c0
    res = linprog(sgn * f, A_ub=Cs, b_ub=d, bounds=bounds, method="highs")
    if res.status != 0:
        raise RuntimeError("Cannot find an optimal solution, exitflag = %d (%s)" % (res.status, res.message))
    return sgn * res.fun + c0


def lp_bounds_hook(batch, relu_layer):
    """The LP half of PosLin.reach_star_approx2 (PosLin.m:813-846) for one ReLU layer of a running reach: for
    every query, getMaxs over the neurons the estimated ranges call crossing (in ascending index order), then
    getMins over those whose maximum is positive; the bounds go back to the engine, which re-classifies.  The
    LPs run on the host (HiGHS standing in for linprog / glpk), as they do in the reference."""
    for q in range(batch.nq):
        idx, l_est, u_est = batch.get_crossing(q, relu_layer)
        k = len(idx)
        if k == 0:
            continue
        P, _ = batch.out_dims(q)
        G, c = batch.get_crossing_rows(q, relu_layer, k, P)
        Cm, d = batch.get_constraints_before(q, relu_layer, P)
        pl, pu = batch.get_pred_bounds(q)
        Cs = sp.csr_matrix(Cm)
        box_only = (Cs.shape[0] == 0 or Cs.nnz == 0) and np.all(np.isfinite(pl)) and np.all(np.isfinite(pu)) \
            and np.all(d >= 0)
        bounds = list(zip(pl, pu))
        xmax = np.array(_lp_map(lambda t: _lp_extreme(G[t], c[t], Cs, d, bounds, box_only, pl, pu, True), range(k)))
        xmin = np.array(l_est, dtype=np.float64, copy=True)       # only read where xmax > 0
        pos = np.nonzero(xmax > 0)[0]
        xmin[pos] = _lp_map(lambda t: _lp_extreme(G[t], c[t], Cs, d, bounds, box_only, pl, pu, False), pos)
        xmin = np.minimum(xmin, xmax)
        batch.tighten_crossing(q, relu_layer, xmin, xmax)


def _matlab_round(x):
    return int(np.floor(x + 0.5))


def relax_select(method, relax_factor, l_est, u_est, rng=None):
    """Positions (within the crossing list) of the n1 = round((1 - relaxFactor) * count) neurons whose ranges are
    optimised (PosLin.m:929-936, 1044-1052, 1483-1491, 1599-1607; MATLAB's sort is stable and its round takes
    halves away from zero)."""
    l_est, u_est = np.asarray(l_est, dtype=np.float64), np.asarray(u_est, dtype=np.float64)
    k = len(l_est)
    n1 = _matlab_round((1.0 - relax_factor) * k)
    if method == "relax-star-area":
        return np.argsort(-(0.5 * np.abs(u_est) * np.abs(l_est)), kind="stable")[:n1]
    if method == "relax-star-range":
        return np.argsort(-(u_est - l_est), kind="stable")[:n1]
    if method == "relax-star-static":
        return np.arange(n1)
    if method == "relax-star-random":
        return (rng or np.random.default_rng(0)).permutation(k)[:n1]
    raise ValueError(method)


def relax_bounds_hook(method, relax_factor, rng=None):
    """Bounds hook of the 'relax-star-*' methods with relaxFactor < 1 (PosLin.reach_relaxed_star_area / _range /
    _static / _random, PosLin.m:986-1105, 863-984, 1541-1646, 1425-1539): of the neurons the estimated ranges call
    crossing, n1 = round((1 - relaxFactor) * count) get LP-optimised ranges (largest triangle area / largest range /
    first in index order / random choice), the others keep the estimated bounds.  Returns the hook function.
    The engine appends the new predicates in ascending neuron order; the reference appends the neurons without
    optimised ranges first (map9 = [map22; map8]): the same set with its new predicate variables permuted."""
    rng = rng or np.random.default_rng(0)

    def hook(batch, relu_layer):
        for q in range(batch.nq):
            idx, l_est, u_est = batch.get_crossing(q, relu_layer)
            k = len(idx)
            if k == 0:
                continue
            sel = relax_select(method, relax_factor, l_est, u_est, rng)
            n1 = len(sel)
            xmin = np.array(l_est, dtype=np.float64, copy=True)
            xmax = np.array(u_est, dtype=np.float64, copy=True)
            if n1 > 0:
                P, _ = batch.out_dims(q)
                G, c = batch.get_crossing_rows(q, relu_layer, k, P)
                Cm, d = batch.get_constraints_before(q, relu_layer, P)
                pl, pu = batch.get_pred_bounds(q)
                Cs = sp.csr_matrix(Cm)
                box_only = (Cs.shape[0] == 0 or Cs.nnz == 0) and np.all(np.isfinite(pl)) and np.all(np.isfinite(pu)) \
                    and np.all(d >= 0)
                bounds = list(zip(pl, pu))
                sel = np.asarray(sel, dtype=np.int64)
                xmax[sel] = _lp_map(lambda t: _lp_extreme(G[t], c[t], Cs, d, bounds, box_only, pl, pu, True), sel)
                pos = sel[xmax[sel] > 0]
                xmin[pos] = _lp_map(lambda t: _lp_extreme(G[t], c[t], Cs, d, bounds, box_only, pl, pu, False), pos)
                xmin[sel] = np.minimum(xmin[sel], xmax[sel])
            batch.tighten_crossing(q, relu_layer, xmin, xmax)

    return hook


_RELAX_WITH_LP = ("relax-star-area", "relax-star-range", "relax-star-static", "relax-star-random")


# ------------------------------------------------------------------------- layers


class _Layer:
    Name = ""

    def _desc(self):
        raise NotImplementedError

    def reach(self, in_set, method="approx-star", option=None, relaxFactor=0, dis_opt=None, lp_solver="linprog"):
        """The reference's 6-argument layer contract; one set or a list of sets."""
        sets = in_set if isinstance(in_set, (list, tuple)) else [in_set]
        shape = _set_shape(sets[0])
        net = NN([self], input_shape=shape)
        out = [net.reach(s, {"reachMethod": method, "relaxFactor": relaxFactor}) for s in sets]
        return out if isinstance(in_set, (list, tuple)) else out[0]


class Conv2DLayer(_Layer):
    """Conv2DLayer.m:84-144 — Weights[kh,kw,Cin,Cout], Bias[1,1,Cout], PaddingSize [t b l r]."""

    def __init__(self, Weights, Bias, PaddingSize=(0, 0, 0, 0), Stride=(1, 1), DilationFactor=(1, 1), Name="conv2d"):
        W = np.asarray(Weights, dtype=np.float64)
        if W.ndim == 2:
            W = W[:, :, None, None]
        if W.ndim == 3:
            W = W[:, :, :, None]
        b = np.asarray(Bias, dtype=np.float64).ravel()
        if b.size != W.shape[3]:
            raise ValueError("Inconsistency between filter weights and filter biases")
        if len(PaddingSize) != 4:
            raise ValueError("Invalid padding size")
        self.Weights, self.Bias = W, b
        self.PaddingSize, self.Stride, self.DilationFactor = tuple(PaddingSize), tuple(Stride), tuple(DilationFactor)
        self.NumChannels, self.NumFilters, self.FilterSize = W.shape[2], W.shape[3], W.shape[:2]
        self.Name = Name

    def _desc(self):
        return {"type": "conv2d", "W": self.Weights, "b": self.Bias, "pad": self.PaddingSize,
                "stride": self.Stride, "dilation": self.DilationFactor}


class FullyConnectedLayer(_Layer):
    """FullyConnectedLayer.m:56-66 — Weights[Out,In], Bias[Out,1]."""

    def __init__(self, Weights, Bias, Name="fc"):
        W = np.atleast_2d(np.asarray(Weights, dtype=np.float64))
        b = np.asarray(Bias, dtype=np.float64).ravel()
        if b.size != W.shape[0]:
            raise ValueError("Inconsistent dimension between the weight matrix and bias vector")
        self.Weights, self.Bias = W, b
        self.OutputSize, self.InputSize = W.shape
        self.Name = Name

    def _desc(self):
        return {"type": "fc", "W": self.Weights, "b": self.Bias}


class BatchNormalizationLayer(_Layer):
    """BatchNormalizationLayer.m:14,72-77 — name/value constructor."""

    def __init__(self, **kw):
        self.Name = kw.get("Name", "bn")
        self.TrainedMean = np.asarray(kw["TrainedMean"], dtype=np.float64).ravel()
        self.TrainedVariance = np.asarray(kw["TrainedVariance"], dtype=np.float64).ravel()
        self.Scale = np.asarray(kw["Scale"], dtype=np.float64).ravel()
        self.Offset = np.asarray(kw["Offset"], dtype=np.float64).ravel()
        self.Epsilon = float(kw.get("Epsilon", 1e-5))
        self.NumChannels = int(kw.get("NumChannels", self.TrainedMean.size))

    def _desc(self):
        return {"type": "bn", "mean": self.TrainedMean, "var": self.TrainedVariance, "scale": self.Scale,
                "offset": self.Offset, "eps": self.Epsilon}


class AveragePooling2DLayer(_Layer):
    """AveragePooling2DLayer.m:109-131 — PoolSize, Stride, PaddingSize.

    ``Divisor`` says how a window that reaches into the padding is averaged: "inside" divides by the
    window entries inside the image, as vl_nnpool does for the reference's host arrays
    (AveragePooling2DLayer.m:247); "window" divides by PoolSize(1)*PoolSize(2), as avgpool does for its
    gpuArray inputs (:242-245) and as compute_averageMap (:316-393) does."""

    def __init__(self, PoolSize=(2, 2), Stride=(1, 1), PaddingSize=(0, 0, 0, 0), Name="average_pooling_2d",
                 Divisor="inside"):
        if len(PoolSize) != 2 or len(Stride) != 2 or len(PaddingSize) != 4:
            raise ValueError("Invalid pooling parameters")
        if Divisor not in ("inside", "window"):
            raise ValueError("Divisor must be 'inside' or 'window'")
        self.PoolSize, self.Stride, self.PaddingSize, self.Name = tuple(PoolSize), tuple(Stride), tuple(PaddingSize), Name
        self.Divisor = Divisor

    def _desc(self):
        return {"type": "avgpool", "pool": self.PoolSize, "stride": self.Stride, "pad": self.PaddingSize,
                "divisor": self.Divisor}


class ReluLayer(_Layer):
    """ReluLayer.m — PosLin applied to every neuron."""

    def __init__(self, Name="relu"):
        self.Name = Name

    def _desc(self):
        return {"type": "relu"}


class LayerNormalizationLayer(_Layer):
    """MATLAB's layerNormalizationLayer on a vector of ``NumChannels`` entries or a sequence [NumChannels, T, 1]: every
    position is normalised over its channels, (x - mean) / sqrt(var + Epsilon) * Scale + Offset.  For
    ``NN.evaluate`` and ``NN.falsify``; the layer has no approx-star reach here."""

    def __init__(self, NumChannels, Scale=None, Offset=None, Epsilon=1e-5, Name="layernorm"):
        self.NumChannels, self.Epsilon, self.Name = int(NumChannels), float(Epsilon), Name
        if self.NumChannels < 1:
            raise ValueError("Invalid number of channels")
        if not (np.isfinite(self.Epsilon) and self.Epsilon >= 0):
            raise ValueError("Epsilon must be finite and not negative")
        self.Scale = None if Scale is None else np.asarray(Scale, dtype=np.float64).ravel()
        self.Offset = None if Offset is None else np.asarray(Offset, dtype=np.float64).ravel()
        for a in (self.Scale, self.Offset):
            if a is not None and a.size != self.NumChannels:
                raise ValueError("Inconsistency between the number of channels and the size of Scale or Offset")

    def _desc(self):
        return {"type": "layernorm", "channels": self.NumChannels, "scale": self.Scale, "offset": self.Offset,
                "eps": self.Epsilon}


class AttentionLayer(_Layer):
    """MATLAB's attentionLayer with the keys and values of a fixed encoder output: the input, a sequence
    [NumHeads * channels, T, 1] or one position as a vector, holds the queries; ``Keys`` and ``Values`` are
    [channels, state heads, states] (or [channels * state heads, states] with ``NumStateHeads``).  Query head h
    reads state head h // (NumHeads / state heads); ``Scale`` defaults to 1/sqrt(channels).  For ``NN.evaluate``
    and ``NN.falsify``; the layer has no approx-star reach here."""

    def __init__(self, NumHeads, Keys, Values, NumStateHeads=None, Scale=None, Name="attention"):
        K, V = np.asarray(Keys, dtype=np.float64), np.asarray(Values, dtype=np.float64)
        self.NumHeads, self.Name = int(NumHeads), Name
        hk = int(NumStateHeads) if NumStateHeads is not None else (K.shape[1] if K.ndim == 3 else self.NumHeads)
        if K.shape != V.shape or K.ndim not in (2, 3):
            raise ValueError("Keys and Values must be [channels, heads, states] of one shape")
        if hk < 1 or self.NumHeads < 1 or self.NumHeads % hk:
            raise ValueError("%d heads cannot share %d state heads evenly" % (self.NumHeads, hk))
        if K.ndim == 2:
            if K.shape[0] % hk:
                raise ValueError("Inconsistency between the rows of Keys and the number of heads")
            K, V = (a.reshape(K.shape[0] // hk, hk, -1, order="F") for a in (K, V))
        if K.shape[1] != hk or K.size == 0 or K.shape[0] > 256:
            raise ValueError("Keys must have %d heads of 1..256 channels and at least one state" % hk)
        if Scale is not None and not (np.isfinite(Scale) and Scale > 0):
            raise ValueError("Scale must be finite and positive")
        self.Keys, self.Values, self.Scale = K, V, Scale

    def _desc(self):
        return {"type": "attention", "heads": self.NumHeads, "keys": self.Keys, "values": self.Values, "scale": self.Scale}


class ImageInputLayer(_Layer):
    """ImageInputLayer.m:14-46 (properties, constructor) and :121-168 (reach_star_single_input): the
    normalisation of the input set.  It is an affine map of the input image with a positive scale, applied to
    the set on the host before upload (generators scaled, offsets added to the centre; for a set given by
    bounds, the bounds are mapped).  Must be the first layer."""

    def __init__(self, InputSize=None, Normalization="none", Mean=None, StandardDeviation=None, Min=None, Max=None,
                 Name="ImageInputLayer"):
        if Normalization not in ("none", "zerocenter", "zscore", "rescale-zero-one", "rescale-symmetric"):
            raise ValueError("The normalization method is not supported yet.")
        self.InputSize, self.Normalization, self.Name = InputSize, Normalization, Name
        self.Mean, self.StandardDeviation, self.Min, self.Max = Mean, StandardDeviation, Min, Max

    @staticmethod
    def _arr(x):
        a = np.asarray(x, dtype=np.float64)
        return a.reshape(a.shape + (1,) * (3 - a.ndim)) if a.ndim < 3 else a

    def _steps(self):
        """[(kind, value)] in the reference's order: 'add' touches the centre only, 'mul' / 'div' every slice."""
        n = self.Normalization
        if n == "none":
            return []
        if n == "zerocenter":
            return [("add", -self._arr(self.Mean))]
        if n == "zscore":
            std = np.asarray(self.StandardDeviation, dtype=np.float64).reshape(1, 1, -1)
            return [("add", -self._arr(self.Mean)), ("div", std)]
        have = self.Min is not None and self.Max is not None
        if n == "rescale-zero-one":
            return [("add", -self._arr(self.Min)), ("mul", 1.0 / (float(self.Max) - float(self.Min)))] if have \
                else [("mul", 1 / 255)]
        if have:
            return [("add", -self._arr(self.Min)), ("mul", 2.0 / (float(self.Max) - float(self.Min))), ("add", -1.0)]
        return [("mul", 2 / 255), ("add", -1.0)]

    def apply_image(self, x):
        """ImageInputLayer.evaluate (ImageInputLayer.m:84-114): the normalised copy of a concrete image."""
        x = np.asarray(x, dtype=np.float64)
        for kind, v in self._steps():
            x = x + v if kind == "add" else (x * v if kind == "mul" else x / v)
        return x

    def apply(self, s):
        """The normalised copy of an input ImageStar."""
        if not isinstance(s, ImageStar):
            raise TypeError("Input is not an ImageStar")
        steps = self._steps()
        if not steps:
            return s
        if s.im_lb is not None and s._V is None:          # given by bounds: map the bounds (the scale is positive)
            lb, ub = s.im_lb, s.im_ub
            for kind, v in steps:
                if kind == "add":
                    lb, ub = lb + v, ub + v
                elif kind == "mul":
                    lb, ub = lb * v, ub * v
                else:
                    lb, ub = lb / v, ub / v
            return ImageStar(lb, ub)
        V = np.array(s.V, dtype=np.float64, copy=True)
        for kind, v in steps:
            if kind == "add":
                V[..., 0] = V[..., 0] + v
            elif kind == "mul":
                V = V * v
            else:
                V = V / v[..., None]
        return ImageStar(V, s.C, s.d, s.pred_lb, s.pred_ub)

    def _desc(self):
        return {"type": "imageinput"}


class FlattenLayer(_Layer):
    """FlattenLayer.m:105-164 — reshape of an H x W x C image into a vector.  The plain MATLAB type keeps the
    column-major order (nothing to do on the device: FC layers consume that order); the Keras C-style and
    ONNX types permute first, which is folded into the columns of the FullyConnectedLayer that follows."""

    TYPES = ("nnet.cnn.layer.FlattenLayer", "nnet.keras.layer.FlattenCStyleLayer", "nnet.onnx.layer.FlattenLayer",
             "nnet.onnx.layer.FlattenInto2dLayer", "nnet.onnx.layer.Flatten3dInto2dLayer")

    def __init__(self, Name="flatten", Type="nnet.cnn.layer.FlattenLayer"):
        if Type not in self.TYPES:
            raise ValueError("Unknown type of flatten layer")
        self.Name, self.Type = Name, Type

    def source_index(self, shape):
        """Column-major position in the H x W x C image of every entry of the flattened vector."""
        h, w, c = shape
        idx = np.arange(h * w * c).reshape((h, w, c), order="F")
        if self.Type == "nnet.cnn.layer.FlattenLayer":
            return idx.reshape(-1, order="F")
        if self.Type == "nnet.keras.layer.FlattenCStyleLayer":
            return np.transpose(idx, (2, 1, 0)).reshape(-1, order="F")
        return np.transpose(idx, (1, 0, 2)).reshape(-1, order="F")

    def _desc(self):
        return {"type": "flatten", "kind": self.Type}


def _set_shape(s):
    if isinstance(s, ImageStar):
        return (s.height, s.width, s.numChannel)
    if isinstance(s, Star):
        return (s.dim, 1, 1)
    raise TypeError('Wrong input set type. Input set must be of type "Star" or "ImageStar"')


_LP_FREE_RELAX = ("relax-star-range", "relax-star-area", "relax-star-bound", "relax-star-ub",
                  "relax-star-random", "relax-star-static")


def _validate_reach_options(opts):
    """The part of NN.validate_reach_options (NN.m:1203-1233) this engine honours:
    'approx-star' with bounds='estimate' (default: the LP-free ranges of Star.estimateRanges, which is also any
    'relax-star-*' method at relaxFactor = 1) or bounds='lp' (PosLin.reach_star_approx2 as the reference runs
    it for 'approx-star': estimated ranges pre-select, host LPs give the bounds of the relaxation)."""
    opts = dict(opts or {})
    method = opts.get("reachMethod", "approx-star")
    rf = opts.get("relaxFactor", 1 if method in _LP_FREE_RELAX else 0)
    if method == "approx-star":
        if opts.get("bounds", "estimate") not in ("estimate", "lp"):
            raise ValueError("bounds must be 'estimate' (LP-free ranges) or 'lp' (the reference's LP-tightened ranges)")
    elif method in _LP_FREE_RELAX:
        if rf != 1 and method not in _RELAX_WITH_LP:
            raise NotImplementedError("%s is implemented for relaxFactor = 1 only (no LP); relaxFactor < 1 is "
                                      "available for %s" % (method, ", ".join(_RELAX_WITH_LP)))
    else:
        raise NotImplementedError("reachMethod %r is outside this engine (approx-star / relax-star-* only)" % (method,))
    if not (0 <= rf <= 1):
        raise ValueError("Invalid relaxFactor. The value of relax factor must be between 0 and 1")
    opts["reachMethod"], opts["relaxFactor"] = method, rf
    return opts


# ---------------------------------------------------------------------------- NN


class NN:
    """NN.m — network container, reach driver and robustness API.

    ``layers`` is a list of layer objects (or neutral layer dicts);
    ``input_shape`` may be given up front, else it is taken from the first set.
    """

    def __init__(self, layers, input_shape=None, Name="nn", ctx=None):
        self.Layers = list(layers)
        self.numLayers = len(self.Layers)
        self.Name = Name
        self.ctx = ctx
        self._nets = {}
        self.reachTime = []
        self.reachStats = []
        self.reachMethod = "approx-star"
        self.relaxFactor = 0
        self.lp_solver = "linprog"
        self.input_shape = tuple(input_shape) if input_shape is not None else None
        self.exactReach = False          # approx methods never promote unknown -> not robust (NN.m:539-543)

    def _layer_dicts(self, shape=None):
        """Neutral layer dicts for the device.  An ImageInputLayer (first layer only) is applied to the input
        sets on the host; a FlattenLayer moves no data: the plain type is the device's own order, the
        permuting types are folded into the weight columns of the FullyConnectedLayer right behind them."""
        from .configs import out_shape
        out = []
        pending = None                       # permutation of a flatten layer waiting for its FC layer
        for i, l in enumerate(self.Layers):
            d = l if isinstance(l, dict) else l._desc()
            if d["type"] == "imageinput":
                if i != 0:
                    raise NotImplementedError("an ImageInputLayer is supported as the first layer only")
                continue
            if d["type"] == "flatten":
                if d["kind"] != "nnet.cnn.layer.FlattenLayer":
                    if shape is None:
                        raise ValueError("the input shape is needed to fold a permuting FlattenLayer")
                    pending = FlattenLayer(Type=d["kind"]).source_index(shape)
                continue
            if pending is not None:
                if d["type"] != "fc":
                    raise NotImplementedError("a permuting FlattenLayer must be followed by a FullyConnectedLayer")
                W = np.asarray(d["W"], dtype=np.float64)
                Wp = np.empty_like(W)
                Wp[:, pending] = W           # flattened entry k reads image entry pending[k]
                d = dict(d, W=np.asfortranarray(Wp))
                pending = None
            out.append(d)
            if shape is not None:
                shape = out_shape([d], shape)
        if pending is not None:
            raise NotImplementedError("a permuting FlattenLayer must be followed by a FullyConnectedLayer")
        return out

    def close(self):
        """Release the device copies of the weights (before the context they live in is closed)."""
        for n in self._nets.values():
            n.close()
        self._nets = {}

    def _network(self, shape):
        shape = tuple(int(x) for x in shape)
        if shape not in self._nets:
            self._nets[shape] = Network(self.ctx or default_context(), self._layer_dicts(shape), shape)
        return self._nets[shape]

    @property
    def OutputSize(self):
        for l in reversed(self.Layers):
            d = l if isinstance(l, dict) else l._desc()
            if d["type"] == "fc":
                return d["W"].shape[0]
        return 0

    # -- reach -----------------------------------------------------------------
    def reach_batch(self, inputSets, reachOptions=None, keep_constraints=False, keep_layer_bounds=False):
        """Push a list of input sets through the network together; returns the Batch
        (device-resident results).  Array-of-sets form of NN.reach."""
        _validate_reach_options(reachOptions)
        first = self.Layers[0] if self.Layers else None
        if isinstance(first, dict) and first.get("type") == "imageinput":
            first = ImageInputLayer(None, first.get("normalization", "none"), first.get("mean"), first.get("std"),
                                    first.get("min"), first.get("max"))
        if isinstance(first, ImageInputLayer):
            inputSets = [first.apply(s) for s in inputSets]      # ImageInputLayer.m:121-168, on the host
        shape = _set_shape(inputSets[0])
        for s in inputSets:
            if _set_shape(s) != shape:
                raise ValueError("all input sets of a batch must have the same shape")
        net = self._network(shape)
        b = Batch(net, [s._query() for s in inputSets])
        ro = dict(reachOptions or {})
        lp = ro.get("bounds", "estimate") == "lp"
        method, rf = ro.get("reachMethod", "approx-star"), ro.get("relaxFactor", None)
        relax_lp = method in _RELAX_WITH_LP and rf is not None and rf < 1
        t0 = time.perf_counter()
        try:
            b.upload()
            if relax_lp:                # a share of the crossing neurons gets LP bounds
                b.set_bounds_hook(relax_bounds_hook(method, rf))
                keep_constraints = True
            elif lp:                    # the LPs read the constraint system: records are kept
                b.set_bounds_hook(lp_bounds_hook)
                keep_constraints = True
            b.reach(keep_constraints=keep_constraints, keep_layer_bounds=keep_layer_bounds)
        except Exception:
            b.close()
            raise
        self.reachTime = [time.perf_counter() - t0]
        self.reachStats = b.relu_stats()
        return b

    def reach(self, inputSet, reachOptions=None):
        """NN.reach (NN.m:189-278): returns the output set (ImageStar for image
        input, Star for vector input).  V and C are fetched from the device when
        first read."""
        if not isinstance(inputSet, (Star, ImageStar)):
            raise TypeError('Wrong input set type. Input set must be of type "Star" or "ImageStar"')
        opts = _validate_reach_options(reachOptions)
        self.reachMethod, self.relaxFactor = opts["reachMethod"], opts["relaxFactor"]
        b = self.reach_batch([inputSet], opts, keep_constraints=True)
        return _result_set(b, 0, isinstance(inputSet, Star))

    # -- concrete evaluation and falsification -----------------------------------
    def evaluate(self, x):
        """NN.evaluate (NN.m:130-145) on the device; ``x`` is one input (image or vector) or a list of them.
        Returns the output vector(s), column-major flattened."""
        many = isinstance(x, (list, tuple))
        xs = [np.asarray(v, dtype=np.float64) for v in (x if many else [x])]
        first = self.Layers[0] if self.Layers else None
        if isinstance(first, ImageInputLayer):
            xs = [first.apply_image(v) for v in xs]
        shape = xs[0].shape if xs[0].ndim == 3 else ((xs[0].shape + (1,)) if xs[0].ndim == 2 else (xs[0].size, 1, 1))
        net = self._network(shape)
        X = np.stack([v.reshape(-1, order="F") for v in xs], axis=1)
        Y = net.evaluate(np.asfortranarray(X))
        return [Y[:, i] for i in range(Y.shape[1])] if many else Y[:, 0]

    def falsify(self, I, U, n_samples, rng=None):
        """NN.falsify (NN.m:930-988): sample ``n_samples`` inputs from the set, evaluate them (one batched
        forward pass on the device) and return those whose output lies in one of the halfspaces U."""
        Us = list(U) if isinstance(U, (list, tuple)) else [U]
        if not all(isinstance(h, HalfSpace) for h in Us):
            raise TypeError("Unsafe region (U) is not a HalfSpace.")
        if not isinstance(I, (ImageStar, Star)):
            raise TypeError("Input set (I) must be a ImageZono, ImageStar, Star, Zono or Box.")
        if n_samples < 1:
            raise ValueError("Invalid number of samples. n_samples > 0")
        pts = I.sample(n_samples, rng)
        if isinstance(I, Star):
            pts = [pts[:, i] for i in range(pts.shape[1])]
        if not pts:
            return []
        ys = self.evaluate(list(pts))
        return [p for p, y in zip(pts, ys) if any(h.contains(y) for h in Us)]

    def verify_safety(self, I, U, reachOptions=None, n_samples=0, rng=None):
        """NN.verify_safety (NN.m:827-927) for the over-approximating methods of this engine: 1 safe (every
        intersection of the reach set with U is empty), else falsification with ``n_samples`` inputs: 0 unsafe
        when one of them reaches U, 2 unknown otherwise (and when n_samples = 0).  Returns (result, counter_inputs)."""
        R = self.reach(I, reachOptions)
        Us = list(U) if isinstance(U, (list, tuple)) else [U]
        if verify_specification([R], Us) == 1:
            return 1, []
        if n_samples == 0:
            return 2, []
        counter = self.falsify(I, Us, n_samples, rng)
        return (0, counter) if counter else (2, [])

    def verify_sample_batch(self, inputSets, images, targets, reachOptions=None, n_samples=0, rng=None):
        """The harness the reference's examples wrap around verify_robustness
        (examples/Tutorial/SPIE/Classification2D/verifySample.m:1-32), for a list of sets: -1 the image itself is
        misclassified, 0 not robust — the upper- or lower-bound image of the set (and, with n_samples > 0, one
        of that many random points of an "unknown" set) is classified differently — else the verdict of
        verify_robustness (1 robust, 2 unknown).  All concrete evaluations run as one batched forward pass."""
        n = len(inputSets)
        res = np.full(n, 2, dtype=np.int64)
        pts = []
        for s, img in zip(inputSets, images):
            if s.im_lb is None:
                lb, ub = s.estimateRanges()
            else:
                lb, ub = s.im_lb, s.im_ub
            pts += [np.asarray(img, dtype=np.float64).reshape(lb.shape), ub, lb]
        ys = self.evaluate(pts)
        lab = np.array([int(np.argmax(y)) + 1 for y in ys]).reshape(n, 3)
        t = np.asarray(targets, dtype=np.int64)
        res[lab[:, 0] != t] = -1
        res[(lab[:, 0] == t) & ((lab[:, 1] != t) | (lab[:, 2] != t))] = 0
        todo = np.nonzero(res == 2)[0]
        if len(todo):
            res[todo] = self.verify_robustness_batch([inputSets[i] for i in todo], reachOptions, list(t[todo]))
        if n_samples > 0:
            for i in np.nonzero(res == 2)[0]:
                if self.falsify(inputSets[i], self.robustness_set(int(t[i]), "max"), n_samples, rng):
                    res[i] = 0
        return res

    # -- robustness ------------------------------------------------------------
    def robustness_set(self, target, class_type="max"):
        """NN.robustness_set (NN.m:1334-1368); ``target`` is 1-based like the reference."""
        outSize = self.OutputSize
        if outSize == 0:
            raise ValueError("Output size is set to 0, but it must be >= 1")
        if target > outSize or target < 1:
            raise ValueError("Target idx must be less than or equal to the output size of the NN.")
        G = np.delete(np.eye(outSize), target - 1, axis=0)
        if class_type == "max":
            G = -G
            G[:, target - 1] = 1.0
        elif class_type == "min":
            G[:, target - 1] = -1.0
        else:
            raise ValueError("class_type must be 'max' or 'min'")
        return [HalfSpace(G[i], 0.0) for i in range(G.shape[0])]

    def checkRobust(self, outputSet, target):
        """NN.checkRobust (NN.m:617-648)."""
        sets = outputSet if isinstance(outputSet, (list, tuple)) else [outputSet]
        R = [s if isinstance(s, Star) else s.toStar() for s in sets]
        if not isinstance(target, (HalfSpace, list, tuple)):
            if np.isscalar(target):
                target = self.robustness_set(int(target), "max")
            else:
                raise ValueError("Target must be a HalfSpace (unsafe/not robust region) or as a scalar determining the output label target.")
        return verify_specification(R, target)

    def verify_robustness(self, inputSet, reachOptions, target):
        """NN.verify_robustness (NN.m:651-667): 1 robust, 2 unknown (0 is never
        produced by an over-approximating method).  ``target`` is the 1-based label
        or HalfSpace(s)."""
        if np.isscalar(target):
            return int(self.verify_robustness_batch([inputSet], reachOptions, [int(target)])[0])
        R = self.reach(inputSet, reachOptions)
        return self.checkRobust(R, target)

    def verify_robustness_batch(self, inputSets, reachOptions, targets, class_type="max", stats=None):
        """verify_robustness over a list of sets with 1-based label targets.

        Device side: reach, then for every halfspace row of the robustness
        specification (a) its minimum over the output set's predicate box — a
        positive minimum proves the intersection empty — and (b) a greedy
        witness point of the output set — a point inside the halfspace proves it
        non-empty.  Host side, only for queries still undecided: the feasibility
        LP of Star.isEmptySet on the open rows, on the constraint system of that
        query re-reached with constraint records kept."""
        try:
            b = self.reach_batch(inputSets, reachOptions, keep_layer_bounds=True)
        except L.NNVError as e:
            if e.status != L.NNVB_E_CAPACITY or len(inputSets) < 2:
                raise
            # the generator tensors of the whole list do not fit the context's arena: two halves, one after the other
            h = len(inputSets) // 2
            parts, part_stats = [], []
            for sl in (slice(0, h), slice(h, None)):
                st = {} if stats is not None else None
                parts.append(self.verify_robustness_batch(inputSets[sl], reachOptions, list(targets[sl]), class_type, st))
                part_stats.append(st)
            if stats is not None:
                for k in set(part_stats[0]) | set(part_stats[1]):
                    stats[k] = part_stats[0].get(k, 0) + part_stats[1].get(k, 0)
            return np.concatenate(parts)
        t0 = np.asarray(targets, dtype=np.int64) - 1
        verdict, status, _ = b.verify_robust(t0, class_type)
        b.close()
        return self.finish_verdicts(inputSets, reachOptions, targets, verdict, class_type, stats)

    def finish_verdicts(self, inputSets, reachOptions, targets, verdict, class_type="max", stats=None):
        """Turn the device's first-pass answers (``Batch.verify_robust``: 1 robust, 2 unknown, -1 undecided) into
        the verdicts of verify_robustness for every set: the undecided ones are re-reached with the crossing rows
        of every ReLU layer kept, so that the device can also bound each open halfspace row by back-substitution
        through the recorded relaxations (decides most rows the LP would find empty), and what is still open
        goes to the feasibility LP of Star.isEmptySet on that pass's constraint system."""
        verdict = np.asarray(verdict)
        t0 = np.asarray(targets, dtype=np.int64) - 1
        result = np.where(verdict == L.VERDICT_EMPTY, 1, np.where(verdict == L.VERDICT_NONEMPTY, 2, 0)).astype(np.int64)
        undecided = np.nonzero(verdict == L.UNDECIDED)[0]
        if stats is not None:
            stats["n_prefilter"] = int((verdict == L.VERDICT_EMPTY).sum())
            stats["n_witness"] = int((verdict == L.VERDICT_NONEMPTY).sum())
            stats["n_lp_queries"] = int(len(undecided))
            stats["n_backsub"] = 0
        group = 32                      # bounds the size of the constraint records
        lp_tasks = []                   # (query, output set, halfspace): one feasibility LP each, all independent
        for g0 in range(0, len(undecided), group):
            qs = undecided[g0:g0 + group]
            try:
                bq = self.reach_batch([inputSets[q] for q in qs], reachOptions, keep_constraints=True,
                                      keep_layer_bounds=True)
            except L.NNVError:
                if len(qs) == 1:
                    raise
                # records of the whole group do not fit: one query at a time
                for q in qs:
                    result[q] = self.verify_robustness_batch([inputSets[q]], reachOptions, [targets[q]], class_type)[0]
                continue
            v2, s2, _ = bq.verify_robust(t0[qs], class_type)
            for k, q in enumerate(qs):
                if v2[k] == L.VERDICT_EMPTY:
                    result[q] = 1
                    if stats is not None:
                        stats["n_backsub"] += 1
                        stats["n_lp_queries"] -= 1
                elif v2[k] == L.VERDICT_NONEMPTY:
                    result[q] = 2
                    if stats is not None:
                        stats["n_lp_queries"] -= 1
                else:
                    S = _result_set(bq, k, True)
                    hs = self.robustness_set(int(targets[q]), class_type)
                    result[q] = 1                                  # until a row's intersection is found non-empty
                    lp_tasks.extend((q, S, hs[i]) for i in np.nonzero(s2[k] == L.UNDECIDED)[0])
            bq.close()
        # verify_specification.m:36-79 stops at the first non-empty intersection of a query; the rows are independent
        # LPs, so those of all groups run at once on the host cores and the verdict is the same OR
        nonempty = _lp_map(lambda t: _row_meets_star(t[1], t[2].G, t[2].g), lp_tasks)
        for (q, _, _), ne in zip(lp_tasks, nonempty):
            if ne:
                result[q] = 2
        return result


def _result_set(b, q, as_star):
    P, m = b.out_dims(q)
    h, w, c = b.net.out_shape
    pl, pu = b.get_pred_bounds(q)
    V = b.get_V(q)
    Cm, d = b.get_constraints(q)
    if as_star:
        return Star(V.reshape(h * w * c, -1, order="F"), Cm, d, pl, pu)
    return ImageStar(V, Cm, d, pl, pu)


def verify_specification(reachSet, property):
    """verify_specification.m:36-79: OR over halfspaces, AND over sets; 1 iff every
    intersection is empty, 2 at the first non-empty one."""
    R = reachSet if isinstance(reachSet, (list, tuple)) else [reachSet]
    prop = property if isinstance(property, (list, tuple)) else [property]
    for hs in prop:
        for S in R:
            if not isinstance(S, Star):
                S = S.toStar()
            if S.intersectHalfSpace(hs.G, hs.g) is not None:
                return 2
    return 1
