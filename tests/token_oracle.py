"""Plain 64-bit implementations of the token operators and of gradient
clipping, written from their definitions, and device buffers for calls of the
pointer-level entries."""
import ctypes

import numpy as np

U = 2.0 ** -24  # half a step of float32, relative


class Buf:
    """A device buffer of the library's pool holding a numpy array."""

    def __init__(self, rt, arr, offset=0):
        """offset: bytes between the allocation's (aligned) start and the array."""
        self.rt, self.arr, self.offset = rt, np.ascontiguousarray(arr), offset
        p = ctypes.c_void_p()
        assert rt.lib.tp_alloc(self.arr.nbytes + offset + 16, ctypes.byref(p)) == 0
        self.base = p.value
        self.ptr = self.base + offset
        self.write(self.arr)

    def write(self, arr):
        arr = np.ascontiguousarray(arr, self.arr.dtype)
        assert arr.nbytes == self.arr.nbytes
        if arr.nbytes:
            assert self.rt.lib.tp_memcpy_h2d(self.ptr, arr.ctypes.data_as(ctypes.c_void_p), arr.nbytes) == 0
            self.rt.synchronize()

    def read(self):
        out = np.empty_like(self.arr)
        if out.nbytes:
            assert self.rt.lib.tp_memcpy_d2h(out.ctypes.data_as(ctypes.c_void_p), self.ptr, out.nbytes) == 0
        return out

    def free(self):
        assert self.rt.lib.tp_free(self.base) == 0


def ids_array(ids, kind):
    return np.asarray(ids, np.int32 if kind else np.float32)


def logprobs(x, ids, K):
    """x [R, V] float32; returns a dict of float64 / int results and the
    quantities the tolerances are made of."""
    x = np.asarray(x, np.float64)
    R, V = x.shape
    out = {"logp": np.empty(R), "entropy": np.empty(R), "stats": np.empty((R, 2)),
           "top_ids": np.full((R, K), -1, np.int64), "top_logp": np.full((R, K), -np.inf),
           "A": np.zeros(R), "lnS": np.zeros(R)}
    for r in range(R):
        row = x[r]
        t = int(ids[r])
        if np.isnan(row).any() or np.isposinf(row).any():
            out["logp"][r] = 0.0 if t < 0 else np.nan
            out["entropy"][r] = np.nan
            out["stats"][r] = np.nan
            out["top_logp"][r] = np.nan
            continue
        m = row.max()
        if np.isneginf(m):
            out["logp"][r] = 0.0 if t < 0 else (np.nan if t >= V else -np.inf)
            out["entropy"][r] = 0.0
            out["stats"][r] = -np.inf
            continue
        with np.errstate(over="ignore"):
            y = row - m
        e = np.exp(y)
        S = e.sum()
        ye = np.where(e > 0, np.where(np.isfinite(y), y, 0.0) * e, 0.0)
        A = -ye.sum() / S
        lnS = np.log(S)
        out["A"][r], out["lnS"][r] = A, lnS
        out["entropy"][r] = lnS + A
        out["stats"][r] = m, lnS
        out["logp"][r] = 0.0 if t < 0 else (np.nan if t >= V else y[t] - lnS)
        if K:
            order = np.argsort(-row, kind="stable")[:K]
            order = order[row[order] > -np.inf]
            out["top_ids"][r, :len(order)] = order
            out["top_logp"][r, :len(order)] = y[order] - lnS
    for k in ("logp", "top_logp"):  # beyond the float32 range, where a rounding gives infinity
        out[k][out[k] < -3.4028235677973366e38] = -np.inf
    return out


def logprobs_tolerance(o, V):
    """Absolute bounds on the float32 kernel's errors, (logp-like given the
    value lp, entropy).  exp(y) of an f32 y = x - m: y is off by u|y|, its
    product with log2(e) by as much again, the exponential by 2 ulp = 4u; terms
    below e^-24 of the maximum add less than their errors can show.  A sum of
    positive terms in chains of at most V/256 + 64 adds: that many u.  So log S
    is off by u (2*24 + 4 + V/256 + 64); the sum of e*y, all of one sign, by
    that relative to A = -sum e y / S plus one product and one division."""
    chain = 2 * 24 + 4 + V / 256 + 64
    lnS, A = np.abs(o["lnS"]), o["A"]
    with np.errstate(invalid="ignore"):
        lp = lambda v: U * (chain + 2 * lnS.reshape((-1,) + (1,) * (v.ndim - 1)) + 3 * np.abs(v))  # noqa: E731
        ent = U * (chain * (1 + 2 * A) + 4 * A + 2 * lnS + np.abs(o["entropy"]))
    return lp, ent


def logprobs_grad(x, ids, stats, entropy, dlogp, dentropy):
    """(gradient, bound) from the float32 stats and entropy the kernel is given."""
    x = np.asarray(x, np.float64)
    R, V = x.shape
    d, tol = np.zeros((R, V)), np.zeros((R, V))
    chain = 2 * 24 + 4 + V / 256 + 64
    for r in range(R):
        t = int(ids[r]) if ids is not None else -1
        # the upstream gradients as the kernel is given them: float32
        c1 = float(np.float32(dlogp[r])) if dlogp is not None and t >= 0 else 0.0
        c2 = float(np.float32(dentropy[r])) if dentropy is not None else 0.0
        if c1 == 0.0 and c2 == 0.0:
            continue
        row = x[r]
        if np.isnan(row).any() or np.isposinf(row).any():
            d[r] = np.nan
            continue
        m = row.max()
        if np.isneginf(m):
            continue
        if c1 != 0.0 and t >= V:
            d[r] = np.nan
            continue
        with np.errstate(over="ignore"):
            lnS = np.log(np.exp(row - m).sum())
            lp = np.maximum((row - m) - lnS, -1e4)
        p = np.exp(lp)
        H = -(p * lp).sum()
        hot = np.zeros(V)
        if 0 <= t < V:
            hot[t] = 1.0
        d[r] = c1 * (hot - p) - c2 * p * (lp + H)
        # p from f32 stats: its exponent is off by the forward's error of log S,
        # the roundings of log S, of two differences and of a product; H likewise
        E = chain + 2 * abs(lnS) + 4 * np.minimum(np.abs(lp), 110) + 4
        EH = chain * (1 + 2 * H) + 4 * H + 2 * abs(lnS) + H
        tol[r] = U * (abs(c1) * (2 * hot + p * (E + 4))
                      + abs(c2) * p * ((np.abs(lp) + H) * (E + 6) + E + EH)) + 1e-37 * (abs(c1) + abs(c2) * 200)
    return d, tol


def embed_grad(dout, ids, V, scale, pad, old=None):
    """(gradient, bound): f32 sums in chains of at most 128 rows, the chains'
    results added with at most as many roundings again, one product by the
    scale and one addition to the old value."""
    D = dout.shape[1]
    ids = np.asarray(ids)
    g, a, cnt = np.zeros((V, D)), np.zeros((V, D)), np.zeros(V)
    keep = (ids >= 0) & (ids < V) & (ids != pad)
    np.add.at(g, ids[keep].astype(np.int64), dout[keep].astype(np.float64))
    np.add.at(a, ids[keep].astype(np.int64), np.abs(dout[keep]).astype(np.float64))
    np.add.at(cnt, ids[keep].astype(np.int64), 1.0)
    s = float(np.float32(scale))
    g, a = g * s, a * abs(s)
    tol = U * (np.minimum(cnt, 256)[:, None] + 3) * a
    if old is not None:
        g = g + old
        tol = tol + U * np.abs(g)
        tol[cnt == 0] = 0.0
    return g, tol


def clip(grads, p, max_norm):
    flat = np.concatenate([np.asarray(g, np.float64).ravel() for g in grads]) if grads else np.zeros(0)
    with np.errstate(invalid="ignore", over="ignore"):
        if flat.size == 0:
            norm = 0.0
        elif np.isinf(p):
            norm = np.abs(flat).max()
        else:
            norm = (np.abs(flat) ** p).sum() ** (1.0 / p)
        coef = np.float64(np.float32(max_norm)) / (norm + 1e-6)
    return norm, (1.0 if coef > 1.0 else coef)
