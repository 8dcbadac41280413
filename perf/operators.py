"""Token operators and gradient clipping: the two ends of a language model's
training step and of its sampling loop, measured.

Six kinds of case:

* ``logprobs``       log-probability of a given token per row of logits, the
                     row's entropy, and its ``topk`` most likely tokens
* ``logprobs_grad``  gradient of the first two with respect to the logits
* ``embed``          rows of a table by token id, scaled
* ``embed_grad``     the table's gradient, summed over the positions of a token
* ``clip``           the global norm of many gradients, scaled in place when it
                     exceeds a bound
* ``clip_step``      that norm, and the AdamW step that reads the scaled gradients

Where ``own`` is false, ``run`` computes them from elementary torch operations;
where it is true, it calls the pointer-level entries of libtpcuda on the same
buffers.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
IGNORED = -100

_runtime = None


def _rt():
    global _runtime
    if _runtime is None:
        pkg = os.path.join(ROOT, "torch-pyodide_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from tpcuda import CudaRuntime
        _runtime = CudaRuntime()
    return _runtime


def _check(status):
    if status:
        raise RuntimeError(_rt().lib.tp_last_error().decode())


# ---- the cases ------------------------------------------------------------------------------------

def listed():
    return [
        # sampling one sequence: one row of logits with the twenty alternatives an API returns
        {"name": "logprobs one row", "kind": "logprobs", "rows": 1, "vocab": 32000, "topk": 20, "pad": 0, "masked": 0.0,
         "bf16": True},
        # scoring prompts: an odd vocabulary, so that no two rows start at the same alignment
        {"name": "logprobs scoring", "kind": "logprobs", "rows": 1999, "vocab": 50021, "topk": 5, "pad": 0,
         "masked": 0.0, "bf16": True},
        # the policy's log-probabilities and entropies over a training batch and a large vocabulary
        {"name": "logprobs policy", "kind": "logprobs", "rows": 8192, "vocab": 131072, "topk": 0, "pad": 0,
         "masked": 0.0, "bf16": False},
        # a byte vocabulary under a grammar's mask
        {"name": "logprobs bytes masked", "kind": "logprobs", "rows": 65536, "vocab": 258, "topk": 3, "pad": 0,
         "masked": 0.5, "bf16": False},
        # a policy's loss with an entropy bonus
        {"name": "logprobs grad entropy", "kind": "logprobs_grad", "rows": 4096, "vocab": 32000, "entropy": True,
         "pad": 0, "ignored": 0.0},
        # a supervised batch whose prompt tokens are ignored, odd vocabulary
        {"name": "logprobs grad ignored", "kind": "logprobs_grad", "rows": 777, "vocab": 50021, "entropy": False,
         "pad": 0, "ignored": 0.3},
        # the next token of four sequences
        {"name": "embed decode", "kind": "embed", "n": 4, "dim": 4096, "vocab": 32000, "scale": 1.0, "ids": "int32"},
        # a training batch's tokens, scaled by the square root of the width
        {"name": "embed batch", "kind": "embed", "n": 32768, "dim": 2048, "vocab": 65536, "scale": 45.25483399593904,
         "ids": "float32"},
        # a training batch's gradient, written whole
        {"name": "embed grad batch", "kind": "embed_grad", "n": 16384, "dim": 4096, "vocab": 32000, "scale": 1.0,
         "ids": "int32", "accumulate": False, "padding": -1},
        # a small padded batch added to a gradient that is there already (a shared table), odd width
        {"name": "embed grad small", "kind": "embed_grad", "n": 301, "dim": 777, "vocab": 5003, "scale": 27.87471972953,
         "ids": "float32", "accumulate": True, "padding": 0},
        # many odd tensors under the bound: the norm is all there is to do
        {"name": "clip under", "kind": "clip", "tensors": 37, "total": 20000003, "norm": "2", "over": False},
        # clipping and AdamW over the 64 tensors of the optimizer benchmark
        {"name": "clip step", "kind": "clip_step", "tensors": 64, "total": 402718720, "over": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["logprobs", "logprobs", "logprobs_grad", "embed", "embed_grad", "embed_grad", "clip", "clip_step"])
    if kind == "logprobs":
        topk = rng.choice([0, 0, 1, 2, 5, 11, 20, 32])
        vocab = _log(rng, max(2, topk), 200000)
        most = (1 << 30 if topk == 0 else 100000000) // vocab
        return {"kind": kind, "rows": _log(rng, 1, min(most, 65536)), "vocab": vocab, "topk": topk,
                "pad": rng.choice([0, 0, 1, 2, 3, 4, 7]),
                "masked": 0.5 if vocab >= 4 * topk + 64 and rng.random() < 0.3 else 0.0, "bf16": rng.random() < 0.5}
    if kind == "logprobs_grad":
        vocab = _log(rng, 2, 200000)
        return {"kind": kind, "rows": _log(rng, 1, min((1 << 28) // vocab, 65536)), "vocab": vocab,
                "entropy": rng.random() < 0.5, "pad": rng.choice([0, 0, 1, 2, 3, 4, 7]),
                "ignored": rng.choice([0.0, 0.25, 0.9])}
    if kind in ("embed", "embed_grad"):
        dim = _log(rng, 1, 8192)
        if rng.random() < 0.5:
            dim = (dim + 3) // 4 * 4
        c = {"kind": kind, "n": _log(rng, 1, min((1 << 26) // dim, 262144)), "dim": dim,
             "vocab": _log(rng, 1, min((1 << 27) // dim, 200000)), "scale": rng.choice([1.0, math.sqrt(dim)]),
             "ids": rng.choice(["int32", "float32"])}
        if kind == "embed_grad":
            c["accumulate"] = rng.random() < 0.5
            c["padding"] = 0 if c["vocab"] > 1 and rng.random() < 0.3 else -1
        return c
    tensors = rng.randint(1, 64)
    c = {"kind": kind, "tensors": tensors, "total": _log(rng, 1000, 400000000), "over": rng.random() < 0.5}
    if kind == "clip":
        c["norm"] = rng.choice(["2", "2", "1", "inf"])
    return c


# ---- inputs ---------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _tokens(g, n, vocab):
    """Token ids as text has them: the k-th most frequent about 1/k as often as the first."""
    u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
    return ((vocab + 1.0) ** u).floor().long().sub_(1).clamp_(0, vocab - 1)


def _sizes(case):
    """Element counts of the case's tensors: the optimizer benchmark's, or odd ones that sum to the total."""
    if case["total"] == 402718720:
        return [(4096 * 4096, 4096, 1024 * 4096, 4096 * 1024)[i % 4] for i in range(case["tensors"])]
    w = np.array([1 + (i * 7919) % 13 for i in range(case["tensors"])], dtype=np.float64)
    ends = np.floor(np.cumsum(w) / w.sum() * case["total"]).astype(np.int64)
    ends[-1] = case["total"]
    return [int(v) for v in np.diff(np.concatenate([[0], ends]))]


def _offsets(case):
    """Where each tensor starts in the flat buffers (256-byte boundaries), and the buffers' length."""
    at, off = [], 0
    for n in _sizes(case):
        at.append(off)
        off += (n + 63) // 64 * 64
    return at, off


def _flat(case, g, std):
    """A flat buffer of the case's tensors, zero between them."""
    at, length = _offsets(case)
    out = torch.zeros(length, device=DEV)
    for o, n in zip(at, _sizes(case)):
        out[o:o + n].normal_(0.0, std, generator=g)
    return out


class _Group:
    """The tensor group a step driver builds once over its flat buffers."""

    def __init__(self, case, p, g, m, v):
        import ctypes
        at, _ = _offsets(case)
        sizes = _sizes(case)
        k = len(sizes)
        rows = [(ctypes.c_void_p * k)(*[t.data_ptr() + 4 * o for o in at]) for t in (p, g, m, v)]
        out = ctypes.c_int64(0)
        self.lib = _rt().lib
        _check(self.lib.tpk_group_create(k, *rows, (ctypes.c_int64 * k)(*sizes), ctypes.byref(out)))
        self.id = out.value

    def __del__(self):
        self.lib.tpk_group_destroy(self.id)


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    s = {"case": dict(case)}
    if kind in ("logprobs", "logprobs_grad"):
        R, V = case["rows"], case["vocab"]
        whole = torch.randn(R, V + case["pad"], generator=g, device=DEV).mul_(4.0)
        if case.get("bf16"):  # logits that a 16-bit product made: many equal values
            whole.copy_(whole.to(torch.bfloat16))
        x = whole[:, :V]
        ids = torch.randint(0, V, (R,), generator=g, device=DEV)
        if kind == "logprobs":
            if case["masked"]:
                gone = torch.rand(R, V, generator=g, device=DEV) < case["masked"]
                gone[:, :max(1, 2 * case["topk"])] = False
                gone.scatter_(1, ids[:, None], False)
                x.masked_fill_(gone, -math.inf)
                del gone
            K = case["topk"]
            s.update(logp=torch.empty(R, device=DEV), entropy=torch.empty(R, device=DEV),
                     stats=torch.empty(R, 2, device=DEV),
                     top_ids=torch.empty(R, K, device=DEV, dtype=torch.int32), top_logp=torch.empty(R, K, device=DEV))
        else:
            ids = torch.where(torch.rand(R, generator=g, device=DEV) < case["ignored"], IGNORED, ids)
            x64 = x.amax(1).double()
            lnS = torch.empty(R, device=DEV, dtype=torch.float64)
            ent = torch.empty(R, device=DEV, dtype=torch.float64)
            step = max(1, (1 << 26) // V)
            for r in range(0, R, step):  # what the forward pass left
                y = x[r:r + step].double() - x64[r:r + step, None]
                e = y.exp()
                lnS[r:r + step] = e.sum(1).log()
                ent[r:r + step] = lnS[r:r + step] - (e * y).sum(1) / e.sum(1)
            s.update(stats=torch.stack([x64, lnS], 1).float(), entropy=ent.float(),
                     dlogp=torch.randn(R, generator=g, device=DEV),
                     dentropy=torch.full((R,), -0.01, device=DEV) if case["entropy"] else None,
                     dlogits=torch.zeros(R, V + case["pad"], device=DEV)[:, :V])
        s.update(logits=x, ids=ids.to(torch.int32))
    elif kind in ("embed", "embed_grad"):
        n, D, V = case["n"], case["dim"], case["vocab"]
        ids = _tokens(g, n, V)
        if kind == "embed":
            s.update(table=torch.randn(V, D, generator=g, device=DEV).mul_(0.02), out=torch.empty(n, D, device=DEV))
        else:
            if case["padding"] >= 0:
                ids[n - n // 4:] = case["padding"]
            s.update(dout=torch.randn(n, D, generator=g, device=DEV),
                     dtable=torch.randn(V, D, generator=g, device=DEV) if case["accumulate"]
                     else torch.empty(V, D, device=DEV))
            if own:  # the workspace a step driver keeps
                import ctypes
                nbytes = ctypes.c_int64(0)
                _check(_rt().lib.tpk_token_embedding_backward_ws(n, V, D, ctypes.byref(nbytes)))
                s["ws"] = torch.empty(max(1, nbytes.value), device=DEV, dtype=torch.uint8)
        s["ids"] = ids.to(torch.int32 if case["ids"] == "int32" else torch.float32)
    else:
        grad = _flat(case, g, 1e-3)
        t = case["total"]
        size = {"2": math.sqrt(t), "1": t * math.sqrt(2.0 / math.pi), "inf": 5.0}[case.get("norm", "2")] * 1e-3
        s.update(grad=grad, max_norm=size * (0.25 if case["over"] else 4.0), norm=torch.empty(2, device=DEV))
        if kind == "clip_step":
            s.update(param=_flat(case, g, 0.02), exp_avg=_flat(case, g, 1e-3).mul_(0.1),
                     exp_avg_sq=_flat(case, g, 1e-3).square_())
        if own:  # the tensor table a step driver builds once
            s["group"] = _Group(case, s.get("param", grad), grad, s.get("exp_avg", grad), s.get("exp_avg_sq", grad))
    return s


HYPER = {"lr": 1e-3, "b1": 0.9, "b2": 0.999, "eps": 1e-8, "wd": 0.01, "step": 10}


def _hyper():
    """Hyper-parameters of the step as the optimizers pass them: bias corrections on the host."""
    h = HYPER
    step_size = h["lr"] / (1.0 - h["b1"] ** h["step"])
    inv = 1.0 / math.sqrt(1.0 - h["b2"] ** h["step"])
    return h["lr"], h["b1"], h["b2"], h["eps"], h["wd"], step_size, inv


# ---- the plain forms ------------------------------------------------------------------------------

def _plain_logprobs(s):
    x, ids, K = s["logits"], s["ids"].long(), s["case"]["topk"]
    m = x.amax(1, keepdim=True)
    y = x - m
    e = y.exp()
    S = e.sum(1, keepdim=True)
    ln = S.log()
    entropy = ln[:, 0] - torch.where(e > 0, e * y, 0.0).sum(1) / S[:, 0]
    del e, S
    logp = y.gather(1, ids[:, None])[:, 0] - ln[:, 0]
    out = {"logp": logp, "entropy": entropy, "stats": torch.cat([m, ln], 1)}
    if K:
        top = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :K]
        out.update(top_ids=top.to(torch.int32), top_logp=y.gather(1, top) - ln)
    return out


def _plain_logprobs_grad(s):
    x, ids = s["logits"], s["ids"].long()
    live = (ids >= 0).float()
    lp = x - s["stats"][:, :1] - s["stats"][:, 1:]
    p = lp.exp()
    c1 = (s["dlogp"] * live)[:, None]
    d = -c1 * p
    d.scatter_add_(1, ids.clamp(min=0)[:, None], c1)
    if s["dentropy"] is not None:
        d -= s["dentropy"][:, None] * (p * (lp + s["entropy"][:, None]))
    return {"dlogits": d}


def _plain_embed(s):
    return {"out": s["table"][s["ids"].long()] * s["case"]["scale"]}


def _plain_embed_grad(s):
    c = s["case"]
    ids = s["ids"].long()
    rows = s["dout"].double() * (ids != c["padding"]).double()[:, None]
    total = torch.zeros(c["vocab"], c["dim"], device=DEV, dtype=torch.float64).index_add_(0, ids, rows)
    total = (total * c["scale"]).float()
    if c["accumulate"]:
        s["dtable"] += total
        return {"dtable": s["dtable"]}
    return {"dtable": total}


def _plain_norm(s):
    g, p = s["grad"], s["case"].get("norm", "2")
    if p == "inf":
        norm = g.abs().amax().double()
    elif p == "1":
        norm = g.abs().sum(dtype=torch.float64)
    else:
        norm = g.double().square().sum().sqrt()
    return norm, (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)


def _plain_clip(s):
    norm, coef = _plain_norm(s)
    s["grad"] *= coef.float()
    return {"norm": torch.stack([norm, coef]).float(), "grad": s["grad"]}


def _plain_clip_step(s):
    lr, b1, b2, eps, wd, step_size, inv = _hyper()
    norm, coef = _plain_norm(s)
    g = s["grad"] * coef.float()
    p, m, v = s["param"], s["exp_avg"], s["exp_avg_sq"]
    p -= (lr * wd) * p
    m.mul_(b1).add_(g * (1.0 - b1))
    v.mul_(b2).add_(g * g * (1.0 - b2))
    p -= m / (v.sqrt() * inv + eps) * step_size
    return {"norm": torch.stack([norm, coef]).float(), "param": p, "exp_avg": m, "exp_avg_sq": v}


# ---- the framework's calls ------------------------------------------------------------------------

def _ptr(t):
    return t.data_ptr() if t is not None else None


def _kind(t):
    return 1 if t.dtype == torch.int32 else 0


def _own_logprobs(s):
    x, K = s["logits"], s["case"]["topk"]
    _check(_rt().lib.tpk_token_logprobs(
        x.data_ptr(), x.stride(0), s["ids"].data_ptr(), _kind(s["ids"]), x.shape[0], x.shape[1], K,
        s["logp"].data_ptr(), s["entropy"].data_ptr(), s["stats"].data_ptr(),
        s["top_ids"].data_ptr() if K else None, s["top_logp"].data_ptr() if K else None))
    out = {k: s[k] for k in ("logp", "entropy", "stats")}
    if K:
        out.update(top_ids=s["top_ids"], top_logp=s["top_logp"])
    return out


def _own_logprobs_grad(s):
    x, d = s["logits"], s["dlogits"]
    _check(_rt().lib.tpk_token_logprobs_backward(
        x.data_ptr(), x.stride(0), s["ids"].data_ptr(), _kind(s["ids"]), s["stats"].data_ptr(),
        s["entropy"].data_ptr(), s["dlogp"].data_ptr(), _ptr(s["dentropy"]), x.shape[0], x.shape[1], d.data_ptr(),
        d.stride(0)))
    return {"dlogits": d}


def _own_embed(s):
    c, t, out = s["case"], s["table"], s["out"]
    _check(_rt().lib.tpk_token_embedding(t.data_ptr(), t.stride(0), s["ids"].data_ptr(), _kind(s["ids"]), c["n"],
                                         c["vocab"], c["dim"], c["scale"], out.data_ptr(), out.stride(0)))
    return {"out": out}


def _own_embed_grad(s):
    c, g, t, ws = s["case"], s["dout"], s["dtable"], s["ws"]
    _check(_rt().lib.tpk_token_embedding_backward(
        g.data_ptr(), g.stride(0), s["ids"].data_ptr(), _kind(s["ids"]), c["n"], c["vocab"], c["dim"], c["scale"],
        c["padding"], 1 if c["accumulate"] else 0, t.data_ptr(), t.stride(0), ws.data_ptr(), ws.numel()))
    return {"dtable": t}


def _own_clip(s):
    _check(_rt().lib.tpk_group_clip_grad_norm(s["group"].id, float(s["case"].get("norm", "2")), s["max_norm"],
                                              s["norm"].data_ptr()))
    return {"norm": s["norm"], "grad": s["grad"]}


def _own_clip_step(s):
    lib, group, norm = _rt().lib, s["group"].id, s["norm"]
    _check(lib.tpk_group_grad_norm(group, 2.0, s["max_norm"], norm.data_ptr()))
    _check(lib.tpk_adam_group_scaled(group, 0, *_hyper(), norm.data_ptr() + 4))
    return {"norm": norm, "param": s["param"], "exp_avg": s["exp_avg"], "exp_avg_sq": s["exp_avg_sq"]}


def run(state):
    kind = state["case"]["kind"]
    return globals()[("_own_" if own else "_plain_") + kind](state)


# ---- what a pass cannot do without ----------------------------------------------------------------

def _distinct(n, vocab):
    """How many different tokens _tokens gives, on average."""
    v = np.arange(vocab, dtype=np.float64)
    p = (np.log(v + 2) - np.log(v + 1)) / math.log(vocab + 1.0)
    return float(-np.expm1(n * np.log1p(-np.minimum(p, 1 - 1e-12))).sum())


def work(case):
    kind = case["kind"]
    if kind == "logprobs":
        R, V, K = case["rows"], case["vocab"], case["topk"]
        return {"bytes": 4 * R * V + 4 * R + 16 * R + 8 * R * K, "flops": 5 * R * V}
    if kind == "logprobs_grad":  # rows without a gradient need not be read
        R, V = case["rows"], case["vocab"]
        live = R if case["entropy"] else R * (1.0 - case["ignored"])
        return {"bytes": 4 * live * V + 4 * R * V + 28 * R, "flops": (8 if case["entropy"] else 4) * live * V}
    if kind == "embed":
        n, D = case["n"], case["dim"]
        return {"bytes": 4 * n * D + 4 * D * _distinct(n, case["vocab"]) + 4 * n, "flops": n * D}
    if kind == "embed_grad":
        n, D, V = case["n"], case["dim"], case["vocab"]
        live = n - n // 4 if case["padding"] >= 0 else n
        table = 8 * D * _distinct(live, V) if case["accumulate"] else 4 * V * D
        return {"bytes": 4 * live * D + table + 4 * n, "flops": live * D}
    t = case["total"]
    if kind == "clip":
        return {"bytes": (12 if case["over"] else 4) * t, "flops": 2 * t}
    return {"bytes": 28 * t, "flops": 16 * t}


# ---- the definitions in 64 bits -------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "logprobs":
        parts = []
        step = max(1, (1 << 26) // case["vocab"])
        for r in range(0, case["rows"], step):
            x = s["logits"][r:r + step].double()
            top = x.amax(1)
            lse = torch.logsumexp(x, 1)
            lp = x - lse[:, None]
            p = lp.exp()
            t = s["ids"][r:r + step].long()
            row = {"logp": lp[torch.arange(len(t), device=DEV), t],
                   "entropy": torch.where(p > 0, -p * lp, 0.0).sum(1),
                   "stats": torch.stack([top, torch.log((x - top[:, None]).exp().sum(1))], 1)}
            if case["topk"]:
                v, i = torch.sort(lp, dim=1, descending=True, stable=True)
                i32 = torch.sort(s["logits"][r:r + step], dim=1, descending=True, stable=True).indices
                row.update(top_ids=i32[:, :case["topk"]].to(torch.int32), top_logp=v[:, :case["topk"]])
            parts.append(row)
        return {k: torch.cat([q[k] for q in parts]) for k in parts[0]}
    if kind == "logprobs_grad":
        out = torch.empty(case["rows"], case["vocab"], device=DEV, dtype=torch.float64)
        step = max(1, (1 << 25) // case["vocab"])
        for r in range(0, case["rows"], step):
            x = s["logits"][r:r + step].double()
            p = torch.softmax(x, 1)
            lp = x - torch.logsumexp(x, 1)[:, None]
            H = -(p * lp).sum(1, keepdim=True)
            t = s["ids"][r:r + step].long()
            hot = torch.zeros_like(p)
            rows = torch.nonzero(t >= 0)[:, 0]
            hot[rows, t[rows]] = 1.0
            up = torch.where(t >= 0, s["dlogp"][r:r + step].double(), 0.0)[:, None]
            d = up * (hot - p)
            if s["dentropy"] is not None:
                d += s["dentropy"][r:r + step].double()[:, None] * (-p * (lp + H))
            out[r:r + step] = d
        return {"dlogits": out}
    if kind == "embed":
        return {"out": s["table"].double().index_select(0, s["ids"].long()).mul_(float(np.float32(case["scale"])))}
    if kind == "embed_grad":
        ids = s["ids"].long()
        total = (s["dtable"].double() if case["accumulate"]
                 else torch.zeros(case["vocab"], case["dim"], device=DEV, dtype=torch.float64))
        keep = torch.nonzero(ids != case["padding"])[:, 0]
        total.index_add_(0, ids[keep], s["dout"][keep].double(), alpha=float(np.float32(case["scale"])))
        return {"dtable": total}
    g = s["grad"].double()
    p = float(case.get("norm", "2"))
    norm = g.abs().amax() if math.isinf(p) else g.abs().pow_(p).sum() ** (1.0 / p)
    coef = torch.clamp(float(np.float32(s["max_norm"])) / (norm + 1e-6), max=1.0)
    g = g * coef
    both = torch.stack([norm, coef])
    if kind == "clip":
        return {"norm": both, "grad": g}
    lr, b1, b2, eps, wd, step_size, inv = (float(np.float32(v)) for v in _hyper())
    m = b1 * s["exp_avg"].double() + (1.0 - b1) * g
    v = b2 * s["exp_avg_sq"].double() + (1.0 - b2) * g * g
    w = s["param"].double() * (1.0 - lr * wd) - step_size * m / (v.sqrt() * inv + eps)
    return {"norm": both, "param": w, "exp_avg": m, "exp_avg_sq": v}
