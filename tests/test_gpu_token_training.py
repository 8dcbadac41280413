"""The token operators together, as a language model's step and its sampling
loop use them: lookup, a linear layer to logits, log-probabilities with
entropy, their gradients, the table's gradient, the global norm and the clipped
AdamW step; captured into a graph and replayed; beside each other on two
streams; the next token fed back without a readback."""
import ctypes

import numpy as np
import pytest

from token_oracle import Buf, clip, logprobs

pytestmark = pytest.mark.gpu

HYPER = (1e-3, 0.9, 0.999, 1e-8, 0.01, 1e-2, 31.6)


def adamw(p, g, m, v):
    lr, b1, b2, eps, wd, step, inv = (float(np.float32(x)) for x in HYPER)
    p = p * (1 - lr * wd)
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    return p - step * m / (np.sqrt(v) * inv + eps), m, v


def model(E, W, ids, targets, c1, c2, scale):
    """The step in 64 bits: gradients of sum(c1 logp + c2 H)."""
    h = E[ids] * scale
    x = h @ W.T
    o = logprobs(x, targets, 0)
    lp = x - (o["stats"][:, :1] + o["stats"][:, 1:])
    p = np.exp(lp)
    hot = np.zeros_like(x)
    live = targets >= 0
    hot[np.arange(len(ids))[live], targets[live]] = 1.0
    d = (c1 * live)[:, None] * (hot - p) - c2[:, None] * p * (lp + o["entropy"][:, None])
    dE = np.zeros_like(E)
    np.add.at(dE, ids, (d @ W) * scale)
    return o, d, dE, d.T @ h


def make(V=97, D=24, n=140, seed=0):
    rng = np.random.default_rng(seed)
    E, W = rng.standard_normal((V, D)) * 0.5, rng.standard_normal((V, D)) * 0.5
    ids = np.minimum((V + 1.0) ** rng.random(n) - 1, V - 1).astype(np.int64)
    targets = np.where(rng.random(n) < 0.2, -100, rng.integers(0, V, n))
    c1, c2 = np.full(n, -1.0 / n), np.full(n, -0.01 / n)
    f = lambda a: a.astype(np.float32).astype(np.float64)  # noqa: E731
    return f(E), f(W), ids, targets, f(c1), f(c2)


def close(got, want, rel, what):
    want = np.asarray(want)
    err = np.linalg.norm(np.asarray(got, np.float64).reshape(want.shape) - want)
    assert err <= rel * np.linalg.norm(want), (what, err, np.linalg.norm(want))


# Sums of at most 140 products of float32 inputs, three of them after each other
# (logits, gradient, table or weight): roundings of 2^-24 each, random in sign,
# are within 1e-5 of the result in norm; the 3xTF32 products drop terms of 2^-21.
REL = 2e-5


def test_training_step_through_the_runtime(cuda_rt):
    rt = cuda_rt
    E, W, ids, targets, c1, c2 = make()
    scale = np.float32(24 ** 0.5)
    T = lambda a, dt="float32": rt.tensorFromData(np.asarray(a, np.float32), list(np.shape(a)), dt)["id"]  # noqa: E731
    e, w, i, t = T(E), T(W), T(ids, "int64"), T(targets, "int64")
    state = [T(np.zeros_like(x)) for x in (E, W, E, W)]
    h = rt.tokenEmbedding(e, i, scale)["id"]
    x = rt.linear(h, w)["id"]
    lp, en, st, ti, tl = (q["id"] for q in rt.tokenLogprobs(x, t, 3))
    dx = rt.tokenLogprobsBackward(T(c1), T(c2), x, t, st, en)["id"]
    dh = rt.matmul(dx, w)["id"]
    dw = rt.matmul(rt.transpose2d(dx)["id"], h)["id"]
    de = rt.tokenEmbeddingBackward(dh, i, 97, scale)["id"]
    o, d, dE, dW = model(E, W, ids, targets, c1, c2, float(scale))
    close(rt.toNumpy(lp), o["logp"], REL, "logp")
    close(rt.toNumpy(en), o["entropy"], REL, "entropy")
    close(rt.toNumpy(dx), d, REL, "logits' gradient")
    close(rt.toNumpy(de), dE, REL, "table's gradient")
    close(rt.toNumpy(dw), dW, REL, "weight's gradient")
    max_norm = 0.5 * clip([dE, dW], 2.0, 1.0)[0]
    norm = rt.adamWClipStepMulti([e, w], [de, dw], state[:2], state[2:], *HYPER, max_norm)["id"]
    n, c = clip([dE, dW], 2.0, max_norm)
    close(rt.toNumpy(norm), [n, c], REL, "norm")
    for got, p, g in ((e, E, dE), (w, W, dW)):
        new, _, _ = adamw(p, g * c, 0.0, 0.0)
        # the first step divides a gradient by its own size: sign(g) where |g| is well above eps / inv
        sure = np.abs(g * c) > 1e-6
        assert sure.mean() > 0.5
        assert np.abs(rt.toNumpy(got).reshape(p.shape) - new)[sure].max() < 1e-5
    # a tied table: its gradient from both ends
    both = rt.tokenEmbeddingBackward(dh, i, 97, scale, into=dw)["id"]
    close(rt.toNumpy(both), dE + dW, REL, "tied gradient")


class Step:
    """The same step on buffers of its own, as a driver keeps them."""

    def __init__(self, rt, E, W, n):
        self.rt, self.n, (self.V, self.D) = rt, n, E.shape
        f = lambda *s: Buf(rt, np.zeros(s, np.float32))  # noqa: E731
        V, D = self.V, self.D
        self.E, self.W = Buf(rt, E.astype(np.float32)), Buf(rt, W.astype(np.float32))
        self.ids, self.t = Buf(rt, np.zeros(n, np.int32)), Buf(rt, np.zeros(n, np.int32))
        self.c1, self.c2, self.h, self.x, self.lp, self.en, self.st = (f(n), f(n), f(n, D), f(n, V), f(n), f(n), f(n, 2))
        self.ti, self.tl = Buf(rt, np.zeros((n, 3), np.int32)), f(n, 3)
        self.dx, self.dh, self.dE, self.dW, self.norm = f(n, V), f(n, D), f(V, D), f(V, D), f(2)
        self.m, self.v = [f(V, D), f(V, D)], [f(V, D), f(V, D)]
        need = ctypes.c_int64()
        assert rt.lib.tpk_token_embedding_backward_ws(n, V, D, ctypes.byref(need)) == 0
        self.ws = Buf(rt, np.zeros(need.value, np.uint8))
        ptrs = lambda *b: (ctypes.c_void_p * 2)(*[q.ptr for q in b])  # noqa: E731
        g = ctypes.c_int64()
        assert rt.lib.tpk_group_create(2, ptrs(self.E, self.W), ptrs(self.dE, self.dW), ptrs(*self.m), ptrs(*self.v),
                                       (ctypes.c_int64 * 2)(V * D, V * D), ctypes.byref(g)) == 0
        self.group = g.value

    def feed(self, ids, targets, c1, c2):
        for b, a in ((self.ids, ids), (self.t, targets), (self.c1, c1), (self.c2, c2)):
            b.write(a)

    def run(self, scale, max_norm, update=True):
        L, n, V, D = self.rt.lib, self.n, self.V, self.D
        ok = [L.tpk_token_embedding(self.E.ptr, D, self.ids.ptr, 1, n, V, D, scale, self.h.ptr, D),
              L.tpk_gemm(self.h.ptr, 0, self.W.ptr, 1, self.x.ptr, n, V, D, None),
              L.tpk_token_logprobs(self.x.ptr, V, self.t.ptr, 1, n, V, 3, self.lp.ptr, self.en.ptr, self.st.ptr,
                                   self.ti.ptr, self.tl.ptr),
              L.tpk_token_logprobs_backward(self.x.ptr, V, self.t.ptr, 1, self.st.ptr, self.en.ptr, self.c1.ptr,
                                            self.c2.ptr, n, V, self.dx.ptr, V),
              L.tpk_gemm(self.dx.ptr, 0, self.W.ptr, 0, self.dh.ptr, n, D, V, None),
              L.tpk_gemm(self.dx.ptr, 1, self.h.ptr, 0, self.dW.ptr, V, D, n, None),
              L.tpk_token_embedding_backward(self.dh.ptr, D, self.ids.ptr, 1, n, V, D, scale, -1, 0, self.dE.ptr, D,
                                             self.ws.ptr, self.ws.arr.nbytes),
              L.tpk_group_grad_norm(self.group, 2.0, max_norm, self.norm.ptr)]
        if update:
            ok.append(L.tpk_adam_group_scaled(self.group, 0, *HYPER, self.norm.ptr + 4))
        assert not any(ok), (ok, L.tp_last_error())

    def outputs(self):
        return [b.read() for b in (self.lp, self.en, self.st, self.ti, self.tl, self.dx, self.dE, self.dW, self.norm,
                                   self.E, self.W, *self.m, *self.v)]


@pytest.mark.parametrize("n, V", [(140, 97), (700, 97), (24, 9001), (2500, 1500)])
def test_captured_step_replays_on_new_inputs(cuda_rt, n, V):
    """A captured step, replayed on inputs written between, gives the bits of
    the same calls made one by one; replays need nothing cleared between."""
    rt = cuda_rt
    E, W, *_ = make(V=V, n=n)
    batches = [make(V=V, n=n, seed=s)[2:] for s in range(1, 5)]
    eager, graph = Step(rt, E, W, n), Step(rt, E, W, n)
    for s in (eager, graph):  # scratch of the linear layers reaches its size
        s.feed(*batches[0])
        s.run(1.5, 0.05, update=False)
    rt.synchronize()
    assert rt.lib.tp_graph_begin() == 0
    graph.run(1.5, 0.05)
    g = ctypes.c_int64()
    assert rt.lib.tp_graph_end(ctypes.byref(g)) == 0, rt.lib.tp_last_error()
    for b in batches + batches[:1]:
        eager.feed(*b)
        eager.run(1.5, 0.05)
        graph.feed(*b)
        assert rt.lib.tp_graph_launch(g.value) == 0
        rt.synchronize()
        for i, (x, y) in enumerate(zip(eager.outputs(), graph.outputs())):
            assert np.array_equal(x, y, equal_nan=True), i
    assert rt.lib.tp_graph_destroy(g.value) == 0


def test_plain_stream_order_gives_the_same_bits(cuda_rt):
    """Without programmatic dependent launches (tp_set_pdl)."""
    rt = cuda_rt
    for n, V in ((140, 97), (24, 9001)):
        E, W, *batch = make(V=V, n=n)
        steps = []
        for pdl in (1, 0):
            assert rt.lib.tp_set_pdl(pdl) == 0
            s = Step(rt, E, W, n)
            s.feed(*batch)
            s.run(1.5, 0.05)
            rt.synchronize()
            steps.append(s.outputs())
        assert rt.lib.tp_set_pdl(1) == 0
        assert all(np.array_equal(a, b, equal_nan=True) for a, b in zip(*steps))


def test_two_steps_on_two_streams(cuda_rt):
    """The operators of two steps queued on the library's stream and on the
    auxiliary one at the same time, each with its own buffers."""
    rt = cuda_rt
    L = rt.lib
    rng = np.random.default_rng(5)
    n, V, D = 3000, 5000, 64

    def side(seed):
        r = np.random.default_rng(seed)
        x, ids = r.standard_normal((n, V)).astype(np.float32), r.integers(0, V, n).astype(np.int32)
        dout = r.standard_normal((n, D)).astype(np.float32)
        need = ctypes.c_int64()
        assert L.tpk_token_embedding_backward_ws(n, V, D, ctypes.byref(need)) == 0
        z = lambda *s, dt=np.float32: Buf(rt, np.zeros(s, dt))  # noqa: E731
        return dict(x=Buf(rt, x), ids=Buf(rt, ids), dout=Buf(rt, dout), lp=z(n), en=z(n), st=z(n, 2),
                    ti=z(n, 7, dt=np.int32), tl=z(n, 7), dx=z(n, V), dt=z(V, D), ws=z(need.value, dt=np.uint8))

    def run(s):
        assert L.tpk_token_logprobs(s["x"].ptr, V, s["ids"].ptr, 1, n, V, 7, s["lp"].ptr, s["en"].ptr, s["st"].ptr,
                                    s["ti"].ptr, s["tl"].ptr) == 0
        assert L.tpk_token_logprobs_backward(s["x"].ptr, V, s["ids"].ptr, 1, s["st"].ptr, s["en"].ptr, s["lp"].ptr,
                                             s["en"].ptr, n, V, s["dx"].ptr, V) == 0
        assert L.tpk_token_embedding_backward(s["dout"].ptr, D, s["ids"].ptr, 1, n, V, D, 1.0, -1, 0, s["dt"].ptr, D,
                                              s["ws"].ptr, s["ws"].arr.nbytes) == 0

    a, b = side(1), side(2)
    keys = ("lp", "en", "st", "ti", "tl", "dx", "dt")
    run(a), run(b)
    rt.synchronize()
    want = [[s[k].read() for k in keys] for s in (a, b)]
    for s in (a, b):
        for k in keys:
            s[k].write(np.zeros_like(s[k].arr))
    for _ in range(3):
        assert L.tp_aux_fork() == 0
        run(b)
        assert L.tp_aux_return() == 0
        run(a)
        assert L.tp_aux_join() == 0
    rt.synchronize()
    for s, ref in zip((a, b), want):
        for k, r in zip(keys, ref):
            assert np.array_equal(s[k].read(), r), k


def test_greedy_decoding_without_a_readback(cuda_rt):
    """The best token of each step is the next step's id: int32 alternatives go
    straight into the lookup."""
    rt = cuda_rt
    rng = np.random.default_rng(9)
    V, D, B = 60, 16, 3
    E, W = (rng.standard_normal((V, D)).astype(np.float32) for _ in range(2))
    e, w = (rt.tensorFromData(a, [V, D], "float32")["id"] for a in (E, W))
    ids = rt.tensorFromData(np.array([1, 2, 3], np.float32), [B], "int64")["id"]
    host = np.array([1, 2, 3])
    for _ in range(8):
        x = rt.linear(rt.tokenEmbedding(e, ids)["id"], w)["id"]
        _, _, _, top, _ = rt.tokenLogprobs(x, ids, 1)
        ids = rt.reshape(top["id"], [B])["id"]
        host = np.argmax(E[host].astype(np.float64) @ W.T.astype(np.float64), axis=1)
        assert rt.toList(ids) == host.tolist()
