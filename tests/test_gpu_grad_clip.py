"""The global gradient norm and clipping against 64-bit plain implementations.

The norm is summed in f64 and rounded once, the coefficient computed in f64 and
rounded once; a scaled gradient is one product by that f32 coefficient.  So the
norm is within one rounding (and the f64 sum's 1e-12), the coefficient too, and
the gradients are bit-equal to numpy's product with the coefficient returned."""
import ctypes

import numpy as np
import pytest

from token_oracle import U, Buf, clip

pytestmark = pytest.mark.gpu

SETS = {"one": [1], "three": [3], "odd": [1, 2, 5, 17, 1000, 4097, 65537], "chunks": [65536, 65535, 131073, 4],
        "many": [((i * 7919) % 3001) + 1 for i in range(300)], "large": [3000001, 12, 1700000],
        "holes": [0, 5, 0, 64, 0]}
TYPES = [2.0, 1.0, float("inf")]


class Group:
    def __init__(self, rt, *arrays):
        """arrays: lists of numpy arrays (grads first); made into one group."""
        self.rt, self.n = rt, len(arrays[0])
        self.bufs = [[Buf(rt, a.astype(np.float32)) for a in side] for side in arrays]
        g = self.bufs[0]
        p, m, v = (self.bufs[1:4] if len(self.bufs) == 4 else (g, g, g))
        out = ctypes.c_int64()
        ptrs = [(ctypes.c_void_p * max(1, self.n))(*[b.ptr for b in side]) for side in (p, g, m, v)]
        sizes = (ctypes.c_int64 * max(1, self.n))(*[a.size for a in arrays[0]])
        assert rt.lib.tpk_group_create(self.n, *ptrs, sizes, ctypes.byref(out)) == 0, rt.lib.tp_last_error()
        self.id = out.value
        self.out = Buf(rt, np.full(3, -5.0, np.float32))

    def grads(self):
        return [b.read() for b in self.bufs[0]]

    def free(self):
        assert self.rt.lib.tpk_group_destroy(self.id) == 0
        for b in sum(self.bufs, []) + [self.out]:
            b.free()


def same_norm(got, norm, coef):
    for g, w in zip(got, (norm, coef)):
        w = np.float64(w)
        if not np.isfinite(w):
            assert np.array_equal(np.float64(g), w, equal_nan=True), (got, norm, coef)
        else:
            assert abs(np.float64(g) - w) <= (1.001 * U + 1e-12) * abs(w) + 1e-45, (got, norm, coef)


@pytest.mark.parametrize("sizes", SETS.values(), ids=SETS.keys())
@pytest.mark.parametrize("p", TYPES)
@pytest.mark.parametrize("over", [False, True])
def test_group(cuda_rt, sizes, p, over):
    rt = cuda_rt
    rng = np.random.default_rng(len(sizes) + sum(sizes))
    g = [rng.standard_normal(n).astype(np.float32) for n in sizes]
    max_norm = np.float32(clip(g, p, 1)[0] * (0.3 if over else 2.0))
    norm, coef = clip(g, p, max_norm)
    G = Group(rt, g)
    assert rt.lib.tpk_group_grad_norm(G.id, p, max_norm, G.out.ptr) == 0
    first = G.out.read()
    same_norm(first[:2], norm, coef)
    assert first[2] == -5.0 and all(np.array_equal(a, b) for a, b in zip(G.grads(), g))
    assert rt.lib.tpk_group_clip_grad_norm(G.id, p, max_norm, G.out.ptr) == 0
    second = G.out.read()
    assert np.array_equal(first, second)
    assert (second[1] < 1) == over
    for a, b in zip(G.grads(), g):
        assert np.array_equal(a, b * second[1] if over else b)
    G.free()


@pytest.mark.parametrize("p", TYPES)
def test_values_at_the_edges(cuda_rt, p):
    rt = cuda_rt
    inf, nan = np.inf, np.nan
    for g in ([[1e30, 2e30], [3e38]], [[1e-30, -2e-30], [1e-42]], [[0.0, -0.0], [0.0]], [[1.0, inf], [2.0]],
              [[1.0], [-inf, 3.0]], [[nan, 1.0], [2.0]], [[1.0], [nan, inf]]):
        g = [np.array(a, np.float32) for a in g]
        for max_norm in (0.0, 1e-3, 1.0, 1e38, inf):
            norm, coef = clip(g, p, max_norm)
            G = Group(rt, g)
            assert rt.lib.tpk_group_clip_grad_norm(G.id, p, max_norm, G.out.ptr) == 0
            got = G.out.read()
            with np.errstate(over="ignore"):
                same_norm(got[:2], np.float32(norm) if np.isfinite(norm) and norm > 3.5e38 else norm, coef)
            for a, b in zip(G.grads(), g):
                with np.errstate(invalid="ignore"):
                    assert np.array_equal(a, b * got[1], equal_nan=True), (g, max_norm, got)
            G.free()


def test_empty_group(cuda_rt):
    G = Group(cuda_rt, [])
    assert cuda_rt.lib.tpk_group_clip_grad_norm(G.id, 2.0, 1.0, G.out.ptr) == 0
    assert G.out.read().tolist() == [0.0, 1.0, -5.0]
    G.free()


def test_overlapping_gradients_are_refused(cuda_rt):
    rt = cuda_rt
    b = Buf(rt, np.ones(100, np.float32))
    out = Buf(rt, np.zeros(2, np.float32))
    for ptrs, sizes in (([b.ptr, b.ptr], [50, 50]), ([b.ptr, b.ptr + 64], [17, 20]), ([b.ptr + 64, b.ptr], [1, 100])):
        g = ctypes.c_int64()
        arr = (ctypes.c_void_p * 2)(*ptrs)
        assert rt.lib.tpk_group_create(2, arr, arr, arr, arr, (ctypes.c_int64 * 2)(*sizes), ctypes.byref(g)) == 0
        assert rt.lib.tpk_group_clip_grad_norm(g.value, 2.0, 1.0, out.ptr) == -1
        assert b"twice" in rt.lib.tp_last_error()
        assert rt.lib.tpk_group_grad_norm(g.value, 2.0, 1.0, out.ptr) == 0  # reading it twice is harmless
        assert rt.lib.tpk_group_destroy(g.value) == 0
    t = rt.ones([5], "float32")["id"]
    with pytest.raises(RuntimeError, match="twice"):
        rt.clipGradNormMulti([t, t], 1.0)
    assert np.all(b.read() == 1.0) and rt.toList(t) == [1.0] * 5


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("over", [False, True])
def test_scaled_step_is_clip_then_step(cuda_rt, kind, over):
    """The step that scales on read gives the bits of clipping, then stepping."""
    rt = cuda_rt
    rng = np.random.default_rng(kind)
    sizes = [1, 3, 4097, 70001, 8]
    make = lambda s: [(rng.standard_normal(n) * s).astype(np.float32) for n in sizes]  # noqa: E731
    g, p, m, v = make(1.0), make(0.1), make(0.01), [np.abs(a) for a in make(0.01)]
    hyper = (1e-3, 0.9, 0.999, 1e-8, 0.01, 1.3e-3, 2.1)
    max_norm = clip(g, 2.0, 1)[0] * (0.1 if over else 3)
    a, b = Group(rt, g, p, m, v), Group(rt, g, p, m, v)
    assert rt.lib.tpk_group_grad_norm(a.id, 2.0, max_norm, a.out.ptr) == 0
    assert rt.lib.tpk_adam_group_scaled(a.id, kind, *hyper, a.out.ptr + 4) == 0
    assert rt.lib.tpk_group_clip_grad_norm(b.id, 2.0, max_norm, b.out.ptr) == 0
    assert rt.lib.tpk_adam_group(b.id, kind, *hyper) == 0
    for x, y in zip(sum(a.bufs[1:], []), sum(b.bufs[1:], [])):
        assert np.array_equal(x.read(), y.read())
    assert all(np.array_equal(x, y) for x, y in zip(a.grads(), g))
    # and through the runtime
    T = lambda arrs: [rt.tensorFromData(x, [x.size], "float32")["id"] for x in arrs]  # noqa: E731
    P, G, M, V = T(p), T(g), T(m), T(v)
    h = (rt.adamWClipStepMulti if kind == 0 else rt.adamClipStepMulti)(P, G, M, V, *hyper, max_norm)
    assert h["shape"] == [2] and np.array_equal(rt.toNumpy(h["id"]), a.out.read()[:2])
    for x, y in zip(P + M + V, sum(a.bufs[1:], [])):
        assert np.array_equal(rt.toNumpy(x), y.read())
    a.free()
    b.free()


def test_runtime_clip(cuda_rt):
    rt = cuda_rt
    rng = np.random.default_rng(3)
    g = [rng.standard_normal(s).astype(np.float32) for s in ((3, 5), (7,), (1, 1, 9))]
    ids = [rt.tensorFromData(a, list(a.shape), "float32")["id"] for a in g]
    before = rt.memoryAllocated()
    h = rt.clipGradNormMulti(ids, 0.5)
    got = rt.toNumpy(h["id"])
    same_norm(got, *clip(g, 2.0, 0.5))
    for i, a in zip(ids, g):
        assert np.array_equal(rt.toNumpy(i), (a * got[1]).ravel())
    rt.destroy(h["id"])
    assert rt.memoryAllocated() == before
    assert rt.toList(rt.clipGradNormMulti([], 1.0, 1.0)["id"]) == [0.0, 1.0]
    with pytest.raises(RuntimeError):
        rt.clipGradNormMulti([rt.argmax(rt.zeros([2, 2], "float32")["id"])["id"]], 1.0)
    with pytest.raises(RuntimeError):
        rt.adamWClipStepMulti(ids[:1], ids[1:2], ids[:1], ids[:1], *[0.1] * 7, 1.0)
    with pytest.raises(RuntimeError):
        rt.adamWClipStepMulti(ids, ids[:1], ids, ids, *[0.1] * 7, 1.0)


def test_equal_inputs_equal_bits(cuda_rt):
    rt = cuda_rt
    rng = np.random.default_rng(4)
    g = [rng.standard_normal(n).astype(np.float32) for n in SETS["large"]]
    G = Group(rt, g)
    got = []
    for _ in range(4):
        assert rt.lib.tpk_group_grad_norm(G.id, 2.0, 1.0, G.out.ptr) == 0
        got.append(G.out.read())
    assert all(np.array_equal(got[0], x) for x in got)
    G.free()
