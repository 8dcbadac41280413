"""tokenEmbedding and its gradient against 64-bit plain implementations.  The
forward is one product, rounded once; the gradient's bound counts the roundings
of its sums (token_oracle.embed_grad)."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest

from token_oracle import U, Buf, embed_grad, ids_array

pytestmark = pytest.mark.gpu

GUARD = np.float32(-12345.0)


def zipf(rng, n, V):
    return np.minimum((V + 1.0) ** rng.random(n) - 1, V - 1).astype(np.int64)


def lookup(rt, table, ids, scale, kind=1, ld=0, ldo=0, offset=0):
    V, D = table.shape
    wide = np.full((V, D + ld), 7e37, np.float32)
    wide[:, :D] = table
    T, I = Buf(rt, wide, offset), Buf(rt, ids_array(ids, kind))
    O = Buf(rt, np.full((len(ids) + 1, D + ldo), GUARD, np.float32), offset)
    assert rt.lib.tpk_token_embedding(T.ptr, D + ld, I.ptr, kind, len(ids), V, D, scale, O.ptr, D + ldo) == 0
    rt.synchronize()
    got = O.read()
    assert np.all(got[len(ids)] == GUARD) and np.all(got[:, D:] == GUARD)
    for b in (T, I, O):
        b.free()
    return got[:len(ids), :D]


@pytest.mark.parametrize("n", [1, 2, 7, 33, 1000])
@pytest.mark.parametrize("V, D", [(1, 1), (7, 3), (11, 4), (100, 31), (64, 128), (50, 777), (33, 1024), (9, 4100)])
def test_lookup(cuda_rt, n, V, D):
    rng = np.random.default_rng(n * 31 + V * 7 + D)
    table, ids = rng.standard_normal((V, D)).astype(np.float32), zipf(rng, n, V)
    scale = np.float32([1.0, np.sqrt(D), -0.37][(n + D) % 3])
    got = lookup(cuda_rt, table, ids, scale, kind=n % 2, ld=D % 3, ldo=(n + V) % 3, offset=4 * (D % 4))
    assert np.array_equal(got, table[ids] * scale)


def test_lookup_of_ids_outside_the_table(cuda_rt):
    table = np.arange(12, dtype=np.float32).reshape(3, 4)
    for kind, ids in ((1, [0, -1, 3, 2, 2 ** 31 - 1, -(2 ** 31)]), (0, [0, -1, 3, 2, 1e30, -np.inf])):
        got = lookup(cuda_rt, table, ids, 2.0, kind=kind)
        assert np.array_equal(got[[0, 3]], table[[0, 2]] * 2)
        assert np.isnan(got[[1, 2, 4, 5]]).all()
    got = lookup(cuda_rt, table, [np.nan, 1.9, -0.9], 1.0, kind=0)
    assert np.isnan(got[0]).all() and np.array_equal(got[1:], table[[1, 0]])


def test_lookup_keeps_what_the_table_holds(cuda_rt):
    table = np.array([[np.inf, -np.inf, np.nan, -0.0], [3e38, 1e-42, 1.0, -1.0]], np.float32)
    got = lookup(cuda_rt, table, [0, 1, 0], 1.0)
    assert np.array_equal(got, table[[0, 1, 0]], equal_nan=True)
    assert np.signbit(got[0, 3])


def grad(rt, dout, ids, V, scale, pad=-1, old=None, kind=1, ld=0, ldo=0, offset=0):
    n, D = dout.shape
    wide = np.full((n, D + ldo), 7e37, np.float32)
    wide[:, :D] = dout
    tab = np.full((V + 1, D + ld), GUARD, np.float32)
    if old is not None:
        tab[:V, :D] = old
    G, I, T = Buf(rt, wide, offset), Buf(rt, ids_array(ids, kind)), Buf(rt, tab, offset)
    need = ctypes.c_int64()
    assert rt.lib.tpk_token_embedding_backward_ws(n, V, D, ctypes.byref(need)) == 0
    W = Buf(rt, np.full(need.value + 64, 0xA5, np.uint8))
    assert rt.lib.tpk_token_embedding_backward(G.ptr, D + ldo, I.ptr, kind, n, V, D, scale, pad, int(old is not None),
                                               T.ptr, D + ld, W.ptr, need.value) == 0, rt.lib.tp_last_error()
    rt.synchronize()
    got, ws = T.read(), W.read()
    assert np.all(got[V] == GUARD) and np.all(got[:, D:] == GUARD)
    assert np.all(ws[need.value:] == 0xA5)
    for b in (G, I, T, W):
        b.free()
    return got[:V, :D]


def check_grad(rt, dout, ids, V, scale=1.0, pad=-1, old=None, **how):
    dout = np.ascontiguousarray(dout, np.float32)
    got = grad(rt, dout, ids, V, scale, pad, old, **how)
    want, tol = embed_grad(dout, ids, V, scale, pad, old)
    over = np.abs(got - want) - tol
    assert over.max() <= 0, (float(over.max()), np.unravel_index(over.argmax(), over.shape))
    return got


@pytest.mark.parametrize("n", [1, 2, 5, 31, 64, 129, 300, 2047, 2049, 5000])
@pytest.mark.parametrize("V, D", [(1, 1), (3, 5), (10, 4), (700, 33), (5003, 64), (40, 777), (300, 1028)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_gradient(cuda_rt, n, V, D, accumulate):
    rng = np.random.default_rng(n * 7 + V * 3 + D)
    dout, ids = rng.standard_normal((n, D)), zipf(rng, n, V)
    old = rng.standard_normal((V, D)).astype(np.float32) if accumulate else None
    check_grad(cuda_rt, dout, ids, V, [1.0, np.sqrt(D)][n % 2], pad=0 if n % 3 == 0 else -1, old=old, kind=D % 2,
               ld=V % 3, ldo=n % 2, offset=4 * (n % 4))


@pytest.mark.parametrize("n", [40, 700, 9000])
@pytest.mark.parametrize("what", ["one token", "all different", "padding only", "alternating", "runs", "outside"])
@pytest.mark.parametrize("accumulate", [False, True])
def test_gradient_patterns(cuda_rt, n, what, accumulate):
    rng = np.random.default_rng(n)
    V, D = 12000, 20
    i = np.arange(n)
    ids = {"one token": np.full(n, 11999), "all different": rng.permutation(V)[:n], "padding only": np.full(n, 5),
           "alternating": np.where(i % 2, 7, 11000), "runs": i // 64, "outside": np.where(i % 3, i % 9, -1 - i)}[what]
    if what == "outside":
        ids[::7] = V + i[::7]
    old = rng.standard_normal((V, D)).astype(np.float32) if accumulate else None
    got = check_grad(cuda_rt, rng.standard_normal((n, D)), ids, V, 1.0, pad=5, old=old)
    if what == "padding only":
        assert np.array_equal(got, old if accumulate else np.zeros((V, D)))


@pytest.mark.parametrize("D, ld, ldo, offset", [(1, 0, 0, 0), (2, 0, 0, 8), (6, 2, 4, 0), (30, 0, 2, 8), (31, 0, 1, 4),
                                                 (34, 0, 0, 0), (500, 2, 0, 8), (521, 3, 7, 12), (1026, 0, 0, 0),
                                                 (1024, 4, 8, 0), (1024, 1, 0, 0), (9001, 0, 0, 0)])
def test_widths_and_strides(cuda_rt, D, ld, ldo, offset):
    """Columns of 4, 8 and 16 bytes, by the widest that both buffers allow; around
    the most tokens that take one launch."""
    rng = np.random.default_rng(D)
    for n, V in ((0, 9), (1, 70), (512, 3), (512, 1500), (513, 70)):
        ids = rng.integers(-1, V + 1, n)
        dout = rng.standard_normal((n, D)).astype(np.float32)
        table = rng.standard_normal((V, D)).astype(np.float32)
        check_grad(cuda_rt, dout, ids, V, 0.75, pad=V // 2, kind=n % 2, ld=ld, ldo=ldo, offset=offset)
        check_grad(cuda_rt, dout, ids, V, 0.75, old=table, kind=n % 2, ld=ld, ldo=ldo, offset=offset)
        if n:
            got = lookup(cuda_rt, table, ids, 0.75, kind=n % 2, ld=ld, ldo=ldo, offset=offset)
            want = np.full((n, D), np.nan, np.float32)
            keep = (ids >= 0) & (ids < V)
            want[keep] = table[ids[keep]] * np.float32(0.75)
            assert np.array_equal(got, want, equal_nan=True)


def test_gradient_of_few_tokens_needs_no_workspace(cuda_rt):
    rt = cuda_rt
    G, I = Buf(rt, np.ones((4, 8), np.float32)), Buf(rt, np.array([2, 0, 2, 7], np.int32))
    T = Buf(rt, np.full((5, 8), GUARD, np.float32))
    assert rt.lib.tpk_token_embedding_backward(G.ptr, 8, I.ptr, 1, 4, 5, 8, 1.0, -1, 0, T.ptr, 8, None, 0) == 0
    assert np.array_equal(T.read(), np.array([1, 0, 2, 0, 0], np.float32)[:, None] * np.ones(8, np.float32))


def test_gradient_of_long_sums(cuda_rt):
    """One token in 70000 of 100000 positions: the bound grows with the sums'
    length as far as two levels of 256 go."""
    rng = np.random.default_rng(8)
    n = 100000
    ids = np.where(rng.random(n) < 0.7, 3, zipf(rng, n, 500))
    check_grad(cuda_rt, rng.standard_normal((n, 36)) + 1.0, ids, 500, 0.5)
    check_grad(cuda_rt, rng.standard_normal((n, 3)), ids, 500, 0.5, old=rng.standard_normal((500, 3)).astype(np.float32))


@pytest.mark.parametrize("n, V", [(600001, 3000), (40000, 1), (33000, 131072), (32769, 140000), (5000, 1000000),
                                  (300001, 2 ** 20 + 5), (20000, 2 ** 20 + 5), (70001, 3 * 2 ** 20 + 17),
                                  (600001, 2 ** 22), (1, 2 ** 22 - 1)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_gradient_of_many_tokens(cuda_rt, n, V, accumulate):
    """Ids that are split by owner before they are sorted, and more positions than
    one sort keeps hits of in shared memory."""
    rng = np.random.default_rng(17)
    old = rng.standard_normal((V, 2)).astype(np.float32) if accumulate else None
    ids = zipf(rng, n, V)
    ids[::9] = -1
    check_grad(cuda_rt, rng.standard_normal((n, 2)), ids, V, 1.0, pad=min(7, V) - 1, old=old, kind=n % 2)


@pytest.mark.parametrize("V", [1, 149, 100000, 2 ** 20])
def test_gradient_vocabularies(cuda_rt, V):
    rng = np.random.default_rng(V)
    for n in (3, 3000):
        check_grad(cuda_rt, rng.standard_normal((n, 8)), rng.integers(0, V, n), V)


@pytest.mark.parametrize("n", [0, 5, 3000])
def test_gradient_largest_vocabulary(cuda_rt, n):
    """Owners of 16384 tokens, which sort them in parts; the last id of each part, and of the table."""
    V = 2 ** 24
    ids = np.random.default_rng(n).integers(0, V, n)
    ids[:4] = [V - 1, 0, 2 ** 20 - 1, 2 ** 20][:n]
    check_grad(cuda_rt, np.random.default_rng(1).standard_normal((n, 1)), ids, V)


def test_gradient_untouched_rows_keep_their_bits(cuda_rt):
    rng = np.random.default_rng(2)
    old = rng.standard_normal((50, 12)).astype(np.float32)
    old[7] = np.nan
    old[8] = -0.0
    for n in (20, 4000):
        got = grad(cuda_rt, rng.standard_normal((n, 12)).astype(np.float32), rng.integers(10, 20, n), 50, 3.0, old=old)
        keep = np.r_[0:10, 20:50]
        assert np.array_equal(got[keep].view(np.uint32), old[keep].view(np.uint32))


def test_gradient_nothing_leaks_from_left_out_rows(cuda_rt):
    rng = np.random.default_rng(4)
    for n in (100, 5000):
        dout, ids = rng.standard_normal((n, 9)).astype(np.float32), rng.integers(1, 40, n)
        ids[::5], ids[1::5] = 0, 40
        clean = dout.copy()
        dout[::5], dout[1::5] = np.nan, np.inf
        clean[::5], clean[1::5] = 0, 0
        a = grad(cuda_rt, dout, ids, 40, 1.0, pad=0)
        assert np.array_equal(a, grad(cuda_rt, clean, ids, 40, 1.0, pad=0)) and np.all(a[0] == 0)


def test_gradient_equal_inputs_equal_bits(cuda_rt):
    rng = np.random.default_rng(6)
    for n, V, D in ((500, 100, 64), (20000, 3000, 33), (30000, 7, 128)):
        dout, ids = rng.standard_normal((n, D)).astype(np.float32), zipf(rng, n, V)
        a = grad(cuda_rt, dout, ids, V, 1.0)
        for _ in range(3):
            assert np.array_equal(a, grad(cuda_rt, dout, ids, V, 1.0))


def test_offsets_beyond_32_bits(cuda_rt):
    """Rows of table, output and gradient 1.1 * 10^9 values apart."""
    rt = cuda_rt
    ld, D, V = 1100000000, 8, 3
    p = ctypes.c_void_p()
    assert rt.lib.tp_alloc((2 * ld + D) * 4, ctypes.byref(p)) == 0
    table = np.random.default_rng(3).standard_normal((V, D)).astype(np.float32)

    def rows(put=None):
        out = np.zeros((V, D), np.float32)
        for r in range(V):
            if put is not None:
                assert rt.lib.tp_memcpy_h2d(p.value + 4 * ld * r, put[r].ctypes.data_as(ctypes.c_void_p), 4 * D) == 0
            else:
                assert rt.lib.tp_memcpy_d2h(out[r].ctypes.data_as(ctypes.c_void_p), p.value + 4 * ld * r, 4 * D) == 0
        return out

    rows(table)
    ids = np.array([2, 0, 2, 1], np.int32)
    I, O = Buf(rt, ids), Buf(rt, np.zeros((4, D), np.float32))
    assert rt.lib.tpk_token_embedding(p.value, ld, I.ptr, 1, 4, V, D, 1.0, O.ptr, D) == 0
    assert np.array_equal(O.read(), table[ids])
    W = Buf(rt, np.zeros(1 << 16, np.uint8))
    for acc, want in ((1, 2 * table), (0, table)):  # a table's rows come back as their gradient
        want = want.copy()
        want[2] += table[2]
        assert rt.lib.tpk_token_embedding_backward(O.ptr, D, I.ptr, 1, 4, V, D, 1.0, -1, acc, p.value, ld, W.ptr,
                                                   1 << 16) == 0
        assert np.allclose(rows(), want, rtol=4 * U)
    J = Buf(rt, np.array([0, 1, 1], np.int32))
    R = Buf(rt, np.zeros((V, D), np.float32))
    rows(table)
    assert rt.lib.tpk_token_embedding_backward(p.value, ld, J.ptr, 1, 3, V, D, 1.0, -1, 0, R.ptr, D, W.ptr, 1 << 16) == 0
    assert np.allclose(R.read(), [table[0], table[1] + table[2], 0 * table[0]], rtol=4 * U)
    assert rt.lib.tp_free(p.value) == 0


def test_first_call_inside_a_capture():
    """In a fresh process the first gradient is captured, not run."""
    code = """
import ctypes, sys
import numpy as np
sys.path[:0] = [%r, %r]
from tpcuda import CudaRuntime
from token_oracle import Buf, embed_grad
rt = CudaRuntime()
rng = np.random.default_rng(0)
n, V, D = 3000, 500, 20
dout, ids = rng.standard_normal((n, D)).astype(np.float32), rng.integers(0, V, n).astype(np.int32)
need = ctypes.c_int64()
assert rt.lib.tpk_token_embedding_backward_ws(n, V, D, ctypes.byref(need)) == 0
G, I, T, W = (Buf(rt, a) for a in (dout, ids, np.zeros((V, D), np.float32), np.zeros(need.value, np.uint8)))
assert rt.lib.tp_graph_begin() == 0
assert rt.lib.tpk_token_embedding_backward(G.ptr, D, I.ptr, 1, n, V, D, 1.0, -1, 0, T.ptr, D, W.ptr, need.value) == 0
g = ctypes.c_int64()
assert rt.lib.tp_graph_end(ctypes.byref(g)) == 0, rt.lib.tp_last_error()
for _ in range(2):
    assert rt.lib.tp_graph_launch(g.value) == 0
want, tol = embed_grad(dout, ids, V, 1.0, -1)
assert np.all(np.abs(T.read() - want) <= tol)
print("captured")
"""
    here = os.path.dirname(os.path.abspath(__file__))
    code = code % (os.path.join(os.path.dirname(here), "torch-pyodide_b200"), here)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_gradient_empty_batch(cuda_rt):
    rt = cuda_rt
    T = Buf(rt, np.full((5, 6), GUARD, np.float32))
    W = Buf(rt, np.zeros(4096, np.uint8))
    assert rt.lib.tpk_token_embedding_backward(None, 6, None, 0, 0, 5, 6, 1.0, -1, 1, T.ptr, 6, W.ptr, 4096) == 0
    assert np.all(T.read() == GUARD)
    assert rt.lib.tpk_token_embedding_backward(None, 6, None, 0, 0, 5, 6, 1.0, -1, 0, T.ptr, 6, W.ptr, 4096) == 0
    assert np.all(T.read() == 0)


def test_gradient_against_differences(cuda_rt):
    """The lookup is linear in the table: <dout, lookup(table + h u) -
    lookup(table)> / h is <grad, u> but for f32 roundings."""
    rng = np.random.default_rng(12)
    V, D, n = 30, 16, 200
    dout, ids = rng.standard_normal((n, D)).astype(np.float32), zipf(rng, n, V)
    u = rng.standard_normal((V, D)).astype(np.float32)
    g = check_grad(cuda_rt, dout, ids, V, 1.5).astype(np.float64)
    moved = lookup(cuda_rt, u, ids, 1.5).astype(np.float64)
    scale = np.abs(dout * moved).sum()
    assert abs((dout * moved).sum() - (g * u).sum()) <= 40 * U * scale


# ---- handles ------------------------------------------------------------------------------------------

def test_runtime_surface(cuda_rt):
    rt = cuda_rt
    rng = np.random.default_rng(13)
    table = rng.standard_normal((40, 12)).astype(np.float32)
    ids = rng.integers(0, 40, (3, 5))
    T = rt.tensorFromData(table, [40, 12], "float32")
    I = rt.tensorFromData(ids.astype(np.float32), [3, 5], "int64")
    before = rt.memoryAllocated()
    y = rt.tokenEmbedding(T["id"], I["id"], 3.0)
    assert y["shape"] == [3, 5, 12]
    assert np.array_equal(rt.toNumpy(y["id"]).reshape(3, 5, 12), table[ids] * np.float32(3))
    dout = rng.standard_normal((3, 5, 12)).astype(np.float32)
    G = rt.tensorFromData(dout, [3, 5, 12], "float32")
    d = rt.tokenEmbeddingBackward(G["id"], I["id"], 40, 3.0, paddingId=int(ids[0, 0]))
    want, tol = embed_grad(dout.reshape(15, 12), ids.ravel(), 40, 3.0, int(ids[0, 0]))
    assert d["shape"] == [40, 12] and np.all(np.abs(rt.toNumpy(d["id"]).reshape(40, 12) - want) <= tol)
    first = rt.toNumpy(d["id"]).reshape(40, 12)
    again = rt.tokenEmbeddingBackward(G["id"], I["id"], 40, 3.0, into=d["id"])
    assert again["id"] == d["id"] and again["shape"] == [40, 12]
    want, tol = embed_grad(dout.reshape(15, 12), ids.ravel(), 40, 3.0, -1, first)
    assert np.all(np.abs(rt.toNumpy(d["id"]).reshape(40, 12) - want) <= tol)
    for h in (y, G, d):
        rt.destroy(h["id"])
    assert rt.memoryAllocated() == before


def test_runtime_refusals(cuda_rt):
    rt = cuda_rt
    T = rt.zeros([6, 4], "float32")["id"]
    ids = rt.zeros([5], "int64")["id"]
    G = rt.zeros([5, 4], "float32")["id"]
    index = rt.argmax(T)["id"]
    for call in (lambda: rt.tokenEmbedding(G + 99999, ids), lambda: rt.tokenEmbedding(ids, ids),
                 lambda: rt.tokenEmbedding(index, ids), lambda: rt.tokenEmbeddingBackward(G, index, 6),
                 lambda: rt.tokenEmbeddingBackward(G, ids, 0), lambda: rt.tokenEmbeddingBackward(G, ids, 6, paddingId=6),
                 lambda: rt.tokenEmbeddingBackward(G, ids, 6, paddingId=-2),
                 lambda: rt.tokenEmbeddingBackward(G, ids, 5, into=T), lambda: rt.tokenEmbeddingBackward(G, ids, 5, into=G)):
        with pytest.raises(RuntimeError):
            call()
    empty = rt.tokenEmbedding(T, rt.zeros([0], "int64")["id"])
    assert empty["shape"] == [0, 4]
