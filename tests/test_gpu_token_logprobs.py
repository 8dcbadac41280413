"""tokenLogprobs and its gradient against 64-bit plain implementations.

Tolerances: token_oracle.logprobs_tolerance and logprobs_grad give, per value,
the sum of the roundings that any one-pass f32 evaluation of the formulas
makes; ids are compared exactly (equal logits: the lower id first)."""
import ctypes

import numpy as np
import pytest

from token_oracle import Buf, ids_array, logprobs, logprobs_grad, logprobs_tolerance

pytestmark = pytest.mark.gpu

LOW = np.finfo(np.float32).min
GUARD = np.float32(-12345.0)


def near(got, want, tol, what):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    odd = ~np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), (what, got[np.isnan(got) != np.isnan(want)][:4])
    assert np.array_equal(got[odd & ~np.isnan(want)], want[odd & ~np.isnan(want)]), what
    with np.errstate(invalid="ignore"):
        over = np.where(odd, -1.0, np.abs(got - want) - tol)
    assert over.size == 0 or over.max() <= 0, (what, float(over.max()), np.unravel_index(over.argmax(), over.shape),
                                               got.ravel()[over.argmax()], want.ravel()[over.argmax()])


def forward(rt, x, ids, K, kind=1, pad=0, offset=0):
    """One pointer-level call on rows of V + pad values starting `offset` bytes
    past a 16-byte boundary; the outputs end in guard values."""
    R, V = x.shape
    whole = np.full((R, V + pad), 7e37, np.float32)
    whole[:, :V] = x
    X, I = Buf(rt, whole, offset), Buf(rt, ids_array(ids, kind))
    outs = [Buf(rt, np.full(n + 3, GUARD, np.float32)) for n in (R, R, 2 * R, R * K)]
    top = Buf(rt, np.full(R * K + 3, -77, np.int32))
    assert rt.lib.tpk_token_logprobs(X.ptr, V + pad, I.ptr, kind, R, V, K, outs[0].ptr, outs[1].ptr, outs[2].ptr,
                                     top.ptr, outs[3].ptr) == 0, rt.lib.tp_last_error()
    rt.synchronize()
    lp, en, st, tl = (b.read() for b in outs)
    ti = top.read()
    for a in (lp, en, st, tl):
        assert np.all(a[-3:] == GUARD)
    assert np.all(ti[-3:] == -77)
    for b in (X, I, top, *outs):
        b.free()
    return {"logp": lp[:R], "entropy": en[:R], "stats": st[:2 * R].reshape(R, 2),
            "top_ids": ti[:R * K].reshape(R, K), "top_logp": tl[:R * K].reshape(R, K)}


def check(rt, x, ids, K, **how):
    x = np.ascontiguousarray(x, np.float32)
    got, want = forward(rt, x, ids, K, **how), logprobs(x, ids, K)
    lp, ent = logprobs_tolerance(want, x.shape[1])
    near(got["logp"], want["logp"], lp(want["logp"]), "logp")
    near(got["entropy"], want["entropy"], ent, "entropy")
    near(got["stats"][:, 0], want["stats"][:, 0], 2.0 ** -24 * np.abs(want["stats"][:, 0]), "max")
    near(got["stats"][:, 1], want["stats"][:, 1], lp(want["stats"][:, 1]), "log sum")
    assert np.array_equal(got["top_ids"], want["top_ids"]), np.argwhere(got["top_ids"] != want["top_ids"])[:4]
    near(got["top_logp"], want["top_logp"], lp(want["top_logp"]), "top logp")
    return got


def bf16(x):
    return ((np.asarray(x, np.float32).view(np.uint32) + 0x8000) & np.uint32(0xFFFF0000)).view(np.float32)


SIZES = [(1, 1), (3, 2), (2, 5), (5, 31), (4, 32), (3, 33), (7, 63), (300, 64), (9, 255), (2, 256), (3, 257), (5, 511),
         (6, 513), (3, 1000), (2, 1023), (5, 1025), (3, 2048), (4, 4099), (37, 5000), (2, 16385), (3, 32000), (1, 50021),
         (2, 65536), (1, 131075), (200, 8192)]


@pytest.mark.parametrize("R, V", SIZES)
@pytest.mark.parametrize("K", [0, 1, 5, 20, 32])
def test_sizes(cuda_rt, R, V, K):
    if K > V:
        K = V
    rng = np.random.default_rng(R * 1000003 + V * 37 + K)
    x = rng.standard_normal((R, V)) * 4
    if K % 2:
        x = bf16(x)
    ids = rng.integers(0, V, R)
    check(cuda_rt, x, ids, K, kind=V % 2, pad=(R + K) % 4, offset=4 * ((V + K) % 4))


@pytest.mark.parametrize("offset", [0, 4, 8, 12])
@pytest.mark.parametrize("pad", [0, 1, 2, 3, 8])
@pytest.mark.parametrize("V", [12, 700, 1500, 9001])
def test_alignment_and_stride(cuda_rt, V, pad, offset):
    rng = np.random.default_rng(V + pad + offset)
    check(cuda_rt, rng.standard_normal((6, V)) * 3, rng.integers(0, V, 6), 7, pad=pad, offset=offset)


@pytest.mark.parametrize("V", [3, 40, 300, 1100, 4097, 33000])
def test_special_rows(cuda_rt, V):
    """Masks that leave nothing, one token or the lowest value; NaN and
    infinities; large offsets; ignored and out-of-range ids."""
    rng = np.random.default_rng(V)
    base = rng.standard_normal(V) * 3
    rows, ids = [], []

    def add(row, t):
        rows.append(np.array(row, np.float64))
        ids.append(t)

    add(np.full(V, -np.inf), 0)
    add(np.full(V, -np.inf), -100)
    add(np.full(V, -np.inf), V)
    one = np.full(V, -np.inf)
    one[V - 1] = -2.5
    add(one, V - 1)
    add(one, 0)
    two = one.copy()
    two[0] = LOW
    add(two, 0)
    add(np.full(V, LOW), V // 2)
    add(np.full(V, 3.25), V - 1)
    add(np.full(V, -np.finfo(np.float32).max / 2), 1)
    low = base.copy()
    low[: V - 1] = LOW
    add(low, 0)
    part = np.where(rng.random(V) < 0.9, -np.inf, base)
    part[0] = 1.0
    add(part, 0)
    add(np.where(rng.random(V) < 0.9, LOW, base), 0)
    nan = base.copy()
    nan[V // 3] = np.nan
    add(nan, 0)
    add(nan, -1)
    inf = base.copy()
    inf[V - 1] = np.inf
    add(inf, 0)
    nan2 = np.full(V, -np.inf)
    nan2[0] = np.nan
    add(nan2, 0)
    add(base + 1e4, V - 1)
    add(base * 40, V // 2)
    add(base - 3e38, 0)
    add(base, -1)
    add(base, -(2 ** 24))
    add(base, V)
    add(base, 2 ** 24)
    add(np.where(np.arange(V) % 2, 0.0, -0.0), 0)
    big = np.full(V, -3e38)
    big[V // 2] = 3e38
    add(big, 0)
    for kind in (0, 1):
        check(cuda_rt, np.array(rows), ids, min(V, 9), kind=kind, pad=1)


def test_float_ids_are_truncated(cuda_rt):
    rt = cuda_rt
    x = np.random.default_rng(0).standard_normal((8, 50)).astype(np.float32)
    ids = np.array([3.9, -0.5, 49.99, -1.5, np.nan, np.inf, -np.inf, 1e30], np.float32)
    X, I, L = Buf(rt, x), Buf(rt, ids), Buf(rt, np.zeros(8, np.float32))
    assert rt.lib.tpk_token_logprobs(X.ptr, 50, I.ptr, 0, 8, 50, 0, L.ptr, None, None, None, None) == 0
    want = logprobs(x, [3, 0, 49, -1, 2 ** 24, 2 ** 24, 2 ** 24, 2 ** 24], 0)["logp"]
    near(L.read(), want, 1e-5, "logp")
    assert L.read()[3] == 0.0


def pattern(shape, V, K, rng):
    i, small = np.arange(V), rng.standard_normal(V)
    if shape == "threads over":  # all but one of K threads' columns hold larger values than its best
        row = np.where((i // 4) % 256 < K, 20 + small, np.minimum(small, 3))
        return np.where((i // 4) % 256 == K - 1, 5.0 + 0.01 * small, row)
    if shape == "lanes over":
        row = np.where((i // 4) % 32 < K, 20 + small, np.minimum(small, 3))
        return np.where((i // 4) % 32 == K - 1, 5.0 + 0.01 * small, row)
    return {"equal": np.zeros(V), "rising": i * 1e-3, "falling": -i * 1e-3, "two values": (i % 7 == 3) * 1.0,
            "few values": np.floor(small * 2), "columns": np.where((i // 4) % 256 == 17, 10 + rng.random(V), small),
            "blocks": np.where(i // 1024 == (V // 1024) // 2, 10 + small, small),
            "tail": np.where(i >= V - K, 9.0 + i * 1e-5, small), "head": np.where(i < 3, 9.0, small),
            "normal": small}[shape]


SHAPES = ["equal", "rising", "falling", "two values", "few values", "columns", "blocks", "threads over", "lanes over",
          "tail", "head"]


@pytest.mark.parametrize("V", [600, 4096, 40000, 140001])
@pytest.mark.parametrize("K", [1, 20, 32])
@pytest.mark.parametrize("shape", SHAPES)
def test_alternatives_wherever_they_stand(cuda_rt, V, K, shape):
    """Rows whose largest logits sit where a split of the row over threads and
    CTAs could lose them: ties, runs, one thread's columns, one block."""
    rng = np.random.default_rng(V + K)
    row = pattern(shape, V, K, rng)
    check(cuda_rt, np.stack([row, row[::-1], rng.standard_normal(V)]), [0, V - 1, V // 2], K)


@pytest.mark.parametrize("R, V", [(2400, 1025), (2400, 2050), (2401, 4096), (2402, 8191), (2368, 12289), (2400, 30001),
                                  (900, 5000), (1000, 20001),
                                  (10000, 258), (5000, 500)])
@pytest.mark.parametrize("K", [0, 3, 8, 20, 32])
def test_alternatives_of_many_rows(cuda_rt, R, V, K):
    """The same patterns in batches, whose rows other teams of threads take:
    warps, CTAs of 128 or 256 threads, groups of lanes."""
    rng = np.random.default_rng(R + V + K)
    rows = [bf16(pattern(s, V, max(K, 1), rng)) for s in SHAPES + ["normal"] * 5]
    mask = np.where(rng.random(V) < 0.97, -np.inf, rows[-1])
    rows += [mask, np.full(V, -np.inf), np.where(np.arange(V) == V // 2, np.nan, rows[-1]),
             np.where(np.arange(V) == V - 1, np.inf, rows[-1]), np.full(V, LOW)]
    x = np.array(rows, np.float32)
    n = len(x)
    ids = rng.integers(-1, V, n)
    big, all_ids = np.tile(x, (R // n + 1, 1))[:R], np.tile(ids, R // n + 1)[:R]
    got, want = forward(cuda_rt, big, all_ids, K, kind=K % 2, pad=K % 3), logprobs(x, ids, K)
    lp, ent = logprobs_tolerance(want, V)
    tol = {"logp": lp(want["logp"]), "entropy": ent, "top_logp": lp(want["top_logp"])}
    for r0 in range(0, R, n):
        m = min(n, R - r0)
        assert np.array_equal(got["top_ids"][r0:r0 + m], want["top_ids"][:m])
        for k in tol:
            near(got[k][r0:r0 + m], want[k][:m], tol[k][:m], k)


def test_offsets_beyond_32_bits(cuda_rt):
    """Rows 1.1 * 10^9 logits apart: the third starts past 2^31 values."""
    rt = cuda_rt
    ld, V = 1100000003, 3001
    p = ctypes.c_void_p()
    assert rt.lib.tp_alloc((2 * ld + V) * 4, ctypes.byref(p)) == 0
    x = (np.random.default_rng(3).standard_normal((3, V)) * 3).astype(np.float32)
    for r in range(3):
        assert rt.lib.tp_memcpy_h2d(p.value + 4 * ld * r, x[r].ctypes.data_as(ctypes.c_void_p), 4 * V) == 0
    I, L, S, E = (Buf(rt, a) for a in (np.array([5, 0, V - 1], np.int32), np.zeros(3, np.float32),
                                       np.zeros((3, 2), np.float32), np.zeros(3, np.float32)))
    T, TL, G = Buf(rt, np.zeros((3, 4), np.int32)), Buf(rt, np.zeros((3, 4), np.float32)), Buf(rt, np.ones(3, np.float32))
    assert rt.lib.tpk_token_logprobs(p.value, ld, I.ptr, 1, 3, V, 4, L.ptr, E.ptr, S.ptr, T.ptr, TL.ptr) == 0
    want = logprobs(x, [5, 0, V - 1], 4)
    lp, _ = logprobs_tolerance(want, V)
    near(L.read(), want["logp"], lp(want["logp"]), "logp")
    assert np.array_equal(T.read(), want["top_ids"])
    assert rt.lib.tpk_token_logprobs_backward(p.value, ld, I.ptr, 1, S.ptr, E.ptr, G.ptr, None, 3, V, p.value, ld) == 0
    d, tol = logprobs_grad(x, [5, 0, V - 1], None, None, np.ones(3), None)
    for r in range(3):
        got = np.empty(V, np.float32)
        assert rt.lib.tp_memcpy_d2h(got.ctypes.data_as(ctypes.c_void_p), p.value + 4 * ld * r, 4 * V) == 0
        near(got, d[r], tol[r], "dlogits")
    assert rt.lib.tp_free(p.value) == 0


def test_many_rows(cuda_rt):
    rng = np.random.default_rng(5)
    check(cuda_rt, rng.standard_normal((5003, 129)) * 3, rng.integers(0, 129, 5003), 4)
    check(cuda_rt, bf16(rng.standard_normal((1501, 2050)) * 3), rng.integers(0, 2050, 1501), 11, pad=1)


@pytest.mark.parametrize("R", [4740, 9480, 20001])
@pytest.mark.parametrize("V", [1, 2, 3, 10, 31, 64, 65, 127, 256, 264, 265, 400, 528, 529])
def test_many_short_rows(cuda_rt, R, V):
    """Rows enough for several to a warp: masks, equal logits, odd values."""
    rng = np.random.default_rng(R + V)
    x = bf16(rng.standard_normal((R, V)) * 2)
    x[rng.random((R, V)) < 0.3] = -np.inf
    x[::7] = 0.5
    x[::11] = -np.inf
    x[3::101, 0] = np.nan
    x[4::103, V - 1] = np.inf
    x[5::107] = LOW
    x = np.concatenate([x[:400], x[-400:]])  # the oracle's rows
    ids = rng.integers(-1, V, 800)
    reps = (R + 799) // 800
    big, K = np.tile(x, (reps, 1))[:R], min(V, 1 + V % 6 if R % 2 else 20)
    got = forward(cuda_rt, big, np.tile(ids, reps)[:R], K, kind=R % 2, pad=V % 4)
    want = logprobs(x, ids, K)
    lp, ent = logprobs_tolerance(want, V)
    tol = {"logp": lp(want["logp"]), "entropy": ent, "top_logp": lp(want["top_logp"])}
    for r0 in range(0, R, 800):
        n = min(800, R - r0)
        assert np.array_equal(got["top_ids"][r0:r0 + n], want["top_ids"][:n])
        for k in tol:
            near(got[k][r0:r0 + n], want[k][:n], tol[k][:n], k)


def test_outputs_left_out(cuda_rt):
    rt = cuda_rt
    x = np.random.default_rng(1).standard_normal((5, 3001)).astype(np.float32)
    X, E = Buf(rt, x), Buf(rt, np.zeros(5, np.float32))
    T, TL = Buf(rt, np.zeros(15, np.int32)), Buf(rt, np.zeros(15, np.float32))
    want = logprobs(x, [0] * 5, 3)
    lp, ent = logprobs_tolerance(want, 3001)
    assert rt.lib.tpk_token_logprobs(X.ptr, 3001, None, 0, 5, 3001, 3, None, E.ptr, None, T.ptr, TL.ptr) == 0
    near(E.read(), want["entropy"], ent, "entropy")
    assert np.array_equal(T.read().reshape(5, 3), want["top_ids"])
    assert rt.lib.tpk_token_logprobs(X.ptr, 3001, None, 0, 5, 3001, 0, None, None, None, None, None) == 0
    rt.synchronize()


def test_equal_inputs_equal_bits(cuda_rt):
    rng = np.random.default_rng(9)
    for R, V in ((1, 131072), (64, 50021), (1000, 300)):
        x, ids = bf16(rng.standard_normal((R, V)) * 4), rng.integers(0, V, R)
        a, b = forward(cuda_rt, x, ids, 20), forward(cuda_rt, x, ids, 20)
        for k in a:
            assert np.array_equal(a[k], b[k], equal_nan=True), k


# ---- gradient ---------------------------------------------------------------------------------------

def backward(rt, x, ids, stats, entropy, dlogp, dentropy, kind=1, pad=0, pad_d=0, offset=0, in_place=False):
    R, V = x.shape
    whole = np.full((R, V + pad), 7e37, np.float32)
    whole[:, :V] = x
    X = Buf(rt, whole, offset)
    I = Buf(rt, ids_array(ids, kind)) if ids is not None else None
    S, E = Buf(rt, stats.astype(np.float32)), Buf(rt, entropy.astype(np.float32))
    g1 = Buf(rt, dlogp.astype(np.float32)) if dlogp is not None else None
    g2 = Buf(rt, dentropy.astype(np.float32)) if dentropy is not None else None
    D = X if in_place else Buf(rt, np.full((R, V + pad_d), GUARD, np.float32))
    ldd = V + (pad if in_place else pad_d)
    p = lambda b: b.ptr if b is not None else None  # noqa: E731
    assert rt.lib.tpk_token_logprobs_backward(X.ptr, V + pad, p(I), kind, S.ptr, E.ptr, p(g1), p(g2), R, V, D.ptr,
                                              ldd) == 0, rt.lib.tp_last_error()
    rt.synchronize()
    got = D.read().reshape(R, ldd)
    assert np.all(got[:, V:] == (np.float32(7e37) if in_place else GUARD))
    if not in_place:
        assert np.array_equal(X.read(), whole, equal_nan=True)
        X.free()
    for b in (D, S, E, I, g1, g2):
        if b is not None:
            b.free()
    return got[:, :V]


def check_grad(rt, x, ids, dlogp, dentropy, **how):
    x = np.ascontiguousarray(x, np.float32)
    o = logprobs(x, ids if ids is not None else [0] * len(x), 0)
    got = backward(rt, x, ids, o["stats"], o["entropy"], dlogp, dentropy, **how)
    want, tol = logprobs_grad(x, ids, o["stats"], o["entropy"], dlogp, dentropy)
    near(got, want, tol, "dlogits")
    return got


@pytest.mark.parametrize("R, V", SIZES)
@pytest.mark.parametrize("with_entropy", [False, True])
def test_gradient_sizes(cuda_rt, R, V, with_entropy):
    rng = np.random.default_rng(R + V)
    ids = np.where(rng.random(R) < 0.2, -100, rng.integers(0, V, R))
    check_grad(cuda_rt, rng.standard_normal((R, V)) * 4, ids, rng.standard_normal(R),
               rng.standard_normal(R) if with_entropy else None, kind=V % 2, pad=R % 4, pad_d=V % 3,
               offset=4 * (V % 4), in_place=(R + V) % 5 == 0)


@pytest.mark.parametrize("V", [5, 400, 3000, 20001])
def test_gradient_special_rows(cuda_rt, V):
    rng = np.random.default_rng(V)
    base = rng.standard_normal(V) * 3
    nan, inf, part = base.copy(), base.copy(), np.where(rng.random(V) < 0.5, -np.inf, base)
    nan[1], inf[V - 1], part[2] = np.nan, np.inf, 0.5
    low = np.where(rng.random(V) < 0.5, LOW, base)
    none = np.full(V, -np.inf)
    x = np.array([base, none, nan, inf, part, part, low, nan, base, base, base + 1e4, none], np.float32)
    ids = np.array([0, 0, 0, 0, 2, 0 if np.isneginf(part[0]) else 1, 0, -1, V, 2 ** 24, V - 1, -5])
    for g2 in (None, rng.standard_normal(len(x)), np.zeros(len(x))):
        check_grad(cuda_rt, x, ids, rng.standard_normal(len(x)), g2, kind=0)
        check_grad(cuda_rt, x, ids, np.zeros(len(x)), g2)
        check_grad(cuda_rt, x, None, None, g2)


def test_gradient_in_place_matches(cuda_rt):
    rng = np.random.default_rng(3)
    for V in (64, 1000, 4097):
        x, ids = (rng.standard_normal((9, V)) * 3).astype(np.float32), rng.integers(0, V, 9)
        g1, g2 = rng.standard_normal(9), rng.standard_normal(9)
        a = check_grad(cuda_rt, x, ids, g1, g2)
        assert np.array_equal(a, check_grad(cuda_rt, x, ids, g1, g2, in_place=True))


def test_gradient_against_differences(cuda_rt):
    """d(sum of g1 logp + g2 H) along random directions, by central differences
    of the 64-bit forward: error h^2 / 6 times the third derivative, which for
    a softmax of unit-scale logits is below 10 per unit direction, and 1e-16 /
    h of cancellation; h = 1e-4 gives 2e-8 and 1e-11."""
    rng = np.random.default_rng(11)
    R, V, h = 4, 37, 1e-4
    x, ids = rng.standard_normal((R, V)).astype(np.float32), rng.integers(0, V, R)
    g1, g2 = rng.standard_normal(R), rng.standard_normal(R)
    d = check_grad(cuda_rt, x, ids, g1, g2).astype(np.float64)
    f32 = np.float32
    for _ in range(8):
        u = rng.standard_normal((R, V))
        u /= np.linalg.norm(u)

        def loss(z):
            o = logprobs(z, ids, 0)
            return float((f32(g1).astype(np.float64) * o["logp"] + f32(g2).astype(np.float64) * o["entropy"]).sum())

        diff = (loss(x + h * u) - loss(x - h * u)) / (2 * h)
        assert abs(diff - (d * u).sum()) < 2e-6  # the gradient itself is float32: 37 * 4 terms of 1e-7 at most


# ---- handles ----------------------------------------------------------------------------------------

def test_runtime_surface(cuda_rt):
    rt = cuda_rt
    rng = np.random.default_rng(21)
    x = (rng.standard_normal((2, 3, 77)) * 3).astype(np.float32)
    ids = rng.integers(0, 77, (2, 3))
    X = rt.tensorFromData(x, [2, 3, 77], "float32")
    I = rt.tensorFromData(ids.astype(np.float32), [2, 3], "int64")
    before = rt.memoryAllocated()
    lp, en, st, ti, tl = rt.tokenLogprobs(X["id"], I["id"], 4)
    assert lp["shape"] == en["shape"] == [2, 3] and st["shape"] == [2, 3, 2]
    assert ti["shape"] == tl["shape"] == [2, 3, 4] and ti["dtype"] == "int64"
    want = logprobs(x.reshape(6, 77), ids.ravel(), 4)
    tol, ent = logprobs_tolerance(want, 77)
    near(rt.toNumpy(lp["id"]), want["logp"], tol(want["logp"]), "logp")
    near(rt.toNumpy(en["id"]), want["entropy"], ent, "entropy")
    assert rt.toList(ti["id"]) == want["top_ids"].ravel().tolist()
    near(rt.toNumpy(tl["id"]).reshape(6, 4), want["top_logp"], tol(want["top_logp"]), "top logp")
    g1 = rt.tensorFromData(rng.standard_normal(6).astype(np.float32), [2, 3], "float32")
    d = rt.tokenLogprobsBackward(g1["id"], None, X["id"], I["id"], st["id"], en["id"])
    assert d["shape"] == [2, 3, 77]
    dw, dt = logprobs_grad(x.reshape(6, 77), ids.ravel(), None, None, rt.toNumpy(g1["id"]), None)
    near(rt.toNumpy(d["id"]).reshape(6, 77), dw, dt, "dlogits")
    # ids of int32 storage: the row's best token
    best = rt.argmax(X["id"])
    three = rt.tokenLogprobs(X["id"], best["id"])
    assert len(three) == 3
    near(rt.toNumpy(three[0]["id"]), want["top_logp"][:, 0], tol(want["top_logp"][:, 0]), "best")
    for h in (lp, en, st, ti, tl, g1, d, best, *three):
        rt.destroy(h["id"])
    assert rt.memoryAllocated() == before


def test_runtime_refusals(cuda_rt):
    rt = cuda_rt
    X = rt.zeros([4, 10], "float32")["id"]
    ids = rt.zeros([4], "int64")["id"]
    lp, en, st = rt.tokenLogprobs(X, ids)
    before = rt.memoryAllocated()
    for call in (lambda: rt.tokenLogprobs(X, rt.zeros([5], "int64")["id"]), lambda: rt.tokenLogprobs(X, ids, 11),
                 lambda: rt.tokenLogprobs(X, ids, -1), lambda: rt.tokenLogprobs(rt.zeros([4, 0], "float32")["id"], ids),
                 lambda: rt.tokenLogprobs(rt.argmax(X)["id"], ids), lambda: rt.tokenLogprobs(12345678, ids),
                 lambda: rt.tokenLogprobsBackward(ids, None, X, ids, en["id"], en["id"]),
                 lambda: rt.tokenLogprobsBackward(X, None, X, ids, st["id"], en["id"]),
                 lambda: rt.tokenLogprobsBackward(rt.argmax(X)["id"], None, X, ids, st["id"], en["id"])):
        with pytest.raises(RuntimeError):
            call()
    assert rt.memoryAllocated() - before < 4096  # the operands made above; no outputs
    empty = rt.tokenLogprobs(rt.zeros([0, 10], "float32")["id"], rt.zeros([0], "int64")["id"], 2)
    assert [h["shape"] for h in empty] == [[0], [0], [0, 2], [0, 2], [0, 2]]
