"""Log-probabilities of rows with one large logit and a flat tail far below it.

Each tail term is less than half a step of a sum that holds the maximum's 1, so
a thread that met the maximum must not add the rest of its logits one by one.
The tolerance counts the roundings of sums that do not: a batch's 16
exponentials among themselves (4 levels), the batches with a compensation
(2 in all), 5 exchanges in a warp, 8 warps, 8 parts of a row; in short rows 9
exponentials in each of a lane's four sums, these (2 levels) and 5 exchanges.
Each is half a step, U, of a sum of at most S.  A tail term is itself off by U (2 y + 4) for y <= 18 below the
maximum, and once more where a thread that did not meet the maximum moves its
sum to it; log S adds 2 U of itself."""
import numpy as np
import pytest

from token_oracle import U, Buf, logprobs

pytestmark = pytest.mark.gpu


def rows_of(V, rng):
    """Peaks in a thread's first, a middle and its last batch; two flat tails and an uneven one."""
    x = np.empty((4, V), np.float32)
    x[0], x[1], x[2] = -16.7, -17.2, -16.7
    x[3] = rng.uniform(-17.9, -16.3, V)
    for r, at in enumerate((0, 5, V - 1, V // 2)):
        x[r, at] = 0.0
    return x, [0, 5, V - 1, V // 2]


# rows of 8 or 16 lanes, or of a warp, in registers; of a warp; of 128 and 256 threads; of clusters
@pytest.mark.parametrize("R, V, K", [(40000, 258, 0), (40000, 258, 3), (10000, 500, 11), (5, 1000, 0), (5, 1020, 20),
                                     (2400, 8192, 0), (2400, 12288, 3), (900, 50021, 5), (900, 131072, 0),
                                     (2400, 24000, 20), (2400, 50021, 0), (600, 131072, 5), (8, 131072, 0),
                                     (4, 200064, 20), (1, 1 << 22, 0)])
def test_far_tails_are_not_lost(cuda_rt, R, V, K):
    rt = cuda_rt
    x, ids = rows_of(V, np.random.default_rng(V))
    want = logprobs(x, ids, 0)
    n = (R + 3) // 4
    X = Buf(rt, np.tile(x, (n, 1))[:R])
    I = Buf(rt, np.tile(np.array(ids, np.int32), n)[:R])
    lp, en, st = (Buf(rt, np.zeros(s, np.float32)) for s in (R, R, (R, 2)))
    top, tl = Buf(rt, np.zeros(R * K + 1, np.int32)), Buf(rt, np.zeros(R * K + 1, np.float32))
    assert rt.lib.tpk_token_logprobs(X.ptr, V, I.ptr, 1, R, V, K, lp.ptr, en.ptr, st.ptr, top.ptr, tl.ptr) == 0
    rt.synchronize()
    term = 2 * 18 + 4
    sums = 4 + 2 + 5 + 8 + 8 if V > 1024 else 9 + 2 + 5
    tail = -np.expm1(-want["lnS"])  # of S
    tol = U * (sums + 2 * term * tail + 2 * want["lnS"])
    # the entropy's second sum, of the tail alone: its terms' errors, a difference and
    # 36 terms or at most V / 512 batches (of a warp) added in a row, 21 exchanges;
    # what it is divided by, the division, the difference from log S
    ent = tol + U * (want["A"] * (2 * term + 1 + 36 + V / 512 + 21 + sums + 1) + 2 * want["entropy"])
    q = np.arange(R) % 4
    got = {"log sum": st.read()[:, 1], "logp": -lp.read()}
    if K:
        got["top logp"] = -tl.read()[:R * K].reshape(R, K)[:, 0]
    for k, v in got.items():
        over = np.abs(v.astype(np.float64) - want["lnS"][q]) - tol[q]
        r = int(over.argmax())
        assert over[r] <= 0, (k, r, v[r], want["lnS"][r % 4], tol[r % 4])
    over = np.abs(en.read().astype(np.float64) - want["entropy"][q]) - ent[q]
    r = int(over.argmax())
    assert over[r] <= 0, ("entropy", r, en.read()[r], want["entropy"][r % 4], ent[r % 4])
    for b in (X, I, lp, en, st, top, tl):
        b.free()
