"""The gradient of short rows of logits on both sides of the sizes at which
another group of lanes takes a row."""
import numpy as np
import pytest

from test_gpu_token_logprobs import backward
from token_oracle import logprobs, logprobs_grad

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [1, 31, 125, 126, 252, 253, 254, 256, 300, 399, 400, 401])
@pytest.mark.parametrize("R", [9, 16575, 16577])
def test_gradient_by_either_group(cuda_rt, R, V):
    rng = np.random.default_rng(V + R)
    n = min(R, 97)  # the oracle's rows, over and over
    x = (rng.standard_normal((n, V)) * 3).astype(np.float32)
    ids, g1, g2 = np.where(rng.random(n) < 0.3, -1, rng.integers(0, V, n)), rng.standard_normal(n), rng.standard_normal(n)
    g2[rng.random(n) < 0.5] = 0.0  # with an ignored id: a row of zeros
    o = logprobs(x, ids, 0)
    want, tol = logprobs_grad(x, ids, o["stats"], o["entropy"], g1, g2)
    reps = (R + n - 1) // n
    many = lambda a: np.tile(a, (reps,) + (1,) * (a.ndim - 1))[:R]  # noqa: E731
    got = backward(cuda_rt, many(x), many(ids), many(o["stats"]), many(o["entropy"]), many(g1), many(g2), pad=V % 3,
                   pad_d=(V // 2) % 3)
    assert np.all(np.abs(got - many(want)) <= many(tol))
    assert np.all(got[many((ids < 0) & (g2 == 0))] == 0)
