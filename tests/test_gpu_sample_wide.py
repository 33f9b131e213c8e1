"""The sampler where the cut's own tokens are too many for a list: top_k of thousands, and logits that are nearly all alike."""
import numpy as np
import pytest

from test_gpu_sample import _check, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("v,gap", [(9000, 0), (33333, 2), (140001, 0)])
def test_large_top_k(accel, v, gap):
    rng = np.random.default_rng(v)
    rows = 8
    x = (rng.standard_normal((rows, v)) * 3).astype(np.float32)
    x[1, rng.integers(0, v, 300)] = -np.inf
    x[2, rng.integers(0, v, 300)] = np.nan
    x[3, ::7] = x[3, 0]                                # the cut among equal logits
    k = np.array([4097, 5000, 6000, v - 3, v // 2, v, 8999, 4500], np.int32)
    p = np.array([1, 1, 0.9, 1, 0.95, 0.5, 1, 0.999], np.float32)
    m = np.array([0, 0.001, 0, 0, 0, 0.2, 0, 0.01], np.float32)
    T = np.array([1, 0.7, 1.5, 3, 1, 1, 0.2, 1], np.float32)
    u = rng.random(rows, dtype=np.float32)
    ids, prob = _run(accel, x, u, T, k, p, m, gap=gap)
    _check(x, ids, prob, u, T, k, p, m)


@pytest.mark.parametrize("spread", [0.0, 1e-6, 1e-3, 0.02])
def test_nearly_equal_logits(accel, spread):
    """One bin of the histogram holds all or most of a row."""
    rng = np.random.default_rng(int(spread * 1e6) + 1)
    rows, v = 6, 60000
    x = (5 + spread * rng.standard_normal((rows, v))).astype(np.float32)
    x[4:, ::3] -= 2
    k = np.array([0, 0, 7000, 20000, 0, 30000], np.int32)
    p = np.array([0.3, 0.9, 1, 0.5, 0.7, 0.99], np.float32)
    u = rng.random(rows, dtype=np.float32)
    ids, prob = _run(accel, x, u, None, k, p)
    _check(x, ids, prob, u, None, k, p, None)
