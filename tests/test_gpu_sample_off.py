"""The sampler with parameters that are no numbers."""
import numpy as np
import pytest

from test_gpu_sample import _run

pytestmark = pytest.mark.gpu


def test_parameters_that_are_no_numbers(accel):
    """A filter is on where its condition holds; it does not for NaN.  A temperature that is not above 0 is greedy."""
    rng = np.random.default_rng(6)
    rows, v = 40, 3000
    x = rng.standard_normal((rows, v)).astype(np.float32)
    u = rng.random(rows, dtype=np.float32)
    nan = np.full(rows, np.nan, np.float32)
    free = _run(accel, x, u)
    for k in ({"p": nan}, {"m": nan}, {"p": nan, "m": nan}):
        got = _run(accel, x, u, **k)
        assert np.array_equal(got[0], free[0]) and np.array_equal(got[1], free[1]), k
    assert np.array_equal(_run(accel, x, u, T=nan)[0], x.argmax(1))
