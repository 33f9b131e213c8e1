"""The cache and the attention where a call's arguments, arrays or values are at the end of what they may be."""
import numpy as np
import pytest

import kv_ref as R

pytestmark = pytest.mark.gpu
TOL = {"f32": 2e-5, "bf16": 2.0 ** -8}   # as the tests of attention derive them


def _dtype(pkg, ty):
    return pkg.DTYPE_F32 if ty == "f32" else pkg.DTYPE_BF16


def _queries(rng, ty, rows, heads, dim, size=1.0):
    q = (rng.standard_normal((rows, heads, dim)) * size).astype(np.float32)
    raw = q if ty == "f32" else R.bf16(q)
    return (q if ty == "f32" else R.from_bf16(raw)), raw


def _attention(accel, pkg, cache, table, lens, new, raw, ty, scale, window=0, **batch):
    """The call's result as fp32, rows that it leaves out as 7."""
    with R.Dev(accel) as dev:
        d = R.OnDevice(pkg, dev, cache)
        out = dev.put(np.full(raw.shape, 7 if ty == "f32" else R.bf16(np.float32(7))[()], raw.dtype))
        accel.attn_dev(d.handle, d.batch(table, lens, new, **batch), dev.put(raw), raw.shape[1], scale, out, window=window, dtype=_dtype(pkg, ty))
        got = dev.get(out, raw.shape, raw.dtype)
    return got if ty == "f32" else R.from_bf16(got)


def _random_cache(rng, page, kv, dim, tokens):
    cache = R.Cache(-(-tokens // page) + 1, page, kv, dim, seed=int(rng.integers(1 << 30)))
    cache.ks[:], cache.vs[:] = (rng.uniform(0.001, 0.02, cache.ks.shape).astype(np.float32) for _ in range(2))
    return cache


@pytest.mark.parametrize("new", [1, 90])
def test_window_without_an_end(accel, pkg, new):
    """The largest window is no window: the host's split has to know that, too."""
    rng = np.random.default_rng(new)
    kv, heads, dim, length = 1, 2, 64, 1500
    cache = _random_cache(rng, 32, kv, dim, length)
    table = R.tables(rng, cache.pages, 32, [length])
    q, raw = _queries(rng, "f32", new, heads, dim)
    none = _attention(accel, pkg, cache, table, [length], [new], raw, "f32", dim ** -0.5)
    assert np.abs(none - R.attend(cache, table, [length], [new], q, dim ** -0.5)).max() <= TOL["f32"] * 128 * 0.02
    for window in (2 ** 64 - 1, 2 ** 64 - 33, 2 ** 63, 2 ** 31, 2 ** 28, length):
        got = _attention(accel, pkg, cache, table, [length], [new], raw, "f32", dim ** -0.5, window=window)
        # (another split is another order of the same sums)
        assert np.abs(got - none).max() <= 2 * TOL["f32"] * 128 * 0.02, window


@pytest.mark.parametrize("ty,dim,new", [("f32", 64, 1), ("f32", 128, 150), ("bf16", 128, 150), ("f32", 256, 70), ("bf16", 80, 3)])
@pytest.mark.parametrize("scale", [-0.125, -1.0, 0.0])
def test_scale_of_either_sign(accel, pkg, ty, dim, new, scale):
    """Scores of up to hundreds, so that a maximum taken for a minimum leaves every range."""
    rng = np.random.default_rng(dim + new)
    kv, heads, length = 1, 4, 700
    cache = _random_cache(rng, 64, kv, dim, length)
    table = R.tables(rng, cache.pages, 64, [length])
    q, raw = _queries(rng, ty, new, heads, dim)
    got = _attention(accel, pkg, cache, table, [length], [new], raw, ty, scale)
    want = R.attend(cache, table, [length], [new], q, scale)
    # |scores| up to 0.02 * 128 * 3 * sqrt(dim) * |scale|: eight times the tests' 31 at the largest, and so is their rounding
    assert np.abs(got - want).max() <= (8 * TOL[ty] if ty == "f32" else TOL[ty]) * 128 * 0.02
