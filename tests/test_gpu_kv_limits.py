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


def _apart(rng, page, dim, length, big, small, at):
    """One sequence whose blocks `at` hold values of scale `big` behind scores about 2^-43 of the others' exponentials; the others' scale is
    `small`.  Channel 0 of every key is +-127, which one large channel of the query turns into the two levels of scores."""
    cache = _random_cache(rng, page, 1, dim, length)
    table = R.tables(rng, cache.pages, page, [length])
    t = np.arange(R.BLOCK)
    for b in range(-(-length // R.BLOCK)):
        where = (table[0][b * R.BLOCK // page], 0, b % (page // R.BLOCK))
        cache.k[where][R.k_byte(cache.dim64, t, 0 * t)] = -127 if b in at else 127
        cache.ks[where] = np.float32(0.01)
        cache.vs[where] = np.float32(big if b in at else small)
        if cache.vs[where] == 0:
            cache.v[where] = 0
    return cache, table


def _weighed(cache, table, length, new, q, scale):
    """Per row and head: the largest probability times |value|, what an error is measured by."""
    k = cache.tokens("k", table[0], 0, length).astype(np.float64)
    v = np.abs(cache.tokens("v", table[0], 0, length).astype(np.float64)).max(1)
    out = np.zeros(q.shape[:2])
    for j in range(new):
        pos = length - new + j
        for h in range(q.shape[1]):
            sc = k[:pos + 1] @ q[j, h].astype(np.float64) * scale
            p = np.exp(sc - sc.max())
            out[j, h] = (p * v[:pos + 1]).sum() / p.sum()
    return out


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("new", [1, 3, 120])
@pytest.mark.parametrize("big,small", [(0.01, 0.01), (1e4, 0.01), (1e7, 1e-5), (1.0, 1e-20)])
def test_value_scales_far_apart(accel, pkg, ty, new, big, small):
    """Blocks of large values whose probabilities are tiny, or that a row does not see, leave the others their bits."""
    rng = np.random.default_rng(new)
    dim, length, heads, scale = 64, 900, 2, 0.125
    cache, table = _apart(rng, 64, dim, length, big, small, (3, 11, 28))
    q, _ = _queries(rng, "f32", new, heads, dim, 0.3)
    q[:, :, 0] = 94.0                             # +-127 * 0.01 * 94 / 8 = +-14.9: exponentials 2^-43 apart
    raw = q if ty == "f32" else R.bf16(q)
    q = q if ty == "f32" else R.from_bf16(raw)
    want = R.attend(cache, table, [length], [new], q, scale)
    got = _attention(accel, pkg, cache, table, [length], [new], raw, ty, scale)
    err = np.abs(got - want).max(2) / _weighed(cache, table, length, new, q, scale)
    print(f"{ty} {new} rows, {big:g} beside {small:g}: {err.max():.1e}")
    assert err.max() <= TOL[ty]


@pytest.mark.parametrize("first,then", [(1.0, 1e-28), (1e-28, 1.0), (1e12, 1e-22), (0.0, 1.0), (1.0, 0.0)])
@pytest.mark.parametrize("new", [1, 70])
def test_value_scales_change_along_a_long_context(accel, pkg, new, first, then):
    """Whole sequences (many of them: nothing is split) of more blocks than one look-up holds, whose values change size behind the first."""
    rng = np.random.default_rng(4)
    dim, length, nseq, scale = 64, 9000, 600, 0.125
    cache, one = _apart(rng, 256, dim, length, then, first, range(256, 300))
    q, raw = _queries(rng, "f32", new, 1, dim, 0.3)
    want = R.attend(cache, one, [length], [new], q, scale)
    table = np.repeat(one, nseq, 0)               # (attention only reads: all of them are one sequence)
    got = _attention(accel, pkg, cache, table, [length] * nseq, [new] * nseq, np.tile(raw, (nseq, 1, 1)), "f32", scale)
    by = _weighed(cache, one, length, new, q, scale)
    assert np.array_equal(got.reshape(nseq, new, 1, dim), np.broadcast_to(got[:new], (nseq, new, 1, dim)))
    assert (np.abs(got[:new] - want).max(2) / by).max() <= TOL["f32"]


def test_scores_below_every_usual_one(accel, pkg):
    """All of a row's scores around -1e32: the largest still takes everything."""
    rng = np.random.default_rng(8)
    dim, length = 64, 200
    cache = _random_cache(rng, 32, 1, dim, length)
    cache.ks[:] = 1e15
    table = R.tables(rng, cache.pages, 32, [length])
    t = np.arange(R.BLOCK)
    for b in range(-(-length // R.BLOCK)):
        block = cache.k[table[0][b], 0, 0]
        block[:] = 0
        block[R.k_byte(64, t, 0 * t)] = rng.integers(-127, 100, R.BLOCK)     # scores of +-127e31 ...
        block[R.k_byte(64, t, 0 * t + 1)] = -127                             # ... less 254e31
    cache.k[table[0][0], 0, 0][R.k_byte(64, 0, 0)] = 127                     # the first token's is the largest
    first = cache.tokens("v", table[0], 0, 1)[0]
    for new in (1, 90):
        q = np.zeros((new, 1, dim), np.float32)
        q[:, :, 0], q[:, :, 1] = 1e16, 2e16
        got = _attention(accel, pkg, cache, table, [length], [new], q, "f32", 1.0)
        assert np.abs(got - first).max() <= TOL["f32"] * np.abs(first).max(), new


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("size", [1e6, 1e10, 1e32])
@pytest.mark.parametrize("dim,sign", [(64, 1), (64, -1), (128, 1), (256, -1)])
def test_scores_of_every_size(accel, pkg, ty, size, dim, sign):
    """Scores of which fp32 keeps no fraction, of both signs: one token stands out for every row and takes everything."""
    rng = np.random.default_rng(9)
    length, best = 300, 77
    cache = _random_cache(rng, 32, 1, dim, length)
    cache.ks[:], cache.vs[:] = 0.5, 0.01
    table = R.tables(rng, cache.pages, 32, [length])
    t = np.arange(R.BLOCK)
    for b in range(-(-length // R.BLOCK)):
        block = cache.k[table[0][b], 0, 0]
        block[:] = 0
        block[R.k_byte(cache.dim64, t, 0 * t)] = rng.integers(-100, 100, R.BLOCK)
    cache.k[table[0][best // 32], 0, 0][R.k_byte(cache.dim64, best % 32, 0)] = 127 * sign
    want = cache.tokens("v", table[0], 0, best + 1)[best]
    for new in (1, 200):
        q = np.zeros((new, 1, dim), np.float32)
        q[:, :, 0] = size / 64.0
        raw = q if ty == "f32" else R.bf16(q)
        got = _attention(accel, pkg, cache, table, [length], [new], raw, ty, float(sign))
        seen = np.arange(length - new, length) >= best       # (earlier rows of the chunk: some other token)
        assert np.isfinite(got).all()
        assert np.abs(got[seen] - want).max() <= TOL[ty] * np.abs(want).max(), new


@pytest.mark.parametrize("ty", ["f32", "bf16"])
def test_nothing_is_stored_outside_the_cache(accel, pkg, ty):
    """Page numbers that name no page: their tokens are left out, every other byte of the cache, of the read-back and of the queries is as it
    was or as the definition says."""
    rng = np.random.default_rng(12)
    kv, heads, dim, page, pages = 2, 4, 64, 32, 6
    lens, new = [70, 40, 33, 65], [70, 40, 2, 1]
    table = np.array([[4, -1, 1], [-7, 5, -1], [6, 3, 0], [99, 2 ** 31 - 1, -2 ** 31]], np.int32)
    rows = sum(new)
    cache = R.Cache(pages, page, kv, dim, seed=2)
    cache.ks[:], cache.vs[:] = 0.01, 0.02
    want = [x.copy() for x in (cache.k, cache.v, cache.ks, cache.vs)]
    k, raw_k = _queries(rng, ty, rows, kv, dim)
    v, raw_v = _queries(rng, ty, rows, kv, dim)
    # the definition, token by token of the pages that exist: a sequence's own table with spare pages behind the cache for the others
    big = R.Cache(pages + 12, page, kv, dim, seed=2)
    for a, b in ((big.k, cache.k), (big.v, cache.v), (big.ks, cache.ks), (big.vs, cache.vs)):
        a[:] = 0
        a[:pages] = b
    own = np.where((table >= 0) & (table < pages), table, pages + np.arange(12).reshape(4, 3)).astype(np.int32)
    R.append(big, own, [a - b for a, b in zip(lens, new)], new, k, v)
    want = [x[:pages] for x in (big.k, big.v, big.ks, big.vs)]
    guard = 4096
    with R.Dev(accel) as dev:
        d = R.OnDevice(pkg, dev, cache)
        held, planes = [], []
        for x in (cache.k, cache.v, cache.ks, cache.vs):     # planes with guards on both sides
            raw = np.concatenate([np.full(guard, 0xA5, np.uint8), np.frombuffer(x.tobytes(), np.uint8), np.full(guard, 0xA5, np.uint8)])
            held.append((dev.put(raw), raw.size))
            planes.append(held[-1][0] + guard)
        handle = pkg.KvCache(pages, page, kv, dim, *planes)
        batch = d.batch(table, lens, new)
        accel.kv_append_dev(handle, batch, dev.put(raw_k), dev.put(raw_v), dtype=_dtype(pkg, ty))
        for (p, n), w in zip(held, want):
            got = dev.get(p, n, np.uint8)
            assert (got[:guard] == 0xA5).all() and (got[n - guard:] == 0xA5).all()
            body = np.frombuffer(got[guard:n - guard].tobytes(), w.dtype).reshape(w.shape)
            same = (body == w) | ((body != body) & (w != w))
            assert same.all(), np.argwhere(~same)[:4]


def _rows_of(x, ranges):
    return np.concatenate([x[a:b] for a, b in ranges])


@pytest.mark.parametrize("how,new", [(h, n) for h in ("max_len", "max_rows", "rows") for n in ([1, 1], [5, 3], [70, 40]) if h != "max_rows" or max(n) > 1])
def test_rows_beyond_the_call_are_left_out(accel, pkg, new, how):
    """Arrays that name more tokens or rows than the call's sizes: the rows within them are at their own positions, the others are neither stored
    nor attended to, and what the sequences held stays."""
    rng = np.random.default_rng(sum(new))
    kv, heads, dim, page = 2, 4, 64, 32
    old = [100, 37]
    lens = [a + b for a, b in zip(old, new)]
    rows = sum(new)
    cache = R.Cache(14, page, kv, dim, seed=5)
    table = R.tables(rng, 14, page, lens)
    R.append(cache, table, [0, 0], old, *(rng.standard_normal((sum(old), kv, dim)).astype(np.float32) for _ in range(2)))
    k, v = (rng.standard_normal((rows, kv, dim)).astype(np.float32) for _ in range(2))
    q, _ = _queries(rng, "f32", rows, heads, dim)
    # what the call's sizes leave of each sequence's rows
    left = {"max_len": [max(0, new[0] - 1), new[1]], "max_rows": [min(n, max(new) - 2) for n in new], "rows": [new[0], new[1] - 1]}[how]
    limits = {"max_len": dict(max_len=lens[0] - 1), "max_rows": {}, "rows": {}}[how]
    rope = R.rope_table(max(lens), dim)
    ranges = [(0, left[0]), (new[0], new[0] + left[1])]
    held = [a + b for a, b in zip(old, left)]
    pos = np.concatenate([np.arange(a, b) for a, b in zip(old, held)])
    with R.Dev(accel) as dev:
        d = R.OnDevice(pkg, dev, cache)
        b = d.batch(table, lens, new, always_row0=how != "max_len" or max(new) > 1, **limits)
        if how == "max_rows":
            b.max_rows = max(new) - 2
        elif how == "rows":
            b.rows -= 1
            b.max_rows = min(b.max_rows, b.rows)
        out, back = dev.put(np.full(q.shape, 7, np.float32)), [dev.put(np.full(k.shape, 7, np.float32)) for _ in range(2)]
        accel.kv_append_dev(d.handle, b, dev.put(k), dev.put(v), rope=pkg.Rope(dev.put(rope), rope.shape[0], dim))
        R.append(cache, table, old, left, R.rotate(_rows_of(k, ranges), rope, pos, dim, False), _rows_of(v, ranges))
        got = d.planes()
        for a, w in zip(got[2:], (cache.ks, cache.vs)):
            assert np.array_equal(a, w, equal_nan=True)
        host = R.Cache(1, page, kv, dim)
        host.k, host.v, host.ks, host.vs = got
        for s, n in enumerate(held):
            for h in range(kv):
                for w in "kv":
                    assert np.array_equal(host.tokens(w, table[s], h, n), cache.tokens(w, table[s], h, n)), (s, h, w)
        accel.attn_dev(d.handle, b, dev.put(q), heads, dim ** -0.5, out)
        accel.kv_read_dev(d.handle, b, *back)
        y, back = dev.get(out, q.shape), [dev.get(p, k.shape) for p in back]
    want = R.attend(cache, table, held, left, _rows_of(q, ranges), dim ** -0.5)
    assert np.abs(_rows_of(y, ranges) - want).max(initial=0) <= TOL["f32"] * 5
    beyond = np.setdiff1d(np.arange(rows), np.concatenate([np.arange(*r) for r in ranges]))
    assert (y[beyond] == 7).all()
    for x, w in zip(back, "kv"):
        assert (x[beyond] == 7).all()
        r = 0
        for s, (o, n) in enumerate(zip(old, held)):
            for h in range(kv):
                assert np.array_equal(x[ranges[s][0]:ranges[s][1], h], cache.tokens(w, table[s], h, n)[o:])


@pytest.mark.parametrize("ty,dim,window,nseq,kv,heads", [("bf16", 256, 1024, 100, 8, 8), ("f32", 128, 900, 150, 8, 8), ("f32", 64, 700, 240, 8, 8), ("bf16", 128, 2040, 112, 8, 8),
                                                 ("f32", 192, 1000, 80, 8, 8), ("f32", 64, 700, 300, 8, 8), ("bf16", 128, 1000, 260, 8, 8), ("f32", 128, 500, 240, 4, 68)])
def test_many_windows(accel, pkg, ty, dim, window, nseq, kv, heads):
    """Sequences that a window makes alike, in the numbers around a second round of workgroups."""
    rng = np.random.default_rng(dim + nseq)
    page, length = 32, 2500
    cache = _random_cache(rng, page, kv, dim, length)
    one = R.tables(rng, cache.pages, page, [length])
    lens = [int(x) for x in rng.integers(1, length + 1, nseq)]
    q, raw = _queries(rng, ty, nseq, heads, dim)
    table = np.repeat(one, nseq, 0)
    want = R.attend(cache, table, lens, [1] * nseq, q, dim ** -0.5, window)
    got = _attention(accel, pkg, cache, table, lens, [1] * nseq, raw, ty, dim ** -0.5, window=window)
    assert np.abs(got - want).max() <= TOL[ty] * 128 * 0.02


@pytest.mark.parametrize("ty,dim,kv,group,few,chunk", [("f32", 64, 1, 1, [1], 700), ("f32", 128, 2, 4, [1, 1, 0, 1], 300), ("bf16", 64, 1, 8, [1, 5], 200),
                                                       ("f32", 64, 2, 2, [1] * 40, 90), ("bf16", 256, 1, 2, [1, 2, 30], 120)])
def test_split_contexts_of_decode_steps_beside_chunks(accel, pkg, ty, dim, kv, group, few, chunk):
    """Sequences of few rows and chunks of many in one call, at contexts that are split: both launches' sums find their rows again, and a second
    call on the same context finds its own."""
    rng = np.random.default_rng(dim + chunk)
    heads, page, length = kv * group, 64, 3000
    cache = _random_cache(rng, page, kv, dim, 4 * length)
    new = few[:len(few) // 2] + [chunk] + few[len(few) // 2:]
    lens = [length - int(x) for x in rng.integers(0, length // 2, len(new))]
    pages = rng.permutation(cache.pages)
    table = np.stack([np.roll(pages, i)[:-(-length // page)] for i in range(len(new))]).astype(np.int32)   # (they may share pages: nothing is stored)
    q, raw = _queries(rng, ty, sum(new), heads, dim)
    want = R.attend(cache, table, lens, new, q, dim ** -0.5)
    for again in range(2):
        got = _attention(accel, pkg, cache, table, lens, new, raw, ty, dim ** -0.5, always_row0=True)
        assert np.abs(got - want).max() <= TOL[ty] * 128 * 0.02
        first = got if again == 0 else first
    assert np.array_equal(first, got)
