"""The paged 8-bit key/value cache and the attention over it against numpy: codes, scales, rotated queries and stored values exactly
(the definitions name every rounding), attention against 64 bits.

Tolerance of attention, as a share of the largest stored value (a result is a weighted mean of values).  A probability is off
by the relative error of its exponent times the exponent's size.  Scores here are sums of up to 256 products whose magnitudes add up
to about 0.64 * 3 * sqrt(dim) <= 31 (queries up to 3 sigma heads, scale dim^-1/2), each product exact, rounded when added, at
most 2^-24 of the running sum at each of dim / 32 matrix steps of about 32 internal additions: typically 31 * 2^-22 = 7.4e-6 of error
in the exponent.  fp32: queries and probabilities carry 2^-22 each, which is below that: 2e-5.  bf16: a probability is rounded to 11 bits
(2^-12) and the result to 8 (2^-9 of a result no larger than the largest value): 2^-8."""
import numpy as np
import pytest

import kv_ref as R

pytestmark = pytest.mark.gpu
TOL = {"f32": 2e-5, "bf16": 2.0 ** -8}


def _rows(rng, ty, rows, heads, dim, gap=0, size=1.0):
    """(fp32 values [rows][heads][dim], their array as the call takes it, elements from row to row)"""
    ld = heads * dim + gap
    x = (rng.standard_normal((rows, ld)) * size).astype(np.float32)
    raw = x if ty == "f32" else R.bf16(x)
    x = x if ty == "f32" else R.from_bf16(raw)
    return x[:, :heads * dim].reshape(rows, heads, dim), raw, ld


def _dtype(pkg, ty):
    return pkg.DTYPE_F32 if ty == "f32" else pkg.DTYPE_BF16


def _same(a, b):
    return np.array_equal(np.asarray(a).view(np.uint32), np.asarray(b).view(np.uint32)) or np.array_equal(a, b, equal_nan=True)


def _filled(rng, pages, page, heads, dim, lens, sizes=None):
    """A cache that holds lens[s] tokens of each sequence, and its page table."""
    cache = R.Cache(pages, page, heads, dim, seed=3)
    table = R.tables(rng, pages, page, lens)
    n = sum(lens)
    k, v = (rng.standard_normal((n, heads, dim)).astype(np.float32) for _ in range(2))
    if sizes is not None:
        k, v = k * sizes[0], v * sizes[1]
    R.append(cache, table, [0] * len(lens), lens, k, v)
    return cache, table


APPENDS = [
    # type, dim, rot, interleaved, page, kv heads, q heads, old, new, gap
    ("f32", 128, 128, False, 64, 8, 32, [0], [1], 0),
    ("f32", 128, 128, False, 32, 2, 4, [31, 32, 33, 0, 63, 95], [1, 1, 1, 1, 1, 1], 24),
    ("bf16", 128, 64, True, 64, 2, 2, [5, 0, 64], [1, 1, 1], 8),
    ("f32", 64, 64, True, 96, 3, 9, [0, 17, 95, 200], [64, 3, 2, 130], 0),
    ("bf16", 80, 40, False, 32, 2, 6, [1, 30], [31, 100], 16),
    ("f32", 256, 256, False, 128, 1, 1, [300], [77], 0),
    ("bf16", 256, 64, True, 256, 2, 4, [1003], [40], 0),
    ("f32", 6, 2, True, 32, 2, 4, [3, 31], [5, 33], 1),
    ("f32", 98, 98, False, 32, 1, 3, [40], [1], 3),
    ("f32", 192, 96, False, 64, 2, 2, [10, 0, 63], [0, 7, 1], 0),   # a sequence without a new row
]


@pytest.mark.parametrize("ty,dim,rot,pairs,page,kv,heads,old,new,gap", APPENDS)
def test_append_equals_its_definition(accel, pkg, ty, dim, rot, pairs, page, kv, heads, old, new, gap):
    rng = np.random.default_rng(dim + page)
    lens = [o + n for o, n in zip(old, new)]
    pages = sum(-(-n // page) for n in lens) + 2
    cache = R.Cache(pages, page, kv, dim, seed=3)
    table = R.tables(rng, pages, page, lens)
    R.append(cache, table, [0] * len(old), old, *(rng.standard_normal((sum(old), kv, dim)).astype(np.float32) for _ in range(2)))
    rope = R.rope_table(max(lens), rot)
    rows = sum(new)
    k, k_raw, ldk = _rows(rng, ty, rows, kv, dim, gap, 1.3)
    v, v_raw, ldv = _rows(rng, ty, rows, kv, dim, gap + 8, 0.7)
    q, q_raw, ldq = _rows(rng, ty, rows, heads, dim, gap)
    pos = np.concatenate([np.arange(o, o + n) for o, n in zip(old, new)])
    with R.Dev(accel) as dev:
        d = R.OnDevice(pkg, dev, cache)
        batch = d.batch(table, lens, new)
        qo = dev.put(np.zeros_like(q_raw))
        turn = pkg.Rope(dev.put(rope), rope.shape[0], rot, interleaved=pairs)
        call = dict(rope=turn, q=dev.put(q_raw), q_heads=heads, q_out=qo, dtype=_dtype(pkg, ty), ldk=ldk, ldv=ldv, ldq=ldq, ldqo=ldq)
        kp, vp = dev.put(k_raw), dev.put(v_raw)
        ko, vo = dev.room(rows * kv * dim * 4), dev.room(rows * kv * dim * 4)
        R.append(cache, table, old, new, R.rotate(k, rope, pos, rot, pairs), v)
        want = R.rotate(q, rope, pos, rot, pairs).reshape(rows, -1)
        for _ in range(2):   # the second time changes nothing
            accel.kv_append_dev(d.handle, batch, kp, vp, **call)
            got = d.planes()
            used = ~np.isnan(cache.ks)
            assert _same(got[2], cache.ks) and _same(got[3], cache.vs)
            for s, n in enumerate(lens):
                host = R.Cache(1, page, kv, dim)
                host.pages, host.k, host.v, host.ks, host.vs = pages, *got
                for h in range(kv):
                    for w in "kv":
                        assert np.array_equal(host.tokens(w, table[s], h, n), cache.tokens(w, table[s], h, n)), (s, h, w)
            out = dev.get(qo, q_raw.shape, q_raw.dtype)[:, :heads * dim]
            assert np.array_equal(out, want if ty == "f32" else R.bf16(want))
        assert used.any()
        accel.kv_read_dev(d.handle, batch, ko, vo)
        r = 0
        back_k, back_v = dev.get(ko, (rows, kv, dim)), dev.get(vo, (rows, kv, dim))
        for s, (o, n) in enumerate(zip(old, new)):
            for h in range(kv):
                assert np.array_equal(back_k[r:r + n, h], cache.tokens("k", table[s], h, o + n)[o:])
                assert np.array_equal(back_v[r:r + n, h], cache.tokens("v", table[s], h, o + n)[o:])
            r += n


@pytest.mark.parametrize("off", [0, 1, 30, 31])
@pytest.mark.parametrize("n", [1, 2, 3, 31, 32, 33, 34, 35, 65, 66])
def test_every_block_that_rows_touch(accel, pkg, off, n):
    """One sequence whose rows begin and end at every kind of place in a block."""
    rng = np.random.default_rng(off * 100 + n)
    kv, dim, page = 1, 64, 32
    cache = R.Cache(6, page, kv, dim)
    table = R.tables(rng, 6, page, [off + n])
    R.append(cache, table, [0], [off], *(rng.standard_normal((off, kv, dim)).astype(np.float32) for _ in range(2)))
    k, kr, _ = _rows(rng, "f32", n, kv, dim)
    v, vr, _ = _rows(rng, "f32", n, kv, dim)
    with R.Dev(accel) as dev:
        d = R.OnDevice(pkg, dev, cache)
        batch = d.batch(table, [off + n], [n], always_row0=True)
        accel.kv_append_dev(d.handle, batch, dev.put(kr), dev.put(vr))
        R.append(cache, table, [off], [n], k, v)
        ko, vo = dev.room(kr.nbytes), dev.room(vr.nbytes)
        accel.kv_read_dev(d.handle, batch, ko, vo)
        got = d.planes()
        assert _same(got[2], cache.ks) and _same(got[3], cache.vs)
        assert np.array_equal(dev.get(ko, k.shape)[:, 0], cache.tokens("k", table[0], 0, off + n)[off:])
        assert np.array_equal(dev.get(vo, v.shape)[:, 0], cache.tokens("v", table[0], 0, off + n)[off:])


def test_append_without_rotation_or_queries_in_place_queries(accel, pkg):
    rng = np.random.default_rng(5)
    kv, dim, rows = 2, 64, 3
    lens = [rows]
    cache = R.Cache(2, 32, kv, dim)
    table = R.tables(rng, 2, 32, lens)
    k, kr, _ = _rows(rng, "f32", rows, kv, dim)
    v, vr, _ = _rows(rng, "f32", rows, kv, dim)
    q, qr, _ = _rows(rng, "f32", rows, 4, dim)
    with R.Dev(accel) as dev:
        d = R.OnDevice(pkg, dev, cache)
        batch = d.batch(table, lens, [rows])
        accel.kv_append_dev(d.handle, batch, dev.put(kr), dev.put(vr))
        R.append(cache, table, [0], [rows], k, v)
        got = d.planes()
        assert _same(got[2], cache.ks) and _same(got[3], cache.vs)
        qp = dev.put(qr)
        rope = R.rope_table(rows, dim)
        accel.kv_append_dev(d.handle, batch, dev.put(kr), dev.put(vr), rope=pkg.Rope(dev.put(rope), rows, dim), q=qp, q_heads=4, q_out=qp)
        assert np.array_equal(dev.get(qp, q.shape), R.rotate(q, rope, np.arange(rows), dim, False))


def test_tokens_one_at_a_time_raise_the_scale(accel, pkg):
    """70 tokens of growing and shrinking size, one call each: earlier codes follow the scale exactly as defined."""
    rng = np.random.default_rng(6)
    kv, dim, page, n = 2, 64, 32, 70
    cache = R.Cache(4, page, kv, dim, seed=1)
    table = R.tables(rng, 4, page, [n, 1])
    with R.Dev(accel) as dev:
        d = R.OnDevice(pkg, dev, cache)
        for i in range(n):
            size = 10.0 ** rng.uniform(-3, 3)
            k, kr, _ = _rows(rng, "f32", 1, kv, dim, 0, size)
            v, vr, _ = _rows(rng, "f32", 1, kv, dim, 0, 1 / size)
            accel.kv_append_dev(d.handle, d.batch(table[:1], [i + 1], [1]), dev.put(kr), dev.put(vr))
            R.append(cache, table, [i], [1], k, v)
        got = d.planes()
        assert _same(got[2], cache.ks) and _same(got[3], cache.vs)
        host = R.Cache(1, page, kv, dim)
        host.k, host.v, host.ks, host.vs = got
        for h in range(kv):
            for w in "kv":
                assert np.array_equal(host.tokens(w, table[0], h, n), cache.tokens(w, table[0], h, n))


@pytest.mark.parametrize("value,scale", [(0.0, 0.0), (1e-30, 0.0), (2.0 ** -96, 2.0 ** -96 / 127), (np.nan, np.nan), (np.inf, np.nan), (3e38, 3e38 / 127)])
def test_append_of_extreme_values(accel, pkg, value, scale):
    kv, dim = 1, 64
    cache = R.Cache(1, 32, kv, dim)
    k = np.zeros((2, kv, dim), np.float32)
    k[0, 0, 3] = value
    v = -k
    with R.Dev(accel) as dev:
        d = R.OnDevice(pkg, dev, cache)
        accel.kv_append_dev(d.handle, d.batch([[0]], [2], [2]), dev.put(k), dev.put(v))
        got = d.planes()
        want = np.float32(value) / np.float32(127) if np.isfinite(scale) and scale else np.float32(scale)
        assert _same(got[2].reshape(-1), np.full(1, want, np.float32)) and _same(got[3].reshape(-1), np.full(1, want, np.float32))
        # a new sequence in the block starts it again
        accel.kv_append_dev(d.handle, d.batch([[0]], [1], [1]), dev.put(np.ones_like(k)), dev.put(np.ones_like(v)))
        got = d.planes()
        assert got[2].reshape(-1)[0] == np.float32(1) / np.float32(127) and got[0].reshape(-1)[0] == 127


def test_rows_outside_what_the_batch_says_are_left_out(accel, pkg):
    """Lengths and rows beyond the sizes of the call, page numbers outside the cache: nothing outside the cache is touched."""
    rng = np.random.default_rng(7)
    kv, dim = 2, 64
    with R.Dev(accel) as dev:
        cache = R.Cache(3, 32, kv, dim)
        cache.ks[:] = cache.vs[:] = 0.01       # sequence 2's earlier tokens are whatever its block holds
        d = R.OnDevice(pkg, dev, cache)
        k, kr, _ = _rows(rng, "f32", 4, kv, dim)
        q, qr, _ = _rows(rng, "f32", 4, 4, dim)
        out = dev.put(np.zeros((4, 4, dim), np.float32))
        lens = dev.put(np.array([200, -5, 9], np.int32))                       # table of 2 pages: 64 tokens
        row0 = dev.put(np.array([0, 2, 3, 90], np.int32))
        table = dev.put(np.array([[0, 1], [7, -7], [-3, 2]], np.int32))
        b = pkg.KvBatch(3, lens, table, 2, 1000, row0=row0, rows=4, max_rows=2)
        accel.kv_append_dev(d.handle, b, dev.put(kr), dev.put(kr))
        accel.attn_dev(d.handle, b, dev.put(qr), 4, 1.0, out)
        accel.kv_read_dev(d.handle, b, dev.room(4 * kv * dim * 4), None)
        got = dev.get(out, (4, 4, dim))
        assert not got[2].any()                                                 # a sequence without a token
        assert np.isfinite(got[3]).all()


def test_rope_table(accel):
    with R.Dev(accel) as dev:
        for rot, n, base in ((128, 4000, 1e4), (64, 3, 1e6), (2, 70000, 1e4)):
            p = dev.room(n * rot * 4)
            accel.rope_table_dev(base, rot, n, p)
            got = dev.get(p, (n, rot // 2, 2))
            # angles of up to 7e4 rounded to 64 bits and cos, sin rounded to fp32
            assert np.abs(got - R.rope_table(n, rot, base).astype(np.float64)).max() <= 2.0 ** -24 + 1e-10


ATTENDS = [
    # type, dim, page, kv heads, q heads, lens, new, window, gap
    ("f32", 128, 64, 2, 8, [1], [1], 0, 0),
    ("f32", 128, 64, 2, 8, [601, 1, 33, 0, 64], [1, 1, 1, 1, 1], 0, 0),
    ("f32", 64, 32, 1, 1, [31, 32, 33], [1, 1, 1], 0, 4),
    ("bf16", 128, 32, 2, 10, [700, 95], [1, 1], 0, 8),
    ("f32", 256, 128, 2, 4, [300, 257], [1, 1], 0, 0),
    ("bf16", 256, 96, 1, 16, [500], [1], 0, 0),
    ("f32", 80, 96, 2, 6, [333, 40], [1, 1], 0, 1),
    ("bf16", 192, 64, 1, 3, [129], [1], 0, 0),
    ("f32", 6, 32, 2, 4, [77, 5], [1, 1], 0, 0),
    ("f32", 128, 64, 1, 32, [200], [1], 0, 0),                       # more heads in a group than a tile has rows
    ("f32", 128, 32, 2, 4, [900, 100, 31], [1, 1, 1], 64, 0),
    ("bf16", 64, 64, 1, 4, [900, 5], [1, 1], 1, 0),                  # a row sees itself alone
    ("f32", 128, 64, 4, 8, [4000, 17, 2049], [1, 1, 1], 0, 0),       # long enough to be split
    ("f32", 64, 256, 1, 2, [9000], [1], 0, 0),                       # more blocks than one look-up
    # a few rows of a sequence
    ("bf16", 80, 96, 4, 20, [1500, 333, 6, 3], [6, 5, 6, 6], 0, 0),  # the last sequence has more rows than tokens
    ("f32", 128, 64, 2, 4, [100, 50, 40], [3, 0, 7], 0, 16),         # one without a row
    ("f32", 128, 64, 2, 4, [300], [8], 5, 0),
    ("f32", 64, 32, 2, 6, [1000], [5], 0, 0),
    ("bf16", 256, 64, 2, 4, [700, 90], [9, 2], 100, 0),
    # prompt chunks
    ("f32", 128, 64, 2, 8, [130], [130], 0, 0),
    ("f32", 128, 32, 1, 3, [500, 77, 301], [200, 77, 1], 0, 0),
    ("bf16", 128, 64, 2, 4, [1111], [300], 0, 0),
    ("bf16", 64, 96, 1, 5, [257, 64], [257, 40], 0, 8),
    ("f32", 256, 64, 1, 2, [400], [150], 0, 0),
    ("bf16", 256, 128, 1, 2, [333], [333], 0, 0),
    ("f32", 192, 64, 1, 1, [190], [140], 0, 0),
    ("f32", 80, 96, 1, 4, [300], [100], 0, 2),
    ("f32", 128, 64, 1, 4, [900], [256], 130, 0),                    # whole tiles out of the window on both sides
    ("bf16", 128, 32, 1, 2, [600, 50], [200, 60], 33, 0),
    ("f32", 64, 64, 1, 2, [4500], [70], 0, 0),                       # split, more blocks than one look-up
]


@pytest.mark.parametrize("ty,dim,page,kv,heads,lens,new,window,gap", ATTENDS)
def test_attention_against_64_bits(accel, pkg, ty, dim, page, kv, heads, lens, new, window, gap):
    rng = np.random.default_rng(dim * 7 + len(lens))
    pages = sum(-(-n // page) for n in lens) + 2
    cache, table = _filled(rng, pages, page, kv, dim, lens)
    rows = sum(new)
    q, raw, ldq = _rows(rng, ty, rows, heads, dim, gap)
    size = (1 + np.arange(heads) % 3)[None, :, None]   # some heads look at few tokens, some at many
    q = q * size.astype(np.float32)
    raw[:, :heads * dim] = (q if ty == "f32" else R.bf16(q)).reshape(rows, -1)
    q = q if ty == "f32" else R.from_bf16(R.bf16(q))
    want = R.attend(cache, table, lens, new, q, dim ** -0.5, window)
    top = max(np.abs(cache.tokens("v", table[s], h, n)).max() for s, n in enumerate(lens) if n for h in range(kv))
    with R.Dev(accel) as dev:
        d = R.OnDevice(pkg, dev, cache)
        ldo = heads * dim + gap
        fill = np.full((rows, ldo), 7, np.float32 if ty == "f32" else np.uint16)
        out = dev.put(fill)
        got = []
        for always in (False, True):
            for max_len in (max(lens), 3 * max(lens) + 500):   # a loose bound gives other pieces
                batch = d.batch(table, lens, new, max_len=max_len, always_row0=always)
                accel.attn_dev(d.handle, batch, dev.put(raw), heads, dim ** -0.5, out, window=window, dtype=_dtype(pkg, ty), ldq=ldq, ldo=ldo)
                y = dev.get(out, fill.shape, fill.dtype)
                assert (y[:, heads * dim:] == fill[:, heads * dim:]).all()   # nothing between the rows is written
                y = (y if ty == "f32" else R.from_bf16(y))[:, :heads * dim].reshape(rows, heads, dim)
                err = np.abs(y - want).max() / top
                print(f"{ty} dim {dim} max_len {max_len}: error {err:.2e}")
                assert err <= TOL[ty]
                got.append(y)
        assert np.array_equal(got[0], got[2])   # row0 given or not


def test_attention_scale_extremes(accel, pkg):
    """Value scales 2^40 apart, tiny and huge queries, keys of zero: f16's range is not the kernel's."""
    rng = np.random.default_rng(9)
    kv, dim, page, lens = 1, 64, 32, [200]
    for size in ((1.0, 1e-30), (1.0, 1e30), (1e-20, 1.0), (1e18, 1.0), (0.0, 1.0)):
        cache, table = _filled(rng, 8, page, kv, dim, lens, size)
        q, raw, _ = _rows(rng, "f32", 1, 2, dim, 0, 1.0 / max(size[0], 1e-15))
        want = R.attend(cache, table, lens, [1], q, 0.125)
        with R.Dev(accel) as dev:
            d = R.OnDevice(pkg, dev, cache)
            out = dev.room(raw.nbytes)
            accel.attn_dev(d.handle, d.batch(table, lens, [1]), dev.put(raw), 2, 0.125, out)
            top = np.abs(cache.tokens("v", table[0], 0, 200)).max()
            assert np.abs(dev.get(out, q.shape) - want).max() <= 2e-5 * top, size


def test_rows_do_not_see_other_rows(accel, pkg):
    """A NaN key poisons its block for the rows that see it and for no other row; other sequences' values change nothing."""
    rng = np.random.default_rng(10)
    kv, dim, page, lens, new = 1, 64, 32, [300, 120], [40, 40]
    cache, table = _filled(rng, 16, page, kv, dim, lens)
    q, raw, _ = _rows(rng, "f32", 80, 2, dim)
    res = []
    for poison in (False, True):
        if poison:
            cache.ks[table[0][280 // 32], 0, 0] = np.nan    # tokens 256..287 of sequence 0 (rows 0..: positions 260..)
            cache.vs[table[0][9], 0, 0] = np.nan            # tokens 288.. of sequence 0
        with R.Dev(accel) as dev:
            d = R.OnDevice(pkg, dev, cache)
            out = dev.room(raw.nbytes)
            accel.attn_dev(d.handle, d.batch(table, lens, new), dev.put(raw), 2, 0.125, out, window=3)
            res.append(dev.get(out, (80, 2, dim)))
    assert np.isfinite(res[0]).all()
    assert np.array_equal(res[1][40:], res[0][40:])          # the other sequence
    assert np.isnan(res[1][:40]).all()                       # every row of sequence 0 sees a poisoned block
    # the rows whose window ends in front of the poisoned blocks
    cache.ks[table[0][8], 0, 0] = cache.ks[table[0][7], 0, 0]
    with R.Dev(accel) as dev:
        d = R.OnDevice(pkg, dev, cache)
        out = dev.room(raw.nbytes)
        accel.attn_dev(d.handle, d.batch(table, lens, new), dev.put(raw), 2, 0.125, out, window=3)
        y = dev.get(out, (80, 2, dim))
        assert np.isfinite(y[:28]).all() and np.isnan(y[28:40]).all()   # row 28 is position 288


def test_decode_step_as_a_graph(accel, pkg):
    """Append and attention captured once and replayed while lengths, tables and rows change."""
    rng = np.random.default_rng(11)
    kv, heads, dim, page, n = 2, 4, 64, 32, 3
    cap = 160
    cache = R.Cache(n * 5 + 1, page, kv, dim)
    table = R.tables(rng, cache.pages, page, [cap] * n)
    rope = R.rope_table(cap, dim)
    with R.Dev(accel) as dev:
        d = R.OnDevice(pkg, dev, cache)
        lens = np.array([1, 40, 127], np.int32)
        start = [int(x) - 1 for x in lens]
        k, v = (rng.standard_normal((sum(start), kv, dim)).astype(np.float32) for _ in range(2))
        if sum(start):
            accel.kv_append_dev(d.handle, d.batch(table, start, start), dev.put(k), dev.put(v))
            R.append(cache, table, [0] * n, start, k, v)
        lp, tp = dev.put(lens), dev.put(table)
        batch = pkg.KvBatch(n, lp, tp, table.shape[1], cap)
        bufs = {x: dev.room(n * w * dim * 4) for x, w in (("q", heads), ("k", kv), ("v", kv), ("qo", heads), ("out", heads))}
        turn = pkg.Rope(dev.put(rope), cap, dim)

        def step():
            accel.kv_append_dev(d.handle, batch, bufs["k"], bufs["v"], rope=turn, q=bufs["q"], q_heads=heads, q_out=bufs["qo"])
            accel.attn_dev(d.handle, batch, bufs["qo"], heads, dim ** -0.5, bufs["out"])

        rows = {x: np.zeros((n, w, dim), np.float32) for x, w in (("q", heads), ("k", kv), ("v", kv))}
        # seen once outside the capture, on a cache that starts its blocks again below
        keep = d.planes()
        step()
        for p, x in zip(d.p, keep):
            accel.h2d(p, x)
        accel.sync()
        accel.graph_begin()
        step()
        g = accel.graph_end()
        for i in range(5):
            for x in rows:
                rows[x] = rng.standard_normal(rows[x].shape).astype(np.float32)
                accel.h2d(bufs[x], rows[x])
            accel.h2d(lp, lens)
            accel.graph_launch(g)
            R.append(cache, table, [int(x) - 1 for x in lens], [1] * n, R.rotate(rows["k"], rope, lens - 1, dim, False), rows["v"])
            q = R.rotate(rows["q"], rope, lens - 1, dim, False)
            want = R.attend(cache, table, [int(x) for x in lens], [1] * n, q, dim ** -0.5)
            got = dev.get(bufs["out"], want.shape)
            assert np.abs(got - want).max() <= 2e-5 * 5, i
            assert np.array_equal(dev.get(bufs["qo"], q.shape), q)
            lens = lens + 1
        accel.graph_destroy(g)


def test_refusals(accel, pkg):
    with R.Dev(accel) as dev:
        cache = R.Cache(2, 32, 2, 64)
        d = R.OnDevice(pkg, dev, cache)
        room = dev.room(1 << 16)
        good = d.batch([[0], [1]], [3, 4], [1, 1])
        call = lambda c=d.handle, b=good, q=room, heads=4, **k: accel.attn_dev(c, b, q, heads, 1.0, room, **k)
        call()

        def other(**k):
            f = {n: getattr(d.handle, n) for n in ("pages", "page_tokens", "kv_heads", "head_dim", "k", "v", "k_scale", "v_scale")}
            f.update(k)
            return pkg.KvCache(*f.values())

        def batch(**k):
            f = dict(nseq=2, len=good.len, table=good.table, table_ld=1, max_len=4)
            f.update(k)
            return pkg.KvBatch(**f)

        for bad in (other(page_tokens=33), other(page_tokens=0), other(head_dim=65), other(head_dim=258), other(head_dim=0), other(pages=0),
                    other(kv_heads=0), other(k=None), other(v_scale=None), other(k=d.handle.k + 8)):
            for f in (call, lambda c: accel.kv_append_dev(c, good, room, room), lambda c: accel.kv_read_dev(c, good, room, None)):
                with pytest.raises(pkg.SmxError):
                    f(bad)
        for bad in (batch(len=None), batch(table=None), batch(table_ld=0), batch(rows=3), batch(row0=room, rows=2, max_rows=5), batch(max_len=1 << 29),
                    batch(nseq=70000)):
            for f in (lambda b: call(b=b), lambda b: accel.kv_append_dev(d.handle, b, room, room), lambda b: accel.kv_read_dev(d.handle, b, room, room)):
                with pytest.raises(pkg.SmxError):
                    f(bad)
        for k in (dict(heads=3), dict(heads=0), dict(q=None), dict(dtype=1), dict(ldq=255), dict(ldo=255)):
            with pytest.raises(pkg.SmxError):
                call(**k)
        rope = lambda **k: pkg.Rope(**{**dict(table=room, n_pos=4, rot_dim=64), **k})
        for k in (dict(rope=rope(table=None)), dict(rope=rope(n_pos=0)), dict(rope=rope(rot_dim=66)), dict(rope=rope(rot_dim=3)), dict(dtype=2),
                  dict(ldk=127), dict(ldv=1), dict(q=room, q_heads=4), dict(q=room, q_heads=0, q_out=room), dict(q=room, q_heads=4, q_out=room, ldq=8)):
            with pytest.raises(pkg.SmxError):
                accel.kv_append_dev(d.handle, good, room, room, **k)
        for k, v in ((None, room), (room, None)):
            with pytest.raises(pkg.SmxError):
                accel.kv_append_dev(d.handle, good, k, v)
        with pytest.raises(pkg.SmxError):
            accel.kv_read_dev(d.handle, good, None, None)
        for base, rot, n, p in ((0.0, 64, 4, room), (1e4, 3, 4, room), (1e4, 64, 0, room), (1e4, 64, 4, None), (1e4, 512, 4, room)):
            with pytest.raises(pkg.SmxError):
                accel.rope_table_dev(base, rot, n, p)
        empty = batch(nseq=0, rows=0)
        call(b=empty)
        accel.kv_append_dev(d.handle, empty, room, room)


def test_sizes(pkg):
    assert pkg.kv_sizes(3, 64, 2, 80) == (3 * 64 * 2 * 128, 3 * 2 * 2)
    for bad in ((0, 64, 2, 80), (3, 65, 2, 80), (3, 64, 2, 81), (3, 64, 2, 258), (3, 64, 0, 80)):
        with pytest.raises(ValueError):
            pkg.kv_sizes(*bad)
