"""The cache, attention and sampler where byte and element offsets pass 32 bits, and attention over every way that a context is split and
its pieces are joined."""
import numpy as np
import pytest

import kv_ref as R

pytestmark = pytest.mark.gpu
KV, DIM, PAGE = 2, 128, 64


def _planes(pkg, accel, dev, pages):
    nb, ns = pkg.kv_sizes(pages, PAGE, KV, DIM)
    return pkg.KvCache(pages, PAGE, KV, DIM, dev.room(nb), dev.room(nb), dev.room(ns * 4), dev.room(ns * 4)), nb


def _everything(pkg, accel, dev, cache, table, lens, new, heads, k, v, q):
    """A chunk appended, read back, attended to; then one row of each sequence (the last, again)."""
    rows = sum(new)
    d = R.OnDevice.__new__(R.OnDevice)
    d.pkg, d.dev, d.host, d.handle = pkg, dev, None, cache
    batch, one = d.batch(table, lens, new, always_row0=True), d.batch(table, lens, [1] * len(lens))
    kd, vd, qd, out = dev.put(k), dev.put(v), dev.put(q), dev.room(q.nbytes)
    accel.kv_append_dev(cache, batch, kd, vd)
    back = [dev.room(k.nbytes), dev.room(v.nbytes)]
    accel.kv_read_dev(cache, batch, *back)
    accel.attn_dev(cache, batch, qd, heads, DIM ** -0.5, out)
    got = [dev.get(p, k.shape) for p in back] + [dev.get(out, q.shape)]
    few = dev.room(q.nbytes)
    accel.attn_dev(cache, one, qd, heads, DIM ** -0.5, few)
    return got + [dev.get(few, (len(lens),) + q.shape[1:])], rows


@pytest.mark.parametrize("new", [[3, 5], [70, 41]])   # rows to the matrix tiles of few rows, of many
def test_pages_past_4_gb(accel, pkg, new):
    """The same step in a small cache and at the end of one whose planes pass 2^32 bytes: the same bits."""
    rng = np.random.default_rng(31)
    heads, lens = 8, new
    k, v = (rng.standard_normal((sum(new), KV, DIM)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((sum(new), heads, DIM)).astype(np.float32)
    small = R.tables(rng, 8, PAGE, lens)
    far = (1 << 32) // (PAGE * KV * DIM) + 8
    res = []
    for pages, table in ((8, small), (far, np.where(small >= 0, far - 1 - small, small))):
        with R.Dev(accel) as dev:
            cache, nb = _planes(pkg, accel, dev, pages)
            assert pages == 8 or nb > 1 << 32
            res.append(_everything(pkg, accel, dev, cache, table, lens, new, heads, k, v, q)[0])
    for a, b in zip(*res):
        assert np.isfinite(a).all() and np.array_equal(a, b)


def test_rows_past_2_to_the_32_bytes(accel, pkg):
    """Queries, results and logits whose rows are 2^31 elements apart."""
    rng = np.random.default_rng(32)
    far, heads, lens = 1 << 31, 4, [40, 7]
    k, v = (rng.standard_normal((sum(lens), KV, DIM)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((2, heads, DIM)).astype(np.float32)
    x = rng.standard_normal((2, 3000)).astype(np.float32)
    with R.Dev(accel) as dev:
        host = R.Cache(4, PAGE, KV, DIM)
        d = R.OnDevice(pkg, dev, host)
        table = R.tables(rng, 4, PAGE, lens)
        accel.kv_append_dev(d.handle, d.batch(table, lens, lens), dev.put(k), dev.put(v))
        one = d.batch(table, lens, [1, 1])
        near = dev.room(q.nbytes)
        accel.attn_dev(d.handle, one, dev.put(q), heads, DIM ** -0.5, near)
        want = dev.get(near, q.shape)
        wide = dev.room((far + 8192) * 4)
        for r in range(2):
            accel.h2d(wide + r * far * 4, q[r])
        accel.attn_dev(d.handle, one, wide, heads, DIM ** -0.5, wide, ldq=far, ldo=far)
        for r in range(2):
            assert np.array_equal(dev.get(wide + r * far * 4, (heads, DIM)), want[r]), r
            accel.h2d(wide + r * far * 4, x[r])
        u, ids, at = dev.put(np.array([0.3, 0.8], np.float32)), dev.room(8), dev.put(np.full(2, 0.9, np.float32))
        accel.sample_dev(wide, 2, 3000, u, ids, top_p=at, ld=far)
        picked = dev.get(ids, 2, np.int32)
        accel.sample_dev(dev.put(x), 2, 3000, u, ids, top_p=at)
        assert np.array_equal(picked, dev.get(ids, 2, np.int32))


@pytest.mark.parametrize("group,new", [(1, 1), (2, 1), (4, 1), (8, 1), (16, 1), (1, 5), (5, 3), (8, 4), (16, 4), (16, 5)])
def test_splits_and_joins(accel, pkg, group, new):
    """1 to 72 rows of a key/value head over contexts of one piece to dozens, ragged, several calls on the same context: fp32 within the
    bound that the tests of attention derive (2e-5 of the largest value)."""
    rng = np.random.default_rng(group * 10 + new)
    for kv, lens in ((1, [new]), (1, [128 + new, 129]), (2, [700, 300, 1]), (1, [2100]), (8, [1000, 40]), (2, [255])):
        heads, dim, page = kv * group, 64, 32
        lens = [max(n, new) for n in lens]
        cache = R.Cache(sum(-(-n // page) for n in lens) + 1, page, kv, dim)
        table = R.tables(rng, cache.pages, page, lens)
        k, v = (rng.standard_normal((sum(lens), kv, dim)).astype(np.float32) for _ in range(2))
        R.append(cache, table, [0] * len(lens), lens, k, v)
        n = [new] * len(lens)
        q = rng.standard_normal((sum(n), heads, dim)).astype(np.float32)
        want = R.attend(cache, table, lens, n, q, dim ** -0.5)
        with R.Dev(accel) as dev:
            d = R.OnDevice(pkg, dev, cache)
            qd, out, b = dev.put(q), dev.put(np.full(q.shape, np.nan, np.float32)), d.batch(table, lens, n)
            for again in range(2):
                accel.attn_dev(d.handle, b, qd, heads, dim ** -0.5, out)
                got = dev.get(out, q.shape)
                assert np.abs(got - want).max() <= 2e-5 * np.abs(v).max(), (kv, lens, again)
                first = got if again == 0 else first
            assert np.array_equal(first, got)   # (whichever workgroup joins the pieces, they are added in the same order)


@pytest.mark.parametrize("new,ty", [(1, "f32"), (3, "f32"), (40, "bf16")])
def test_one_long_sequence_among_many(accel, pkg, new, ty):
    """A batch that fills the chip with short sequences, and a long one that is split all the same."""
    rng = np.random.default_rng(33 + new)
    kv, heads, dim, page = 8, 16, 128, 64
    lens = [int(n) for n in rng.integers(new, 90, 63)] + [16500]
    cache = R.Cache(sum(-(-n // page) for n in lens) + 1, page, kv, dim, seed=new)
    cache.ks[:], cache.vs[:] = (rng.uniform(0.001, 0.02, cache.ks.shape).astype(np.float32) for _ in range(2))
    table = R.tables(rng, cache.pages, page, lens)
    n = [new] * len(lens)
    q = rng.standard_normal((sum(n), heads, dim)).astype(np.float32)
    raw = q if ty == "f32" else R.bf16(q)
    q = q if ty == "f32" else R.from_bf16(raw)
    want = R.attend(cache, table, lens, n, q, dim ** -0.5)
    with R.Dev(accel) as dev:
        d = R.OnDevice(pkg, dev, cache)
        out = dev.room(raw.nbytes)
        accel.attn_dev(d.handle, d.batch(table, lens, n), dev.put(raw), heads, dim ** -0.5, out, dtype=pkg.DTYPE_F32 if ty == "f32" else pkg.DTYPE_BF16)
        got = dev.get(out, raw.shape, raw.dtype)
    got = got if ty == "f32" else R.from_bf16(got)
    # values of up to 128 * 0.02; the bounds that the tests of attention derive: 2e-5 of that, bf16 2^-8 of it
    assert np.abs(got - want).max() <= (2e-5 if ty == "f32" else 2.0 ** -8) * 128 * 0.02


@pytest.mark.parametrize("nseq,chunks,ty,dim", [(3, [1], "f32", 64), (70, [5, 69], "f32", 64), (200, [0, 63, 64, 130, 199], "bf16", 128), (130, [], "f32", 80),
                                                (4200, [17, 4199], "f32", 64)])
def test_decode_steps_beside_prompt_chunks(accel, pkg, nseq, chunks, ty, dim):
    """Sequences of one row (and of none) in a call with chunks of 33 rows and more: each kind has its own launch, the chunks wherever they
    stand among the others."""
    rng = np.random.default_rng(nseq)
    kv, heads, page = 1, 2, 32
    n = [1 if i % 11 else 0 for i in range(nseq)]
    for j, c in enumerate(chunks):
        n[c] = 33 + 7 * j
    if not chunks:
        n[40] = 32   # 64 rows of the key/value head: still few
    lens = [m + int(x) for m, x in zip(n, rng.integers(0, 60, nseq))]
    cache = R.Cache(sum(-(-m // page) for m in lens) + 1, page, kv, dim, seed=nseq)
    cache.ks[:], cache.vs[:] = (rng.uniform(0.001, 0.02, cache.ks.shape).astype(np.float32) for _ in range(2))
    table = R.tables(rng, cache.pages, page, lens)
    q = rng.standard_normal((sum(n), heads, dim)).astype(np.float32)
    raw = q if ty == "f32" else R.bf16(q)
    q = q if ty == "f32" else R.from_bf16(raw)
    want = R.attend(cache, table, lens, n, q, dim ** -0.5)
    with R.Dev(accel) as dev:
        d = R.OnDevice(pkg, dev, cache)
        out = dev.put(np.full(raw.shape, 0x7fc0 if ty == "bf16" else np.nan, raw.dtype))
        accel.attn_dev(d.handle, d.batch(table, lens, n, always_row0=True), dev.put(raw), heads, dim ** -0.5, out,
                       dtype=pkg.DTYPE_F32 if ty == "f32" else pkg.DTYPE_BF16)
        got = dev.get(out, raw.shape, raw.dtype)
    got = got if ty == "f32" else R.from_bf16(got)
    assert np.abs(got - want).max() <= (2e-5 if ty == "f32" else 2.0 ** -8) * 128 * 0.02


@pytest.mark.parametrize("ty,dim,new,window", [("f32", 64, 1, 0), ("bf16", 128, 1, 50), ("f32", 192, 2, 0), ("bf16", 256, 3, 0), ("f32", 80, 4, 33)])
def test_many_short_sequences(accel, pkg, ty, dim, new, window):
    """Enough of them for a wave each: lengths from none to several hundred."""
    rng = np.random.default_rng(dim + new)
    kv, heads, page, nseq = 8, 32, 32, 140
    lens = [int(x) for x in rng.integers(0, 60, nseq)]
    lens[3], lens[70], lens[139] = 0, 470, 256
    n = [new if new > 1 else 1] * nseq
    cache = R.Cache(sum(-(-m // page) for m in lens) + 1, page, kv, dim, seed=dim)
    cache.ks[:], cache.vs[:] = (rng.uniform(0.001, 0.02, cache.ks.shape).astype(np.float32) for _ in range(2))
    table = R.tables(rng, cache.pages, page, lens)
    q = rng.standard_normal((sum(n), heads, dim)).astype(np.float32)
    raw = q if ty == "f32" else R.bf16(q)
    q = q if ty == "f32" else R.from_bf16(raw)
    want = R.attend(cache, table, lens, n, q, dim ** -0.5, window)
    with R.Dev(accel) as dev:
        d = R.OnDevice(pkg, dev, cache)
        out = dev.put(np.full(raw.shape, 0x7fc0 if ty == "bf16" else np.nan, raw.dtype))
        accel.attn_dev(d.handle, d.batch(table, lens, n), dev.put(raw), heads, dim ** -0.5, out, window=window,
                       dtype=pkg.DTYPE_F32 if ty == "f32" else pkg.DTYPE_BF16)
        got = dev.get(out, raw.shape, raw.dtype)
    got = got if ty == "f32" else R.from_bf16(got)
    assert np.abs(got - want).max() <= (2e-5 if ty == "f32" else 2.0 ** -8) * 128 * 0.02
