"""The sampler against its definition in 64 bits.

A pick i is right when u lies in the share of the kept weight that token i takes, in index order.  The device's weights are fp32
exponentials (up to 2 units in the last place, 2^-23 relative, and the fp32 quotient in front of them: |(x - max) / T| <= 28 with 2^-24
of it, 1.7e-6) cut to 2^-40: a running total is off by less than 2e-6 of the total, and so may be the limits of top_p.  Tokens that the
cuts decide between within that distance may be kept or not."""
import numpy as np
import pytest

import kv_ref as R

pytestmark = pytest.mark.gpu
EPS = 4e-6


def _weights(x, T):
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    m = x.max()
    with np.errstate(invalid="ignore"):
        w = np.where(x == m, 1.0, np.exp((x - m) / T))
    return np.where(x == -np.inf, 0.0, w)


def _kept(x, T, k, p, m, slack):
    """Kept weights of one row; slack > 0: every token that may be kept, < 0: only those that must be."""
    w = _weights(x, T)
    clean = np.where(np.isnan(x), -np.inf, x)
    order = np.lexsort((np.arange(x.size), -clean.astype(np.float64)))
    n = min(k, x.size) if k > 0 else x.size
    keep = np.zeros(x.size, bool)
    ahead = np.cumsum(w[order[:n]]) - w[order[:n]]
    total = w[order[:n]].sum()
    keep[order[:n]] = True if p >= 1 else ahead < (p + slack) * total
    keep[order[0]] = True
    return np.where(keep & (w >= m * (1 - slack)), w, 0.0)


def _check(x, ids, prob, u, T, k, p, m):
    for r in range(x.shape[0]):
        t, kk, pp, mm = (a[r] if a is not None else d for a, d in ((T, 1.0), (k, 0), (p, 1.0), (m, 0.0)))
        i = int(ids[r])
        if t <= 0 or kk == 1:
            clean = np.where(np.isnan(x[r]), -np.inf, x[r])
            assert i == int(np.argmax(clean)), r
            continue
        may, must = _kept(x[r], t, kk, pp, mm, EPS), _kept(x[r], t, kk, pp, mm, -EPS)
        assert may[i] > 0, (r, i)
        # u between the running totals in front of and behind the pick, whichever of the doubtful tokens are kept
        doubt = (may.sum() - must.sum()) / must.sum() + EPS
        total = must.sum()
        lo, hi = (must[:i].sum() - EPS * total) / may.sum(), (may[:i + 1].sum() + EPS * total) / total
        assert lo - doubt <= u[r] <= hi + doubt, (r, i, lo, float(u[r]), hi)
        assert abs(prob[r] - may[i] / total) <= (doubt + 1e-5) * max(prob[r], 1e-30) + 1e-9, r


def _run(accel, x, u, T=None, k=None, p=None, m=None, gap=0):
    rows, v = x.shape
    with R.Dev(accel) as dev:
        put = lambda a, t: None if a is None else dev.put(np.asarray(a, t))
        full = np.full((rows, v + gap), 1e9, np.float32)   # between the rows: larger than any logit
        full[:, :v] = x
        ids, prob = dev.put(np.full(rows, -1, np.int32)), dev.put(np.full(rows, -1, np.float32))
        accel.sample_dev(dev.put(full), rows, v, dev.put(np.asarray(u, np.float32)), ids, temperature=put(T, np.float32), top_k=put(k, np.int32),
                         top_p=put(p, np.float32), min_p=put(m, np.float32), prob=prob, ld=v + gap)
        return dev.get(ids, rows, np.int32), dev.get(prob, rows)


@pytest.mark.parametrize("v,gap", [(1, 0), (2, 0), (63, 1), (64, 0), (65, 3), (1000, 0), (4097, 5), (32000, 0), (50001, 7)])
@pytest.mark.parametrize("what", ["free", "temperature", "top_k", "top_p", "min_p", "all"])
def test_picks(accel, v, gap, what):
    rng = np.random.default_rng(v + len(what))
    rows = 24 if v < 5000 else 6
    x = (rng.standard_normal((rows, v)) * 2.5).astype(np.float32)
    x[:, rng.integers(0, v, 5)] += 6
    u = rng.random(rows, dtype=np.float32)
    u[0] = 0.0
    u[-1] = np.float32(1 - 2.0 ** -24)
    T = rng.uniform(0.3, 1.7, rows).astype(np.float32) if what in ("temperature", "all") else None
    k = rng.integers(0, max(2, min(v, 300)) + 3, rows).astype(np.int32) if what in ("top_k", "all") else None
    p = rng.uniform(0.05, 1.02, rows).astype(np.float32) if what in ("top_p", "all") else None
    m = rng.uniform(0.0, 0.3, rows).astype(np.float32) if what in ("min_p", "all") else None
    ids, prob = _run(accel, x, u, T, k, p, m, gap)
    _check(x, ids, prob, u, T, k, p, m)


@pytest.mark.parametrize("rows,v", [(1, 262144), (1, 151937), (3, 100000), (40, 30000), (300, 3001)])
def test_rows_of_every_number(accel, rows, v):
    """The same rows in calls of other sizes give the same picks and probabilities, bit for bit."""
    rng = np.random.default_rng(rows)
    x = (rng.standard_normal((rows, v)) * 2).astype(np.float32)
    u = rng.random(rows, dtype=np.float32)
    T = np.where(np.arange(rows) % 5 == 4, 0, 0.9).astype(np.float32)
    k = np.where(np.arange(rows) % 3 == 1, 50, 0).astype(np.int32)
    p = np.where(np.arange(rows) % 2 == 0, 0.9, 1.0).astype(np.float32)
    ids, prob = _run(accel, x, u, T, k, p)
    _check(x[:8], ids, prob, u, T, k, p, None)
    for a, b in ((0, 1), (rows // 2, rows)):
        i2, p2 = _run(accel, x[a:b], u[a:b], T[a:b], k[a:b], p[a:b])
        assert np.array_equal(i2, ids[a:b]) and np.array_equal(p2, prob[a:b])


def test_equal_logits_lowest_index_first(accel):
    v = 3000
    x = np.zeros((6, v), np.float32)
    x[:, 1::2] = -0.0                        # equal to +0
    u = np.array([0, 0.5, 0.999, 0.25, 0.75, 0.5], np.float32)
    k = np.array([10, 10, 10, 0, 0, 1], np.int32)
    p = np.array([1, 1, 1, 0.1, 0.1, 1], np.float32)
    ids, prob = _run(accel, x, u, k=k, p=p)
    assert ids.tolist() == [0, 5, 9, 75, 225, 0]
    # (0.1 in fp32 times 3000 is a little over 300: the token with 300 in front of it stays)
    assert prob.tolist() == [np.float32(0.1)] * 3 + [np.float32(1 / 301)] * 2 + [1.0]
    # ties at the cut of top_k: of the 7 tokens at 2.0 the two with the lowest indices stay
    x = np.zeros((1, 500), np.float32)
    x[0, [5, 90, 91, 200, 300, 301, 499]] = 2
    x[0, [400, 10, 77]] = 3
    picks = {int(_run(accel, x, [w], k=[5])[0][0]) for w in np.linspace(0, 0.9999, 60)}
    assert picks == {5, 10, 77, 90, 400}


def test_masked_and_extreme_logits(accel):
    inf, nan, low = np.inf, np.nan, np.finfo(np.float32).min
    x = np.full((8, 700), -inf, np.float32)
    x[0, 300] = 1                                         # one token left by the mask
    x[1] = nan                                            # none
    x[2] = -inf                                           # none
    x[3] = low; x[3, 699] = 0                             # the type's lowest value as the mask
    x[4] = nan; x[4, [7, 9]] = 2                          # NaN among logits
    x[5] = 0; x[5, [100, 600]] = inf                      # +inf takes everything, in equal shares
    x[6] = low                                            # every token masked by the lowest value: equal
    x[7] = 3e38; x[7, 5] = -3e38                          # differences beyond fp32
    u = np.array([0.7, 0.5, 0.5, 0.99, 0.6, 0.6, 0.5, 0.0], np.float32)
    for p in (None, np.full(8, 0.9999, np.float32)):
        ids, prob = _run(accel, x, u, p=p)
        assert ids.tolist()[:6] == [300, 0, 0, 699, 9, 600]
        assert prob.tolist()[:6] == [1.0, 0.0, 0.0, 1.0, 0.5, 0.5]
        assert abs(int(ids[6]) - 350) <= 1 and ids[7] == 0
    ids, prob = _run(accel, x, u, T=np.zeros(8, np.float32))
    assert ids.tolist() == [300, 0, 0, 699, 7, 100, 0, 0] and prob.tolist() == [1, 0, 0, 1, 1, 1, 1, 1]


def test_extreme_parameters(accel):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((8, 900)).astype(np.float32)
    best = x.argmax(1)
    one = np.ones(8, np.float32)
    u = np.full(8, 0.9, np.float32)
    assert np.array_equal(_run(accel, x, u, p=0 * one)[0], best)              # top_p 0 keeps the first
    assert np.array_equal(_run(accel, x, u, p=-one)[0], best)
    assert np.array_equal(_run(accel, x, u, m=2 * one)[0], best)              # more than any share: the largest stay
    assert np.array_equal(_run(accel, x, u, T=1e-6 * one)[0], best)
    assert np.array_equal(_run(accel, x, u, k=np.full(8, 5000))[0], _run(accel, x, u)[0])   # more than there are
    assert np.array_equal(_run(accel, x, u, T=-one)[0], best)
    last = _run(accel, np.zeros((2, 900), np.float32), [1.0, 7.5])[0]        # u outside [0, 1) stays inside the row
    assert last.tolist() == [899, 899]
    assert _run(accel, np.zeros((2, 900), np.float32), [-1.0, np.nan])[0].tolist() == [0, 0]


def test_graph_and_lm_head(accel, pkg, synth):
    rng = np.random.default_rng(4)
    n, kdim, m = 5000, 512, 3
    raw = synth.make_weight(8, n, kdim, seed=8)
    assert accel.upload_q8_0("t.sample", raw, kdim, n)
    xs = synth.make_acts(m, kdim, seed=2)
    u = np.array([0.1, 0.5, 0.9], np.float32)
    ids, prob = accel.lm_head_sample_rows("t.sample", xs, m, u, temperature=0.8, top_k=[0, 40, 1], top_p=0.95)
    assert accel.lm_head_sample_rows("t.nothing", xs, m, u) is None
    with pytest.raises(pkg.SmxError):
        accel.lm_head_sample_rows("t.sample", xs[:, :256].copy(), m, u)
    assert np.array_equal(accel.lm_head_sample_rows("t.sample", xs, m, u, temperature=0.0)[0], accel.lm_head_argmax_rows("t.sample", xs, m))
    with R.Dev(accel) as dev:
        xd, logits, idp, pp = dev.put(xs), dev.room(m * n * 4), dev.room(m * 4), dev.room(m * 4)
        up, tp, kp, pt = dev.put(u), dev.put(np.full(m, 0.8, np.float32)), dev.put(np.array([0, 40, 1], np.int32)), dev.put(np.full(m, 0.95, np.float32))

        def step():
            assert accel.gemv_dev("t.sample", xd, m, logits)
            accel.sample_dev(logits, m, n, up, idp, temperature=tp, top_k=kp, top_p=pt, prob=pp)

        step()
        assert np.array_equal(dev.get(idp, m, np.int32), ids) and np.array_equal(dev.get(pp, m), prob)
        accel.sync()
        accel.graph_begin()
        step()
        g = accel.graph_end()
        for i in range(4):
            xs2, u2 = synth.make_acts(m, kdim, seed=20 + i), rng.random(m, dtype=np.float32)
            accel.h2d(xd, xs2)
            accel.h2d(up, u2)
            accel.graph_launch(g)
            got = dev.get(idp, m, np.int32), dev.get(pp, m)
            want = accel.lm_head_sample_rows("t.sample", xs2, m, u2, temperature=0.8, top_k=[0, 40, 1], top_p=0.95)
            assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]), i
        accel.graph_destroy(g)


def test_refusals(accel, pkg):
    with R.Dev(accel) as dev:
        p = dev.room(1 << 16)
        accel.sample_dev(p, 0, 100, p, p)
        for a in ((None, 1, 100, p, p), (p, 1, 100, None, p), (p, 1, 100, p, None), (p, 1, 0, p, p), (p, 1, 1 << 23, p, p), (p, 1 << 25, 4, p, p)):
            with pytest.raises(pkg.SmxError):
                accel.sample_dev(*a)
        with pytest.raises(pkg.SmxError):
            accel.sample_dev(p, 2, 100, p, p, ld=99)


@pytest.mark.parametrize("v", [700, 9000, 40000])
@pytest.mark.parametrize("levels", [1, 3, 400])
def test_many_equal_logits(accel, v, levels):
    """Logits of a few levels (as bf16 logits of a large vocabulary are): cuts inside thousands of equal tokens, by index."""
    rng = np.random.default_rng(v + levels)
    rows = 16
    x = (rng.integers(0, levels, (rows, v)) * (6.0 / max(1, levels - 1))).astype(np.float32)
    u = rng.random(rows, dtype=np.float32)
    k = np.array([0, 0, 0, 0, 2, 100, 255, 256, 257, 600, 3000, 4096, 4097, 8000, v - 1, v], np.int32)
    p = np.array([0.05, 0.5, 0.95, 1, 1, 0.5, 0.9, 1, 0.3, 0.7, 1, 0.6, 1, 0.8, 1, 0.2], np.float32)
    T = np.where(np.arange(rows) % 2 == 0, 1.0, 2.5).astype(np.float32)
    m = np.where(np.arange(rows) % 5 == 3, 0.01, 0.0).astype(np.float32)
    ids, prob = _run(accel, x, u, T, k, p, m, gap=v % 3)
    _check(x, ids, prob, u, T, k, p, m)


def test_cut_far_below_the_largest(accel):
    """top_k reaches past a gap of hundreds between logits."""
    rng = np.random.default_rng(8)
    v = 6000
    x = rng.standard_normal((4, v)).astype(np.float32)
    x[:, 17] = 300
    x[2:, 40:] -= 1000
    k = np.array([50, 5000, 30, 4500], np.int32)
    T = np.full(4, 100.0, np.float32)
    u = np.array([0.3, 0.99, 0.6, 0.9], np.float32)
    ids, prob = _run(accel, x, u, T, k)
    _check(x, ids, prob, u, T, k, None, None)
