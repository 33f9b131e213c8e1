"""The paged 8-bit key/value cache and the attention over it in numpy: the layout, the append in the fp32 operations that its
definition names (so codes and scales compare exactly), attention in 64 bits."""
import numpy as np

BLOCK = 32
F = np.float32


def bf16(x):
    """fp32 -> bf16 bits, round to nearest even."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def from_bf16(b):
    return (np.asarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32)


def k_byte(dim64, t, d):
    return ((t // 16) * (dim64 // 64) + d // 64) * 1024 + (d // 16 % 4) * 256 + (t % 16) * 16 + d % 16


def v_byte(t, d):
    return (d // 32) * 1024 + (t // 4 % 4) * 256 + (d % 16) * 16 + (d // 16 % 2) * 8 + (t // 16) * 4 + t % 4


class Cache:
    """Planes of a cache; unused codes and scales are whatever they are (NaN scales, to show that nothing reads them)."""

    def __init__(self, pages, page, heads, dim, seed=0):
        self.pages, self.page, self.heads, self.dim = pages, page, heads, dim
        self.dim64 = (dim + 63) // 64 * 64
        rng = np.random.default_rng(seed)
        blocks = page // BLOCK
        self.k, self.v = (rng.integers(-128, 128, (pages, heads, blocks, BLOCK * self.dim64)).astype(np.int8) for _ in range(2))
        self.ks, self.vs = (np.full((pages, heads, blocks), np.nan, np.float32) for _ in range(2))
        t, d = np.meshgrid(np.arange(BLOCK), np.arange(dim), indexing="ij")
        self.at = {"k": k_byte(self.dim64, t, d), "v": v_byte(t, d)}

    def block(self, which, page, head, blk):
        """Codes [32][dim] (a copy) and the scale of one block."""
        plane, scale = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        return plane[page, head, blk][self.at[which]], scale[page, head, blk]

    def put(self, which, page, head, blk, codes, scale):
        plane, scales = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        plane[page, head, blk][self.at[which]] = codes
        scales[page, head, blk] = scale

    def tokens(self, which, table, head, n):
        """Stored values (fp32) of the first n tokens of a sequence with page list `table`: [n][dim]."""
        out = np.zeros((n, self.dim), np.float32)
        for b in range(-(-n // BLOCK)):
            codes, scale = self.block(which, table[b * BLOCK // self.page], head, b % (self.page // BLOCK))
            m = min(BLOCK, n - b * BLOCK)
            out[b * BLOCK:b * BLOCK + m] = codes[:m].astype(F) * scale
        return out


def rope_table(n_pos, rot, base=1e4):
    ang = np.arange(n_pos, dtype=np.float64)[:, None] * base ** (-np.arange(0, rot, 2) / rot)
    return np.stack([np.cos(ang), np.sin(ang)], -1).astype(np.float32)


def rotate(x, table, pos, rot, interleaved):
    """x [rows][heads][dim] fp32; every product and sum rounded by itself."""
    x = x.astype(np.float32)
    y = x.copy()
    c, s = table[pos][:, None, :, 0], table[pos][:, None, :, 1]
    a, b = (np.arange(0, rot, 2), np.arange(1, rot, 2)) if interleaved else (np.arange(rot // 2), np.arange(rot // 2) + rot // 2)
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    return y


def append(cache, table, old, new, k, v):
    """Rows of every sequence in turn: k (rotated), v [rows][heads][dim] fp32; old, new: tokens before, rows of each sequence."""
    r = 0
    for s, (o, n) in enumerate(zip(old, new)):
        for which, x in (("k", k), ("v", v)):
            for h in range(cache.heads):
                for b in range(o // BLOCK, (o + n - 1) // BLOCK + 1 if n else 0):
                    t0, t1 = max(o - b * BLOCK, 0), min(o + n - b * BLOCK, BLOCK)
                    rows = x[r + b * BLOCK + t0 - o:r + b * BLOCK + t1 - o, h]
                    page, blk = table[s][b * BLOCK // cache.page], b % (cache.page // BLOCK)
                    codes, before = cache.block(which, page, h, blk)
                    with np.errstate(all="ignore"):
                        top = np.abs(rows).max() if np.isfinite(rows).all() else np.nan
                        fresh = F(np.nan) if np.isnan(top) else top / F(127) if top >= F(2.0 ** -96) else F(0)
                        scale = fresh
                        if t0:
                            if np.isnan(before) or np.isnan(fresh):
                                scale = F(np.nan)
                            elif before < fresh:
                                codes[:t0] = np.rint(codes[:t0].astype(F) * (before / fresh)).astype(np.int8)
                            else:
                                scale = before
                        inv = F(1) / scale if scale > 0 else F(0)
                        c = np.rint(rows * inv)
                        codes[t0:t1] = np.where(np.isnan(c), 0, np.clip(c, -127, 127)).astype(np.int8)
                    cache.put(which, page, h, blk, codes, scale)
        r += n


def attend(cache, table, lens, new, q, scale, window=0):
    """q [rows][heads][dim] -> fp64 [rows][heads][dim]; rows are the last new[s] tokens of each sequence."""
    out = np.zeros(q.shape, np.float64)
    group = q.shape[1] // cache.heads
    r = 0
    for s, (length, n) in enumerate(zip(lens, new)):
        for kvh in range(cache.heads if n and length else 0):
            k = cache.tokens("k", table[s], kvh, length).astype(np.float64)
            v = cache.tokens("v", table[s], kvh, length).astype(np.float64)
            for j in range(n):
                pos = length - n + j
                lo = max(0, pos - window + 1) if window else 0
                if pos < 0:
                    continue
                for h in range(kvh * group, (kvh + 1) * group):
                    sc = k[lo:pos + 1] @ q[r + j, h].astype(np.float64) * scale
                    p = np.exp(sc - sc.max())
                    out[r + j, h] = p @ v[lo:pos + 1] / p.sum()
        r += n
    return out


class Dev:
    """Arrays on the device through a context; freed together."""

    def __init__(self, acc):
        self.acc, self.ptrs = acc, []

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.acc.sync()
        for p in self.ptrs:
            self.acc.dev_free(p)

    def room(self, nbytes):
        p = self.acc.dev_alloc(max(int(nbytes), 16))
        self.ptrs.append(p)
        return p

    def put(self, a):
        a = np.ascontiguousarray(a)
        p = self.room(a.nbytes)
        if a.nbytes:
            self.acc.h2d(p, a)
        return p

    def get(self, p, shape, dtype=np.float32):
        return self.acc.d2h(np.empty(shape, dtype), p)


class OnDevice:
    """A Cache's planes on the device, and the batches over them."""

    def __init__(self, pkg, dev, cache):
        self.pkg, self.dev, self.host = pkg, dev, cache
        self.p = [dev.put(x) for x in (cache.k, cache.v, cache.ks, cache.vs)]
        self.handle = pkg.KvCache(cache.pages, cache.page, cache.heads, cache.dim, *self.p)

    def batch(self, table, lens, new, max_len=None, always_row0=False):
        new, lens = list(new), list(lens)
        row0 = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        plain = all(n == 1 for n in new) and not always_row0
        t = np.asarray(table, np.int32)
        b = self.pkg.KvBatch(len(new), self.dev.put(np.asarray(lens, np.int32)), self.dev.put(t), t.shape[1], max(lens) if max_len is None else max_len,
                             row0=None if plain else self.dev.put(row0), rows=int(row0[-1]), max_rows=max(new) if not plain else 1)
        return b

    def planes(self):
        c = self.host
        return [self.dev.get(p, x.shape, x.dtype) for p, x in zip(self.p, (c.k, c.v, c.ks, c.vs))]


def tables(rng, pages, page, lens, spare=1):
    """Page lists that share no page, in random order; entries behind a sequence's last page name none."""
    need = [-(-n // page) for n in lens]
    assert sum(need) <= pages
    order = rng.permutation(pages)
    t = np.full((len(lens), max(need + [1]) + spare), -7, np.int32)
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = order[at:at + n]
        at += n
    return t
