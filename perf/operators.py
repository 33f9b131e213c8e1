"""Cases of the operators around a paged key/value cache and of the sampler behind the lm_head: what a decode or prefill step
of a language model does between its projections.

    listed()             the named cases
    draw(rng)            one more case of the same ranges
    prepare(case, seed)  what a serving program has in hand before the call: activations, the cache, page tables, buffers
    run(state)           one pass of the call(s); returns its outputs
    exact(case, seed)    the same outputs from the definitions, in 64 bits
    work(case)           bytes and operations that a pass cannot do without

`own` says whose arithmetic `run` is: the library's calls, or the same operators in elementary torch operations.

Kinds of case:
    append  a step's new keys and values (and queries) take their position rotation, the keys and values go into the cache in
            8 bits, and the blocks that they touched are read back as fp32 values
    attend  attention of a step's query rows over the cache
    sample  one token for each row of logits, by temperature, top-k, top-p and min-p from given uniform numbers

The cache is int8 codes with one fp32 scale for each block of 32 tokens and key/value head; a page holds page_tokens tokens of
every head (a multiple of 32).  Its planes, dim = head_dim rounded up to 64:
    keys    [page][head][block][token / 16][d / 64][d / 16 % 4][token % 16][d % 16]
    values  [page][head][block][d / 32][token / 4 % 4][d % 16][d / 16 % 2][token / 16][token % 4]
    scales  [page][head][block], one plane for keys and one for values
"""
import importlib.util
import math
import os
import sys

import torch

own = False

BLOCK = 32                 # tokens that share a scale
TINY = 2.0 ** -96          # a block whose largest value is below this is stored as zeros
ONE = float(1 << 40)       # weight of the likeliest token in the sampler's whole-number weights
BASE = 1e4                 # of the position rotation


# ---- the cases

def listed():
    return [
        # one token of one conversation: nothing but latency
        {"name": "append_token", "kind": "append", "nseq": 1, "lo": 777, "hi": 777, "new": 1, "heads": 32, "kv": 8, "dim": 128, "rot": 128,
         "pairs": False, "page": 64, "type": "f32"},
        # a decode step of 64 conversations of different lengths
        {"name": "append_batch", "kind": "append", "nseq": 64, "lo": 0, "hi": 4001, "new": 1, "heads": 32, "kv": 8, "dim": 128, "rot": 128,
         "pairs": False, "page": 64, "type": "f32"},
        # a prompt chunk that goes on inside a block, rotated in neighbouring pairs over part of the head
        {"name": "append_prompt", "kind": "append", "nseq": 1, "lo": 1003, "hi": 1003, "new": 2048, "heads": 16, "kv": 8, "dim": 256, "rot": 64,
         "pairs": True, "page": 256, "type": "bf16"},
        # one token of one short conversation: nothing but latency
        {"name": "attend_token", "kind": "attend", "nseq": 1, "lo": 601, "hi": 601, "new": 1, "heads": 32, "kv": 8, "dim": 128, "window": 0,
         "page": 64, "type": "f32"},
        # one token of one very long conversation
        {"name": "attend_long", "kind": "attend", "nseq": 1, "lo": 131071, "hi": 131071, "new": 1, "heads": 32, "kv": 8, "dim": 128, "window": 0,
         "page": 256, "type": "f32"},
        # a decode step of 64 conversations of different lengths: the cache is what is read
        {"name": "attend_batch", "kind": "attend", "nseq": 64, "lo": 33, "hi": 8192, "new": 1, "heads": 32, "kv": 8, "dim": 128, "window": 0,
         "page": 64, "type": "f32"},
        # a layer with a sliding window and wide heads, bf16 activations
        {"name": "attend_window", "kind": "attend", "nseq": 96, "lo": 100, "hi": 4000, "new": 1, "heads": 16, "kv": 8, "dim": 256, "window": 1024,
         "page": 32, "type": "bf16"},
        # a few drafted tokens of several conversations are checked at once; a head size that is no power of two
        {"name": "attend_verify", "kind": "attend", "nseq": 5, "lo": 1500, "hi": 3333, "new": 6, "heads": 20, "kv": 4, "dim": 80, "window": 0,
         "page": 96, "type": "bf16"},
        # a prompt chunk behind an earlier part of the same prompt: the largest work
        {"name": "attend_prompt", "kind": "attend", "nseq": 1, "lo": 6000, "hi": 6000, "new": 2048, "heads": 32, "kv": 8, "dim": 128, "window": 0,
         "page": 64, "type": "f32"},
        # one row of a large vocabulary with every filter on
        {"name": "sample_token", "kind": "sample", "rows": 1, "vocab": 262144, "temps": "one", "top_k": 40, "top_p": 0.95, "min_p": 0.05},
        # a batch whose rows ask for different things, greedy ones and unfiltered ones among them; an odd vocabulary
        {"name": "sample_mixed", "kind": "sample", "rows": 48, "vocab": 49999, "temps": "mixed", "top_k": 100, "top_p": 0.9, "min_p": 0.02},
        # a large batch over a large vocabulary, cut by probability alone
        {"name": "sample_batch", "kind": "sample", "rows": 256, "vocab": 262144, "temps": "mixed", "top_k": 0, "top_p": 0.9, "min_p": 0.0},
    ]


def _log(rng, lo, hi, step=1):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step))


def draw(rng):
    """A case of the same ranges: sizes spread over their logarithm, odd ones among them."""
    kind = rng.choice(("append", "attend", "attend", "sample"))
    if kind == "sample":
        vocab = _log(rng, 5000, 262144)
        return {"kind": kind, "rows": _log(rng, 1, min(256, 67108864 // vocab)), "vocab": vocab, "temps": rng.choice(("one", "mixed")),
                "top_k": rng.choice((0, _log(rng, 1, 2000))), "top_p": rng.choice((1.0, round(rng.uniform(0.2, 0.99), 3))),
                "min_p": rng.choice((0.0, round(rng.uniform(0.001, 0.3), 3)))}
    for _ in range(1000):
        kv, group = rng.randint(1, 8), rng.choice((1, 2, 3, 4, 5, 8))
        dim = rng.choice((64, 80, 96, 128, 128, 192, 256))
        c = {"kind": kind, "nseq": 1, "lo": 0, "hi": 0, "new": 1, "heads": kv * group, "kv": kv, "dim": dim}
        shape = rng.choice(("decode", "verify", "prompt"))
        if shape == "decode":
            c["nseq"] = _log(rng, 1, 96)
        elif shape == "verify":
            c.update(nseq=_log(rng, 1, 16), new=rng.randint(2, 12))
        else:
            c.update(nseq=rng.randint(1, 3), new=_log(rng, 13, 2048))
        most = 131071 if shape == "decode" else 8192
        c["hi"] = _log(rng, 1, most)
        c["lo"] = c["hi"] if c["nseq"] == 1 else int(c["hi"] * rng.uniform(0.0, 1.0))
        c["page"] = rng.choice((32, 64, 96, 128, 256))
        c["type"] = rng.choice(("f32", "bf16"))
        if kind == "append":
            c.update(rot=rng.choice((dim, dim // 2)), pairs=rng.random() < 0.5)
        else:
            c["window"] = rng.choice((0, 0, _log(rng, 16, 4096)))
        if c["nseq"] * (c["hi"] + c["new"]) * kv * dim <= 5.4e8 and c["nseq"] * c["new"] * c["heads"] * (c["hi"] + c["new"]) <= 5.3e8:
            return c
    raise AssertionError("no case of these ranges")


def _spread(n, lo, hi):
    """n whole numbers between lo and hi in no order."""
    return [lo + (hi - lo) * ((i * 37 + 11) % n) // max(1, n - 1) for i in range(n)]


def _shape(c):
    """(tokens in the cache before the call, new rows) of each sequence; the new rows differ by up to an eighth."""
    old = _spread(c["nseq"], c["lo"], c["hi"])
    new = [max(1, c["new"] - (c["new"] * ((i * 5) % 8)) // 64) for i in range(c["nseq"])]
    return old, new


# ---- what a serving program has in hand before the call

class State:
    pass


def prepare(case, seed):
    c = case
    s = State()
    s.case = c
    gen = torch.Generator("cuda").manual_seed(seed)
    if c["kind"] == "sample":
        return _prepare_sample(s, c, gen)
    dt = torch.float32 if c["type"] == "f32" else torch.bfloat16
    old, new = _shape(c)
    s.rows, s.max_rows, s.max_len = sum(new), max(new), max(o + n for o, n in zip(old, new))
    s.dim64 = (c["dim"] + 63) // 64 * 64
    per = -(-s.max_len // c["page"])
    used = [-(-(o + n) // c["page"]) for o, n in zip(old, new)]
    s.npages = sum(used) + 3
    order = torch.randperm(s.npages, device="cuda", generator=gen).to(torch.int32)
    table, at = torch.full((c["nseq"], per), -1, dtype=torch.int32, device="cuda"), 0
    for i, n in enumerate(used):
        table[i, :n] = order[at:at + n]
        at += n
    s.table = table
    s.len = torch.tensor([o + n for o, n in zip(old, new)], dtype=torch.int32, device="cuda")
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s.row0 = torch.tensor(starts, dtype=torch.int32, device="cuda")
    blocks = c["page"] // BLOCK
    n = s.npages * c["kv"] * blocks
    bytes_per = BLOCK * s.dim64
    s.k, s.v = (_codes(n, bytes_per, gen).view(s.npages, -1) for _ in range(2))
    s.ks, s.vs = ((torch.rand(s.npages, c["kv"], blocks, device="cuda", generator=gen) + 0.5) * 0.03 for _ in range(2))
    # queries, keys and values as the rows of one fused projection
    h, kv, d = c["heads"], c["kv"], c["dim"]
    s.qkv = torch.randn(s.rows, (h + 2 * kv) * d, device="cuda", generator=gen).to(dt)
    s.q, s.k_new, s.v_new = s.qkv[:, :h * d], s.qkv[:, h * d:(h + kv) * d], s.qkv[:, (h + kv) * d:]
    if c["kind"] == "attend":
        s.q *= 1 + torch.arange(h, device="cuda").repeat_interleave(d).to(dt) % 3   # some heads look at few tokens, some at many
        s.out = torch.empty(s.rows, h, d, dtype=dt, device="cuda")
    else:
        angle = torch.arange(s.max_len, device="cuda", dtype=torch.float64)[:, None] * BASE ** (
            -torch.arange(0, c["rot"], 2, device="cuda", dtype=torch.float64) / c["rot"])
        s.rope = torch.stack([angle.cos(), angle.sin()], -1).float()
        s.q_out = torch.empty(s.rows, h, d, dtype=dt, device="cuda")
        # what is read back: the tokens of every block that the call touches
        back = [n + o % BLOCK for o, n in zip(old, new)]
        s.back, s.max_back = sum(back), max(back)
        ends = [0]
        for n in back:
            ends.append(ends[-1] + n)
        s.back0 = torch.tensor(ends, dtype=torch.int32, device="cuda")
        s.k_out, s.v_out = (torch.empty(s.back, kv, d, device="cuda") for _ in range(2))
    return s


def _codes(blocks, nbytes, gen):
    """Codes as keys and values leave them: normal values whose largest of a block is near 127."""
    return (torch.randn(blocks, nbytes, device="cuda", generator=gen) * 34).round_().clamp_(-127, 127).to(torch.int8)


def _prepare_sample(s, c, gen):
    rows, v = c["rows"], c["vocab"]
    # a head of likely tokens over a broad body, as a model's logits are
    s.logits = torch.randn(rows, v, device="cuda", generator=gen) * 2.2
    hot = torch.randint(0, v, (rows, 32), device="cuda", generator=gen)
    s.logits.scatter_add_(1, hot, torch.rand(rows, 32, device="cuda", generator=gen) * 9)
    s.u = torch.rand(rows, device="cuda", generator=gen)
    one = torch.ones(rows, device="cuda")
    i = torch.arange(rows, device="cuda")
    if c["temps"] == "one":
        s.temperature, on = one * 0.8, torch.ones(rows, dtype=torch.bool, device="cuda")
    else:
        s.temperature = torch.where(i % 8 == 3, 0.0, 0.5 + torch.rand(rows, device="cuda", generator=gen))
        on = i % 4 != 1
    s.top_k = torch.where(on, c["top_k"], 0).to(torch.int32)
    s.top_p = torch.where(on, c["top_p"], 1.0).float()
    s.min_p = torch.where(on, c["min_p"], 0.0).float()
    s.ids, s.prob = torch.empty(rows, dtype=torch.int32, device="cuda"), torch.empty(rows, device="cuda")
    return s


# ---- one pass

def run(s):
    kind = s.case["kind"]
    if own:
        return {"append": _own_append, "attend": _own_attend, "sample": _own_sample}[kind](s)
    return {"append": _append, "attend": _attend, "sample": _sample}[kind](s)


# ---- the library's calls

_ACC = []


def _lib():
    """The package and the process's one context (a serving program keeps one per device)."""
    if not _ACC:
        name, here = "strix_rs_amd", os.path.join(os.getcwd(), "strix.rs_amd")
        if name not in sys.modules:
            spec = importlib.util.spec_from_file_location(name, os.path.join(here, "__init__.py"), submodule_search_locations=[here])
            mod = importlib.util.module_from_spec(spec)
            sys.modules[name] = mod
            spec.loader.exec_module(mod)
        _ACC.extend((sys.modules[name], sys.modules[name].Mi355WeightAccel(0)))
    return _ACC


def _handles(s):
    """The descriptions of cache, batch and rotation that a program makes once and passes to every layer's calls."""
    if not hasattr(s, "cache"):
        pkg, _ = _lib()
        c = s.case
        s.cache = pkg.KvCache(s.npages, c["page"], c["kv"], c["dim"], s.k.data_ptr(), s.v.data_ptr(), s.ks.data_ptr(), s.vs.data_ptr())
        row0 = None if s.rows == c["nseq"] else s.row0.data_ptr()
        s.batch = pkg.KvBatch(c["nseq"], s.len.data_ptr(), s.table.data_ptr(), s.table.shape[1], s.max_len, row0=row0, rows=s.rows, max_rows=s.max_rows)
        s.dtype = pkg.DTYPE_F32 if c["type"] == "f32" else pkg.DTYPE_BF16
        if c["kind"] == "append":
            s.turn = pkg.Rope(s.rope.data_ptr(), s.rope.shape[0], c["rot"], interleaved=c["pairs"])
            s.touched = pkg.KvBatch(c["nseq"], s.len.data_ptr(), s.table.data_ptr(), s.table.shape[1], s.max_len, row0=s.back0.data_ptr(), rows=s.back,
                                    max_rows=s.max_back)


def _own_append(s):
    _handles(s)
    acc, ld = _ACC[1], s.qkv.shape[1]
    acc.kv_append_dev(s.cache, s.batch, s.k_new.data_ptr(), s.v_new.data_ptr(), rope=s.turn, q=s.q.data_ptr(), q_heads=s.case["heads"],
                      q_out=s.q_out.data_ptr(), dtype=s.dtype, ldk=ld, ldv=ld, ldq=ld)
    acc.kv_read_dev(s.cache, s.touched, s.k_out.data_ptr(), s.v_out.data_ptr())
    return {"q": s.q_out, "k": s.k_out, "v": s.v_out}


def _own_attend(s):
    _handles(s)
    c = s.case
    _ACC[1].attn_dev(s.cache, s.batch, s.q.data_ptr(), c["heads"], c["dim"] ** -0.5, s.out.data_ptr(), window=c["window"], dtype=s.dtype, ldq=s.qkv.shape[1])
    return s.out


def _own_sample(s):
    c = s.case
    _lib()[1].sample_dev(s.logits.data_ptr(), c["rows"], c["vocab"], s.u.data_ptr(), s.ids.data_ptr(), temperature=s.temperature.data_ptr(),
                         top_k=s.top_k.data_ptr(), top_p=s.top_p.data_ptr(), min_p=s.min_p.data_ptr(), prob=s.prob.data_ptr())
    return {"id": s.ids, "prob": s.prob}


# ---- the plain forms

def _positions(row0, length, rows):
    """(sequence, position) of each of `rows` rows, the last ones of their sequences."""
    r = torch.arange(rows, device=row0.device)
    seq = torch.searchsorted(row0[1:].contiguous(), r.to(torch.int32), right=True)
    return seq, (length[seq] - row0[seq + 1]).long() + r


def _k_view(s):
    """Keys as [block][token / 16][d / 64][d / 16 % 4][token % 16][d % 16]."""
    return s.k.view(-1, 2, s.dim64 // 64, 4, 16, 16)


def _v_view(s):
    """Values as [block][d / 32][token / 4 % 4][d % 16][d / 16 % 2][token / 16][token % 4]."""
    return s.v.view(-1, s.dim64 // 32, 4, 16, 2, 2, 4)


def _plain_blocks(s, which, index):
    """fp32 values of the cache's blocks `index` ([...]): [..., 32 tokens, dim64]."""
    c = s.case
    if which == "k":
        x = _k_view(s)[index].movedim(-2, -4).reshape(*index.shape, BLOCK, s.dim64)
        scale = s.ks.view(-1)[index]
    else:
        x = _v_view(s)[index]                       # [..., d32, t4, d1, d16, t16, t1]
        n = index.dim()
        x = x.permute(*range(n), n + 4, n + 1, n + 5, n, n + 3, n + 2).reshape(*index.shape, BLOCK, s.dim64)
        scale = s.vs.view(-1)[index]
    return x.float() * scale[..., None, None]


def _block_index(s, seq, pos):
    """Block (of all heads' blocks of the cache) of head 0 of a sequence's token, and the step to the next head's."""
    c = s.case
    blocks = c["page"] // BLOCK
    page = s.table[seq, pos // c["page"]].long()
    return page * c["kv"] * blocks + pos % c["page"] // BLOCK, blocks


def _rotate(x, rope, pos, rot, pairs):
    """x [rows][heads][dim] in fp32; every product and sum is rounded by itself."""
    cos, sin = (rope[pos][:, None, :, i] for i in range(2))
    part = x[..., :rot]
    a, b = (part[..., 0::2], part[..., 1::2]) if pairs else (part[..., :rot // 2], part[..., rot // 2:])
    lo, hi = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([lo, hi], -1).reshape(part.shape) if pairs else torch.cat([lo, hi], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _append(s):
    c = s.case
    h, kv, d = c["heads"], c["kv"], c["dim"]
    seq, pos = _positions(s.row0, s.len, s.rows)
    q = _rotate(s.q.float().view(-1, h, d), s.rope, pos, c["rot"], c["pairs"]).to(s.q.dtype)
    k = _rotate(s.k_new.float().reshape(-1, kv, d), s.rope, pos, c["rot"], c["pairs"])
    v = s.v_new.float().reshape(-1, kv, d)
    first, step = _block_index(s, seq, pos)
    index = first[:, None] + torch.arange(kv, device=k.device) * step                     # [rows][kv]
    # the block in front of each sequence's new rows may hold earlier tokens
    start = s.len.long() - (s.row0[1:] - s.row0[:-1]).long()
    every = torch.arange(c["nseq"], device=k.device)
    head, _ = _block_index(s, every, start)
    head = head[:, None] + torch.arange(kv, device=k.device) * step                       # [nseq][kv]
    kept = (start % BLOCK)[:, None].expand(-1, kv)                                        # earlier tokens in it
    tok, chan = pos % BLOCK, torch.arange(d, device=k.device)
    t, e = tok[:, None, None], chan[None, None, :]
    for plane, view, x in ((s.ks, _k_view(s), k), (s.vs, _v_view(s), v)):
        scale = plane.view(-1)
        most = torch.zeros_like(scale).scatter_reduce(0, index.view(-1), x.abs().amax(-1).view(-1), "amax")
        fresh = torch.where(most >= TINY, most / torch.full_like(most, 127.0), 0.0)
        before = torch.where(kept > 0, scale[head], 0.0)
        grown = torch.maximum(before, fresh[head])
        scale[index] = fresh[index]
        scale[head] = grown
        # earlier tokens of a block whose scale has grown are rounded again
        ratio = torch.where(before < grown, before / grown, 1.0)
        codes = view[head].float()
        view[head] = (codes * ratio[(...,) + (None,) * (codes.dim() - 2)]).round().to(torch.int8)
        sc = scale[index]
        inv = torch.where(sc > 0, 1.0 / sc, 0.0)
        code = (x * inv[..., None]).round().clamp(-127, 127).to(torch.int8)
        if view.dim() == 6:
            view[index[..., None], t // 16, e // 64, e // 16 % 4, t % 16, e % 16] = code
        else:
            view[index[..., None], e // 32, t // 4 % 4, e % 16, e // 16 % 2, t // 16, t % 4] = code
    seq, pos = _positions(s.back0, s.len, s.back)
    first, step = _block_index(s, seq, pos)
    index = first[:, None] + torch.arange(kv, device=k.device) * step
    t, e = (pos % BLOCK)[:, None, None], chan[None, None, :]
    back_k = _k_view(s)[index[..., None], t // 16, e // 64, e // 16 % 4, t % 16, e % 16].float() * s.ks.view(-1)[index][..., None]
    back_v = _v_view(s)[index[..., None], e // 32, t // 4 % 4, e % 16, e // 16 % 2, t // 16, t % 4].float() * s.vs.view(-1)[index][..., None]
    return {"q": q, "k": back_k, "v": back_v}


def _attend(s):
    c = s.case
    h, kv, d, n = c["heads"], c["kv"], c["dim"], c["nseq"]
    g, blocks = h // kv, c["page"] // BLOCK
    pages = s.table.long().clamp(min=0)                                                    # [nseq][pages]
    index = ((pages[:, None, :, None] * kv + torch.arange(kv, device=pages.device)[None, :, None, None]) * blocks
             + torch.arange(blocks, device=pages.device))                                  # [nseq][kv][pages][blocks]
    index = index.reshape(n, kv, -1)[:, :, :-(-s.max_len // BLOCK)]
    k = _plain_blocks(s, "k", index).reshape(n * kv, -1, s.dim64)[..., :d]
    seq, pos = _positions(s.row0, s.len, s.rows)
    at = torch.arange(s.rows, device=pos.device) - s.row0[seq].long()
    q = torch.zeros(n, s.max_rows, h, d, device=pos.device)
    q[seq, at] = s.q.float().view(-1, h, d)
    where = torch.full((n, s.max_rows), -1, dtype=torch.int64, device=pos.device)
    where[seq, at] = pos
    q = q.view(n, s.max_rows, kv, g, d).permute(0, 2, 1, 3, 4).reshape(n * kv, s.max_rows * g, d)
    p = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(d ** -0.5).view(n, kv, s.max_rows, g, -1)
    del k
    key = torch.arange(p.shape[-1], device=p.device)
    seen = key <= where[..., None]
    if c["window"]:
        seen &= key > where[..., None] - c["window"]
    p.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    p.sub_(p.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = p.sum(-1)
    v = _plain_blocks(s, "v", index).reshape(n * kv, -1, s.dim64)[..., :d].contiguous()
    out = torch.matmul(p.view(n * kv, s.max_rows * g, -1), v).view(n, kv, s.max_rows, g, d)
    out = torch.where(total[..., None] > 0, out / total[..., None], 0.0)
    return out.permute(0, 2, 1, 3, 4).reshape(n, s.max_rows, h, d)[seq, at].to(s.q.dtype)


def _sample(s):
    x = torch.where(torch.isnan(s.logits), -math.inf, s.logits)
    v = x.shape[1]
    greedy = s.temperature <= 0
    k = torch.where(greedy, 1, torch.where(s.top_k <= 0, v, s.top_k))
    t = torch.where(greedy, 1.0, s.temperature)
    most = x.amax(-1, keepdim=True)
    e = torch.where(x == most, 1.0, torch.exp((x - most) / t[:, None]))
    e = torch.where(x > -math.inf, e, 0.0)
    w = (e * ONE).to(torch.int64)                          # whole-number weights: their sums have one value in any order
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    rank = torch.arange(v, device=x.device)
    ws = torch.where(rank < k[:, None], ws, 0)
    total = ws.sum(-1)
    ahead = ws.cumsum(-1) - ws
    limit = (s.top_p.double() * total.double()).to(torch.int64)
    keep = (rank < k[:, None]) & ((rank == 0) | (ahead < limit[:, None]) | (s.top_p >= 1)[:, None])
    keep = torch.zeros_like(keep).scatter(1, order, keep) & (e >= s.min_p[:, None])
    w = torch.where(keep, w, 0)
    total = w.sum(-1)
    target = torch.minimum((s.u.double() * total.double()).to(torch.int64), total - 1)
    ids = (w.cumsum(-1) <= target[:, None]).sum(-1).clamp(max=v - 1)
    prob = torch.where(total > 0, w.gather(1, ids[:, None])[:, 0].double() / total.double().clamp(min=1), 0.0).float()
    return {"id": ids.to(torch.int32), "prob": prob}


# ---- the definitions in 64 bits, one sequence, head or row at a time

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["kind"]](s)


def _tokens(s, which, i, j, length):
    """Codes (as float64) and scales of the first `length` tokens of sequence i, head j: [length][dim], [length]."""
    c = s.case
    blocks, d64 = c["page"] // BLOCK, s.dim64
    pages = s.table[i, :-(-length // c["page"])].long()
    if which == "k":
        x = s.k.view(s.npages, c["kv"], blocks, 2, d64 // 64, 4, 16, 16)[pages, j]
        x = x.permute(0, 1, 2, 5, 3, 4, 6)
    else:
        x = s.v.view(s.npages, c["kv"], blocks, d64 // 32, 4, 16, 2, 2, 4)[pages, j]
        x = x.permute(0, 1, 6, 3, 7, 2, 5, 4)
    scale = (s.ks if which == "k" else s.vs)[pages, j].double().reshape(-1).repeat_interleave(BLOCK)
    return x.reshape(-1, d64)[:length, :c["dim"]].double(), scale[:length]


def _exact_append(s):
    c = s.case
    h, kv, d, rot = c["heads"], c["kv"], c["dim"], c["rot"]
    ends, lens, backs = s.row0.tolist(), s.len.tolist(), s.back0.tolist()
    half = torch.arange(rot // 2, device="cuda")
    a, b = (2 * half, 2 * half + 1) if c["pairs"] else (half, half + rot // 2)

    def turn(x, first):
        cs = s.rope[first:first + x.shape[0]].double()[:, None]
        y = x.clone()
        y[..., a] = x[..., a] * cs[..., 0] - x[..., b] * cs[..., 1]
        y[..., b] = x[..., a] * cs[..., 1] + x[..., b] * cs[..., 0]
        return y

    q_out = torch.empty(s.rows, h, d, dtype=torch.float64, device="cuda")
    outs = {w: torch.empty(s.back, kv, d, dtype=torch.float64, device="cuda") for w in "kv"}
    for i in range(c["nseq"]):
        rows, n = slice(ends[i], ends[i + 1]), ends[i + 1] - ends[i]
        start = lens[i] - n
        off = start % BLOCK
        q_out[rows] = turn(s.q[rows].double().view(n, h, d), start)
        for w, x in (("k", turn(s.k_new[rows].double().reshape(n, kv, d), start)), ("v", s.v_new[rows].double().reshape(n, kv, d))):
            padded = torch.zeros(-(-(off + n) // BLOCK) * BLOCK, kv, d, dtype=torch.float64, device="cuda")
            padded[off:off + n] = x
            scale = padded.view(-1, BLOCK, kv, d).abs().amax((1, 3)) / 127                  # [blocks][kv]
            for j in range(kv if off else 0):
                codes, before = _tokens(s, w, i, j, start)
                was = before[-1]
                scale[0, j] = torch.maximum(scale[0, j], was)
                earlier = codes[start - off:]
                padded[:off, j] = earlier * was if scale[0, j] == was else torch.round(earlier * was / scale[0, j]) * scale[0, j]
            by = scale.repeat_interleave(BLOCK, 0)[..., None].clamp(min=1e-300)
            padded[off:] = torch.round(padded[off:] / by[off:]).clamp(-127, 127) * by[off:]
            outs[w][backs[i]:backs[i + 1]] = padded[:off + n]
    return {"q": q_out, **outs}


def _exact_attend(s):
    c = s.case
    h, kv, d = c["heads"], c["kv"], c["dim"]
    g = h // kv
    ends, lens = s.row0.tolist(), s.len.tolist()
    out = torch.zeros(s.rows, h, d, dtype=torch.float64, device="cuda")
    q = s.q.double().view(-1, h, d)
    for i in range(c["nseq"]):
        n, length = ends[i + 1] - ends[i], lens[i]
        pos = torch.arange(length - n, length, device="cuda")[:, None]
        key = torch.arange(length, device="cuda")[None]
        seen = (key <= pos) & ((key > pos - c["window"]) if c["window"] else True)
        for j in range(kv):
            k, ks = _tokens(s, "k", i, j, length)
            v, vs = _tokens(s, "v", i, j, length)
            kt, v = (k * ks[:, None]).T.contiguous(), v * vs[:, None]
            for m in range(j * g, (j + 1) * g):
                score = torch.where(seen, q[ends[i]:ends[i + 1], m] @ kt / math.sqrt(d), -math.inf)
                out[ends[i]:ends[i + 1], m] = torch.softmax(score, -1) @ v
    return out


def _exact_sample(s):
    rows = []
    for r in range(s.case["rows"]):
        x, t = s.logits[r].double(), float(s.temperature[r])
        k, p, m, u = int(s.top_k[r]), float(s.top_p[r]), float(s.min_p[r]), float(s.u[r])
        if t <= 0:
            rows.append(torch.ones((), dtype=torch.float64, device="cuda"))
            continue
        w = torch.exp((x - x.max()) / t)
        ordered, order = torch.sort(w, descending=True, stable=True)
        n = min(k, w.numel()) if k > 0 else w.numel()
        if p < 1:
            sums = torch.cumsum(ordered[:n], 0)
            n = max(1, int((sums - ordered[:n] < p * sums[-1]).sum()))
        kept = torch.zeros_like(w)
        kept[order[:n]] = ordered[:n]
        kept = torch.where(w >= m, kept, 0.0)
        sums = torch.cumsum(kept, 0)
        at = int((sums <= u * sums[-1]).sum())
        rows.append(kept[min(at, w.numel() - 1)] / sums[-1])
    return {"id": None, "prob": torch.stack(rows)}


# ---- what a pass cannot do without

def work(case):
    c = case
    if c["kind"] == "sample":
        n = c["rows"] * c["vocab"]
        return {"bytes": 4 * n + 28 * c["rows"], "flops": 4 * n}
    size = 4 if c["type"] == "f32" else 2
    h, kv, d = c["heads"], c["kv"], c["dim"]
    old, new = _shape(c)
    rows = sum(new)
    if c["kind"] == "append":
        back = sum(n + o % BLOCK for o, n in zip(old, new))
        moved = rows * (2 * h + 2 * kv) * d * size + 2 * rows * kv * d + 2 * back * kv * d * (1 + 4) + rows * c["rot"] * 4
        return {"bytes": moved, "flops": rows * (3 * (h + kv) * c["rot"] + 4 * kv * d)}
    seen = pairs = 0
    for o, n in zip(old, new):
        for_row = [min(o + i + 1, c["window"] or o + i + 1) for i in (0, n - 1)]
        seen += min(o + n, (c["window"] or o + n) + n - 1)
        pairs += n * (for_row[0] + for_row[1]) // 2
    return {"bytes": seen * kv * d * 2 + seen * kv * 8 // BLOCK + 2 * rows * h * d * size, "flops": 4 * pairs * h * d}
