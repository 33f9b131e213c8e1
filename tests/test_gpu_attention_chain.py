"""The attention half of a decode step as a user runs it (strix.rs_amd/chain.py: AttentionChain): a prompt chunk of ragged sequences, then
decode steps, eager and as a replayed graph, every operator against plain numpy on the device's own input to it."""
import importlib.util
import os
import sys

import numpy as np
import pytest

import kv_ref as R
from test_gpu_sample import _check

pytestmark = pytest.mark.gpu
PKG_DIR = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "strix.rs_amd")
LAYERS, HIDDEN, HEADS, KV, DIM, VOCAB, PAGE, N = 2, 256, 8, 2, 64, 1500, 32, 3
PROMPT = [70, 1, 33]


@pytest.fixture(scope="module")
def chain_mod():
    name = "strix_rs_amd_chain"
    if name not in sys.modules:
        spec = importlib.util.spec_from_file_location(name, os.path.join(PKG_DIR, "chain.py"))
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name]


@pytest.fixture
def weights(accel, synth):
    """Keys of synthetic weights: q, k, v and o of each layer, and the lm_head."""
    shapes = [(f"t.at.{t}{l}", i, o) for l in range(LAYERS)
              for t, i, o in (("q", HIDDEN, HEADS * DIM), ("k", HIDDEN, KV * DIM), ("v", HIDDEN, KV * DIM), ("o", HEADS * DIM, HIDDEN))]
    shapes.append(("t.at.head", HIDDEN, VOCAB))
    for n, (key, i, o) in enumerate(shapes):
        assert accel.upload_q8_0(key, synth.make_weight(8, o, i, seed=300 + n), i, o)
    yield
    for key, _, _ in shapes:
        accel.evict(key)


def _chain(chain_mod, pkg, accel, norm, rows, pages, keep):
    return chain_mod.AttentionChain(pkg, accel, LAYERS, HIDDEN, HEADS, KV, DIM, lambda l: tuple(f"t.at.{t}{l}" for t in "qkvo"), "t.at.head", VOCAB,
                                    norm, rows, pages, PAGE, 256, keep_stages=keep)


def test_prompt_then_decode(accel, pkg, synth, chain_mod, weights):
    rng = np.random.default_rng(21)
    steps, rows = 4, sum(PROMPT)
    table = R.tables(rng, 12, PAGE, [n + steps for n in PROMPT])
    rope = R.rope_table(256, DIM)
    with R.Dev(accel) as dev:
        norm = dev.put((rng.standard_normal(HIDDEN) * 0.1 + 1.0).astype(np.float32))
        ch = _chain(chain_mod, pkg, accel, norm, rows, 12, keep=True)
        host = [R.Cache(12, PAGE, KV, DIM, seed=l) for l in range(LAYERS)]
        xd, lens, row0, tab = dev.room(rows * HIDDEN * 4), dev.room(N * 4), dev.put(np.cumsum([0] + PROMPT).astype(np.int32)), dev.put(table)
        temperature, top_k, top_p = np.array([0.8, 0.0, 1.3], np.float32), np.array([40, 0, 0], np.int32), np.array([0.95, 1.0, 0.9], np.float32)
        u, ids, prob = dev.room(N * 4), dev.room(N * 4), dev.room(N * 4)
        knobs = {"temperature": dev.put(temperature), "top_k": dev.put(top_k), "top_p": dev.put(top_p)}
        prompt = pkg.KvBatch(N, lens, tab, table.shape[1], max(PROMPT), row0=row0, rows=rows, max_rows=max(PROMPT))
        decode = pkg.KvBatch(N, lens, tab, table.shape[1], max(PROMPT) + steps)

        def step(batch, length, new, x):
            """One step, and its operators against numpy on what the device gave them."""
            n = int(sum(new))
            accel.h2d(lens, np.asarray(length, np.int32))
            accel.h2d(xd, x)
            y = ch.enqueue(xd, batch)
            accel.sync()
            pos = np.concatenate([np.arange(a - b, a) for a, b in zip(length, new)])
            for l in range(LAYERS):
                b = ch.buffers(l)[0]
                q, k, v, o = (dev.get(b[t], (n, h, DIM)) for t, h in (("q", HEADS), ("k", KV), ("v", KV), ("o", HEADS)))
                # k is what the projection left (the cache holds it rotated), q was rotated in place
                R.append(host[l], table, [a - b for a, b in zip(length, new)], list(new), R.rotate(k, rope, pos, DIM, False), v)
                want = R.attend(host[l], table, list(length), list(new), q, DIM ** -0.5)
                # (the values' size times the error of a probability's two f16 terms and of an fp32 exponential of arguments up to 100)
                assert np.abs(o - want).max() <= 2e-5 * np.abs(v).max() * 5, l
            return y

        x = rng.standard_normal((rows, HIDDEN)).astype(np.float32)
        step(prompt, PROMPT, PROMPT, x)
        length = np.array(PROMPT)
        for i in range(steps):
            length = length + 1
            x = rng.standard_normal((N, HIDDEN)).astype(np.float32)
            y = step(decode, length, [1] * N, x)
            un = rng.random(N, dtype=np.float32)
            accel.h2d(u, un)
            ch.sample(y, N, u, ids, prob=prob, **knobs)
            accel.sync()
            _check(dev.get(ch.logits, (N, VOCAB)), dev.get(ids, N, np.int32), dev.get(prob, N), un, temperature, top_k, top_p, None)
        ch.close()


def test_decode_as_a_graph_equals_eager_steps(accel, pkg, synth, chain_mod, weights):
    """The same tokens through an eager chain and a captured one: every output and pick has the same bits."""
    rng = np.random.default_rng(22)
    steps = 6
    table = R.tables(rng, 6, PAGE, [steps + 31] * N)
    with R.Dev(accel) as dev:
        norm = dev.put(np.ones(HIDDEN, np.float32))
        eager, captured = (_chain(chain_mod, pkg, accel, norm, N, 6, keep=False) for _ in range(2))
        xd, lens, u, ids, tab = dev.room(N * HIDDEN * 4), dev.room(N * 4), dev.room(N * 4), dev.room(N * 4), dev.put(table)
        top_p = dev.put(np.full(N, 0.9, np.float32))
        batch = pkg.KvBatch(N, lens, tab, table.shape[1], steps + 31)

        def step(ch):
            y = ch.enqueue(xd, batch)
            ch.sample(y, N, u, ids, top_p=top_p)
            return y

        # (a first call outside the capture brings the scratch to size; tokens of a first step start their blocks again)
        accel.h2d(lens, np.ones(N, np.int32))
        accel.h2d(xd, np.zeros((N, HIDDEN), np.float32))
        accel.h2d(u, np.zeros(N, np.float32))
        step(captured)
        accel.sync()
        accel.graph_begin()
        out = step(captured)
        g = accel.graph_end()
        seen = set()
        for i in range(steps):
            accel.h2d(lens, np.full(N, i + 1, np.int32))
            accel.h2d(xd, rng.standard_normal((N, HIDDEN)).astype(np.float32))
            accel.h2d(u, rng.random(N, dtype=np.float32))
            want_y = dev.get(step(eager), (N, HIDDEN))
            want = dev.get(ids, N, np.int32)
            accel.h2d(ids, np.full(N, -1, np.int32))
            accel.sync()
            accel.graph_launch(g)
            accel.sync()
            assert np.array_equal(dev.get(out, (N, HIDDEN)), want_y), i
            assert np.array_equal(dev.get(ids, N, np.int32), want), i
            seen.add(tuple(want))
        assert len(seen) > 1
        accel.graph_destroy(g)
        eager.close()
        captured.close()


def test_refusals(accel, pkg, chain_mod, weights):
    with R.Dev(accel) as dev:
        norm, x, lens, tab = dev.put(np.ones(HIDDEN, np.float32)), dev.put(np.zeros((4, HIDDEN), np.float32)), dev.put(np.ones(4, np.int32)), dev.put(np.zeros((4, 1), np.int32))
        ch = _chain(chain_mod, pkg, accel, norm, 2, 4, keep=False)
        with pytest.raises(ValueError, match="4 rows"):
            ch.enqueue(x, pkg.KvBatch(4, lens, tab, 1, 1))
        ch.keys = lambda l: ("t.at.q0", "t.at.absent", "t.at.v0", "t.at.o0")
        with pytest.raises(RuntimeError, match="layer 0"):
            ch.enqueue(x, pkg.KvBatch(1, lens, tab, 1, 1))
        ch.close()
