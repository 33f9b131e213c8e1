"""AttentionChain without a GPU: what it refuses before anything is enqueued, and what its calls are given."""
import importlib.util
import os
import types

import pytest

from conftest import PKG_DIR


class Calls:
    """An accelerator that counts the calls made of it."""

    def __init__(self):
        self.made, self.args = [], []

    def __getattr__(self, name):
        def call(*a, **k):
            self.made.append(name)
            self.args.append(a)
            return 0x1000 * len(self.made)
        return call


@pytest.fixture
def make(pkg):
    spec = importlib.util.spec_from_file_location("strix_rs_amd_chain_host", os.path.join(PKG_DIR, "chain.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    fake = types.SimpleNamespace(kv_sizes=lambda *a: (64, 64), KvCache=lambda *a: None, Rope=lambda *a: None, ACT_RMSNORM=pkg.ACT_RMSNORM)
    return lambda layers=1, norm=0x2000: mod.AttentionChain(fake, Calls(), layers, 64, 2, 1, 32, lambda l: tuple(f"{t}{l}" for t in "qkvo"), "head", 100,
                                                            norm, 3, 1, 32, 32)


def test_more_rows_than_the_buffers_hold(make):
    """Rows beyond the chain's would be written behind its buffers: the step's as well as the sampled end's."""
    chain = make()
    chain.acc.made.clear()
    with pytest.raises(ValueError, match="4 rows"):
        chain.enqueue(0x1000, types.SimpleNamespace(rows=4))
    with pytest.raises(ValueError, match="4 rows"):
        chain.layer(0, 0x1000, types.SimpleNamespace(rows=4))
    with pytest.raises(ValueError, match="4 rows"):
        chain.sample(0x1000, 4, 0x1000, 0x1000)
    assert not chain.acc.made
    chain.sample(0x1000, 3, 0x1000, 0x1000)
    assert chain.acc.made == ["gemm_fused_dev", "sample_dev"]


def test_a_layer_at_a_time(make):
    """Layers called one by one, each with its own rmsnorm weight, are what enqueue() calls."""
    batch = types.SimpleNamespace(rows=3)
    with pytest.raises(ValueError, match="2 rmsnorm weights"):
        make(2, [1, 2])
    whole, apart = make(2, [11, 12, 13]), make(2, [11, 12, 13])
    for c in (whole, apart):
        c.acc.made.clear(), c.acc.args.clear()
    out = whole.enqueue(0x77, batch)
    y = apart.layer(0, 0x77, batch)
    assert apart.layer(1, y, batch) == out
    assert whole.acc.made == apart.acc.made == 2 * (["gemm_fused_dev"] * 3 + ["kv_append_dev", "attn_dev", "gemv_dev"])
    normed = [a for n, a in zip(apart.acc.made, apart.acc.args) if n == "gemm_fused_dev"]
    assert [a[0] for a in normed] == ["q0", "k0", "v0", "q1", "k1", "v1"] and [a[3] for a in normed] == [11] * 3 + [12] * 3
    assert [a[2] for a in normed] == [0x77] * 3 + [y] * 3
    apart.acc.made.clear(), apart.acc.args.clear()
    apart.sample(y, 2, 0x1000, 0x1000)
    assert apart.acc.args[0][3] == 13
