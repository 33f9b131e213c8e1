"""AttentionChain without a GPU: what it refuses before anything is enqueued."""
import importlib.util
import os
import types

import pytest

from conftest import PKG_DIR


class Calls:
    """An accelerator that counts the calls made of it."""

    def __init__(self):
        self.made = []

    def __getattr__(self, name):
        def call(*a, **k):
            self.made.append(name)
            return 0x1000
        return call


@pytest.fixture
def chain(pkg):
    spec = importlib.util.spec_from_file_location("strix_rs_amd_chain_host", os.path.join(PKG_DIR, "chain.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    fake = types.SimpleNamespace(kv_sizes=lambda *a: (64, 64), KvCache=lambda *a: None, Rope=lambda *a: None, ACT_RMSNORM=pkg.ACT_RMSNORM)
    return mod.AttentionChain(fake, Calls(), 1, 64, 2, 1, 32, lambda l: ("q", "k", "v", "o"), "head", 100, 0x2000, 3, 1, 32, 32)


def test_more_rows_than_the_buffers_hold(chain):
    """Rows beyond the chain's would be written behind its buffers: the step's as well as the sampled end's."""
    chain.acc.made.clear()
    with pytest.raises(ValueError, match="4 rows"):
        chain.enqueue(0x1000, types.SimpleNamespace(rows=4))
    with pytest.raises(ValueError, match="4 rows"):
        chain.sample(0x1000, 4, 0x1000, 0x1000)
    assert not chain.acc.made
    chain.sample(0x1000, 3, 0x1000, 0x1000)
    assert chain.acc.made == ["gemm_fused_dev", "sample_dev"]
