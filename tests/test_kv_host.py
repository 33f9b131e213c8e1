"""The host side of the cache and attention calls on the test double of the HIP runtime: what they refuse, and the memory they ask for."""
import pytest

from test_host_runtime import fake, run  # noqa: F401 (fixtures)

SETUP = """
a = pkg.Mi355WeightAccel(0)
room = a.dev_alloc(1 << 20)
KV, HEADS, DIM = 2, 8, 64
cache = pkg.KvCache(64, 64, KV, DIM, room, room, room, room)
def batch(nseq, rows, max_rows, max_len=4000):
    return pkg.KvBatch(nseq, room, room, 64, max_len, row0=room, rows=rows, max_rows=max_rows)
def refused(f, code=-1):
    try:
        f()
    except pkg.SmxError as e:
        assert e.code == code, e
    else:
        raise AssertionError("not refused")
"""


def test_no_rows_to_a_sequence(run):   # noqa: F811
    """Rows of which no sequence may have one."""
    run(SETUP + """
for rows in (1, 3, 500):
    b = batch(3, rows, 0)
    refused(lambda: a.attn_dev(cache, b, room, HEADS, 1.0, room))
    refused(lambda: a.kv_append_dev(cache, b, room, room))
    refused(lambda: a.kv_read_dev(cache, b, room, room))
b = batch(3, 0, 0)                                   # a step without a row is a step
a.attn_dev(cache, b, room, HEADS, 1.0, room)
a.kv_append_dev(cache, b, room, room)
a.kv_read_dev(cache, b, room, room)
""")


def test_more_rows_than_are_counted(run):   # noqa: F811
    """Rows times heads of 2^31 and more: refused by the attention as by the append."""
    run(SETUP + """
one = pkg.KvCache(64, 64, 1, 2, room, room, room, room)
for rows, heads in ((1 << 24, 128), (1 << 23, 256), (1 << 20, 2048), (1 << 24, 65535)):
    b = batch(1, rows, rows)
    refused(lambda: a.attn_dev(one, b, room, heads, 1.0, room), -3)
    refused(lambda: a.kv_append_dev(one, b, room, room, q=room, q_heads=heads, q_out=room), -3)
launches = F.fake_launches()
a.attn_dev(one, batch(1, 1 << 16, 1 << 16, 64), room, 1, 1.0, room)
assert F.fake_launches() > launches
""")


@pytest.mark.parametrize("nseq,rows,max_rows,max_len", [
    (2, 8193, 8192, 100000),      # a prompt chunk beside one decode step
    (9, 8200, 8192, 131072), (65, 8256, 8192, 16384),
    (4097, 4129, 33, 16384),      # one short chunk beside thousands of decode steps
    (1000, 1063, 64, 131072), (65, 65, 1, 131072), (1, 2048, 2048, 8192)])
def test_scratch_of_calls_whose_rows_differ(run, nseq, rows, max_rows, max_len):   # noqa: F811
    """The attention's scratch goes by the rows whose context is split, not by those beside them."""
    run(SETUP + """
F.fake_device_live.restype = C.c_size_t
wide = pkg.KvCache(1 << 20, 64, 8, 128, room, room, room, room)
before = F.fake_device_live()
a.attn_dev(wide, pkg.KvBatch(nseq, room, room, 1 << 12, max_len, row0=room, rows=rows, max_rows=max_rows), room, 32, 0.1, room)
assert F.fake_device_live() - before <= 257 << 20, (F.fake_device_live() - before) >> 20
""", nseq=nseq, rows=rows, max_rows=max_rows, max_len=max_len)


def test_cache_whose_bytes_pass_64_bits(pkg):
    """Sizes that have wrapped would be those of a far smaller cache than the kernels index."""
    for bad in ((1 << 31, 1 << 20, 65535, 256), (1 << 31, 1 << 20, 8, 128), (1 << 30, 1 << 20, 32, 2)):
        with pytest.raises(ValueError):
            pkg.kv_sizes(*bad)
    assert pkg.kv_sizes(1 << 20, 1 << 15, 8, 256) == (1 << 46, 1 << 33)
