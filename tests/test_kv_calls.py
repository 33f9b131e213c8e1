"""The cache, attention and sampling calls without a GPU: what the Python methods hand to the library through either binding, the C
structures' layout, and the sizes of a cache."""
import ctypes as C
import importlib.util
import os
import subprocess

import pytest

from conftest import PKG_DIR, ROOT, _load_by_path
from test_native_binding import _recorder


@pytest.fixture(scope="module")
def rec(tmp_path_factory):
    """(extension module linked to a recording library, that library); its name is its own, since a process loads a name once"""
    d = str(tmp_path_factory.mktemp("kv_binding"))
    with open(os.path.join(d, "rec.c"), "w") as f:
        f.write(_recorder())
    lib = os.path.join(d, "libsmx_kv_recorder.so")
    subprocess.run(["gcc", "-shared", "-fPIC", "-w", "-I" + os.path.join(ROOT, "include"), os.path.join(d, "rec.c"), "-o", lib], check=True)
    path = _load_by_path("strix_rs_amd_build", os.path.join(PKG_DIR, "build.py")).build_pybind(d, "smx_kv_recorder")
    spec = importlib.util.spec_from_file_location("_smx_native", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    L = C.CDLL(lib)
    L.rec_text.restype = C.c_char_p
    return mod, L


def _accel(pkg, calls):
    a = pkg.Mi355WeightAccel.__new__(pkg.Mi355WeightAccel)
    a._n, a._a, a._h, a._L = calls, 16, C.c_void_p(16), None
    a.close = lambda: None
    return a


@pytest.mark.parametrize("binding", ["native", "ctypes"])
def test_arguments_arrive_in_order(pkg, rec, binding):
    mod, L = rec
    if binding == "ctypes":
        table = pkg.load_library()
        for name in ("smx_kv_append_dev", "smx_kv_read_dev", "smx_attn_dev"):   # the product library's argument types for the recorder
            getattr(L, name).argtypes = getattr(table, name).argtypes
        a = _accel(pkg, pkg.CtypesCalls(L))
        a._a = a._h
    else:
        a = _accel(pkg, mod)
    cache = pkg.KvCache(3, 64, 2, 80, 0x1000, 0x2000, 0x3000, 0x4000)
    batch = pkg.KvBatch(5, 0x5000, 0x6000, 7, 400, row0=0x7000, rows=9, max_rows=4)
    rope = pkg.Rope(0x8000, 512, 64, interleaved=True)
    said = lambda: L.rec_text().decode().split()
    at = lambda s: hex(s.addr)
    a.kv_append_dev(cache, batch, 0x9000, 0xa000, rope=rope, q=0xb000, q_heads=6, q_out=0xc000, dtype=pkg.DTYPE_BF16, ldv=200)
    assert said() == ["smx_kv_append_dev", "0x10", at(cache), at(batch), "30", "0x9000", "160", "0xa000", "200", at(rope), "0xb000", "480", "6", "0xc000", "480"]
    a.kv_append_dev(cache, batch, 0x9000, 0xa000)
    assert said() == ["smx_kv_append_dev", "0x10", at(cache), at(batch), "0", "0x9000", "160", "0xa000", "160", "(nil)", "(nil)", "0", "0", "(nil)", "0"]
    a.kv_read_dev(cache, batch, None, 0xd000)
    assert said() == ["smx_kv_read_dev", "0x10", at(cache), at(batch), "(nil)", "0xd000"]
    a.attn_dev(cache, batch, 0xb000, 6, 0.125, 0xe000, window=33, ldo=500)
    assert said() == ["smx_attn_dev", "0x10", at(cache), at(batch), "0", "0xb000", "480", "6", "0.125", "33", "0xe000", "500"]


def test_sampling_arguments(pkg, rec):
    mod, L = rec
    a = _accel(pkg, mod)
    a.sample_dev(0x1000, 3, 1000, 0x2000, 0x3000, temperature=0x4000, top_p=0x5000, prob=0x6000, ld=1024)
    got = L.rec_text().decode().split()
    assert got[:5] == ["smx_sample_dev", "0x10", "0x1000", "3", "1000"] and got[5] == "1024" and got[7:] == ["0x2000", "0x3000", "0x6000"]


def test_wrong_arguments_are_refused_by_the_binding(rec):
    mod, _ = rec
    for name, count in (("kv_append_dev", 14), ("kv_read_dev", 5), ("attn_dev", 11), ("sample_dev", 12)):
        with pytest.raises(TypeError):
            getattr(mod, name)(*[1] * (count - 1))
        with pytest.raises((TypeError, AttributeError)):
            getattr(mod, name)(*["no address"] * count)


def test_structures_have_the_headers_layout(pkg, tmp_path):
    src = tmp_path / "layout.c"
    names = {"smx_kv_cache": pkg.KvCache, "smx_kv_batch": pkg.KvBatch, "smx_rope": pkg.Rope, "smx_sample_params": pkg._SampleParams}
    lines = [f'printf("{n} %zu", sizeof({n}));' + "".join(f'printf(" %zu", offsetof({n}, {f}));' for f, _ in t._fields_) + 'printf("\\n");' for n, t in names.items()]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "strix_mi355.h"\nint main(void) {' + "".join(lines) + "}\n")
    subprocess.run(["gcc", "-I" + os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.splitlines()
    for line in out:
        name, *numbers = line.split()
        t = names[name]
        assert [int(n) for n in numbers] == [C.sizeof(t)] + [getattr(t, f).offset for f, _ in t._fields_], name


@pytest.mark.parametrize("pages,page,heads,dim", [(1, 32, 1, 2), (7, 96, 3, 80), (4, 256, 8, 128), (100000, 1024, 8, 256)])
def test_cache_sizes(pkg, pages, page, heads, dim):
    nb, ns = pkg.kv_sizes(pages, page, heads, dim)
    assert nb == pages * page * heads * ((dim + 63) // 64 * 64) and ns == pages * heads * page // pkg.KV_BLOCK


@pytest.mark.parametrize("pages,page,heads,dim", [(1, 33, 1, 64), (1, 0, 1, 64), (1, 32, 0, 64), (1, 32, 1, 0), (1, 32, 1, 63), (1, 32, 1, 258)])
def test_no_such_cache(pkg, pages, page, heads, dim):
    with pytest.raises(ValueError):
        pkg.kv_sizes(pages, page, heads, dim)
