"""The sampler's kernels on the CPU (host_waves.h), their waves in orders that a GPU run shows only by chance: the picks are those of the
definition whichever wave runs ahead between two barriers."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from conftest import ROOT
from test_gpu_sample import _check

INTERNAL = r"""
#pragma once
#include "host_waves.h"
#include "strix_mi355.h"
#include <algorithm>
#include <cstdarg>
typedef int hipError_t;
namespace smx { struct DevBuf { char* p = nullptr; size_t cap = 0; }; }
struct smx_ctx { smx::DevBuf work; int stream = 0; };
namespace smx {
inline int fail(smx_ctx*, int code, const char*, ...) { return code; }
inline int ensure(smx_ctx*, DevBuf& b, size_t n) {
    if (n > b.cap) { std::free(b.p); b.p = (char*)std::malloc(n); b.cap = n; }
    std::memset(b.p, 0xaa, b.cap);   // whatever an earlier call has left there
    return SMX_OK;
}
template <class K> int set_dyn_lds(smx_ctx*, K, size_t) { return SMX_OK; }
struct ProfScope { ProfScope(smx_ctx*, const char*) {} ~ProfScope() {} };
}
#define SMX_HIP(c, call) do { } while (0)
"""
BEHIND = r"""
namespace smx { namespace { alignas(16) unsigned long long room[1 << 15]; } }
extern "C" smx_ctx* waves_context(int order) { static smx_ctx c; waves::order = order; return &c; }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("waves")
    text = open(os.path.join(ROOT, "strix.rs_amd", "csrc", "sample.hip")).read()
    for a, b in (("extern __shared__", "extern"), ('asm volatile("s_waitcnt vmcnt(0)" ::: "memory");', "")):   # (workgroups run one after the other)
        assert a in text
        text = text.replace(a, b)
    (d / "sample.cpp").write_text(text + BEHIND)
    (d / "smx_internal.h").write_text(INTERNAL)
    out = str(d / "libsample.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-w", "-ffp-contract=off", "-shared", "-fPIC", "-I", str(d), "-I", os.path.join(ROOT, "tests"),
                    "-I", os.path.join(ROOT, "include"), str(d / "sample.cpp"), "-o", out], check=True)
    L = C.CDLL(out)
    L.waves_context.restype = C.c_void_p
    return L


def _run(L, pkg, order, x, u, T=None, k=None, p=None, m=None):
    rows, v = x.shape
    keep = [np.ascontiguousarray(x, np.float32), np.ascontiguousarray(u, np.float32)]
    at = lambda a, t: None if a is None else keep.append(np.ascontiguousarray(a, t)) or keep[-1].ctypes.data
    ids, prob = np.full(rows, -1, np.int32), np.full(rows, -1, np.float32)
    params = pkg._SampleParams(at(T, np.float32), at(k, np.int32), at(p, np.float32), at(m, np.float32))
    ptr = lambda a: C.c_void_p(a.ctypes.data)
    rc = L.smx_sample_dev(C.c_void_p(L.waves_context(order)), ptr(keep[0]), C.c_size_t(rows), C.c_size_t(v), C.c_size_t(v), C.byref(params), ptr(keep[1]),
                          ptr(ids), ptr(prob))
    assert rc == 1
    return ids, prob


@pytest.mark.parametrize("order", [0, 1, 2, 3])
def test_two_cuts_behind_an_overflowing_list(lib, pkg, order):
    """top_k of thousands and top_p behind it: the second cut begins where the first one's last token has just been found."""
    rng = np.random.default_rng(5)
    rows, v = 3, 9000
    x = (rng.standard_normal((rows, v)) * 1.5).astype(np.float32)
    x[1, ::3] = x[1, 0]                                     # the first cut among equal logits, the last token by its index
    x[2] = np.round(x[2])
    k, p = np.array([5000, 6500, 7000], np.int32), np.array([0.9, 0.97, 0.999], np.float32)
    T, u = np.array([1.0, 2.0, 3.0], np.float32), np.array([0.3, 0.97, 0.999], np.float32)
    ids, prob = _run(lib, pkg, order, x, u, T, k, p)
    _check(x, ids, prob, u, T, k, p, None)


@pytest.mark.parametrize("order", [0, 1, 2])
@pytest.mark.parametrize("what", ["free", "top_k", "top_p", "both", "levels", "all"])
def test_picks_in_every_order(lib, pkg, order, what):
    """The other ways to a pick: short lists, long ones in steps of keys, cuts among equal logits, no cut at all."""
    rng = np.random.default_rng(len(what))
    rows, v = 4, 5003
    x = (rng.standard_normal((rows, v)) * 2).astype(np.float32)
    if what == "levels":
        x = rng.integers(0, 3, (rows, v)).astype(np.float32)
    x[1, 17] = np.nan
    x[2, 5:90] = -np.inf
    u = np.array([0.0, 0.4, 0.8, 0.99], np.float32)
    T = np.array([0.7, 1.0, 1.5, 0.0 if what == "all" else 0.9], np.float32)
    k = np.array([40, 300, 4096, 1000], np.int32) if what in ("top_k", "both", "levels", "all") else None
    p = np.array([0.3, 0.9, 0.95, 0.99], np.float32) if what in ("top_p", "both", "levels", "all") else None
    m = np.array([0.0, 0.05, 0.001, 0.0], np.float32) if what == "all" else None
    ids, prob = _run(lib, pkg, order, x, u, T, k, p, m)
    _check(x, ids, prob, u, T, k, p, m)
    again = _run(lib, pkg, 7, x, u, T, k, p, m)
    assert np.array_equal(ids, again[0]) and np.array_equal(prob, again[1])
