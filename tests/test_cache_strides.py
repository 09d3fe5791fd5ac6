"""Strides of results whose rows would run into each other: the check against
all pairs of rows, and the calls that refuse such results."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from manta_amd import _lib, rocm

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SHIM = r"""
#include "cache_layout.hpp"
using namespace manta;
extern "C" const char* out_strides(long long t, long long h, long long d, long long ts, long long hs) {
    return check_out_strides(t, h, d, ts, hs);
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("cache_strides")
    src, so = d / "shim.cpp", d / "libshim.so"
    src.write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I" + os.path.join(ROOT, "include"),
                    "-I" + os.path.join(ROOT, "manta_amd", "csrc"), str(src), "-o", str(so)], check=True)
    L = C.CDLL(str(so))
    L.out_strides.restype = C.c_char_p
    L.out_strides.argtypes = [C.c_longlong] * 5
    return L


def test_against_all_pairs_of_rows(lib):
    rng = np.random.default_rng(1)
    seen = [0, 0]
    for _ in range(3000):
        t, h, d = (int(x) for x in rng.integers(1, 9, 3))
        ts, hs = (int(x) for x in d + rng.integers(0, 10 * d, 2))
        starts = np.sort((np.arange(t)[:, None] * ts + np.arange(h)[None] * hs).ravel())
        overlap = bool((np.diff(starts) < d).any())
        got = lib.out_strides(t, h, d, ts, hs)
        assert (got is not None) == overlap, (t, h, d, ts, hs)
        seen[overlap] += 1
    assert min(seen) > 300


@pytest.mark.parametrize("args,text", [
    ((5, 4, 64, 64, 64), "run into"), ((5, 4, 64, 256, 64), None), ((5, 4, 64, 64, 320), None),
    ((5, 4, 64, 255, 64), "run into"), ((1, 4, 64, 0, 64), None), ((5, 1, 64, 64, 0), None),
    ((5, 4, 64, -64, 64), "negative"), ((5, 4, 64, 256, 32), "head stride"), ((5, 4, 64, 32, 256), "token stride"),
    ((1 << 25, 65535, 256, 1 << 40, 1 << 40), "run into"), ((1 << 25, 65535, 256, 1 << 62, 256), None),
    ((3, 2, 64, 128, 192), None), ((4, 2, 64, 128, 192), None), ((4, 3, 64, 128, 192), "run into"),
])
def test_cases(lib, args, text):
    got = lib.out_strides(*args)
    assert (got is None) if text is None else (got is not None and text in got.decode())


def test_rotary_refuses_before_it_needs_a_device():
    h = _lib.Heads(4096, 8192, 4, 256, 64, 64, 64)
    with pytest.raises(_lib.MantaRocmError, match="tensor 0: rows of the result run into each other"):
        _lib.call("manta_rocm_rotary", None, None, _lib.F16, 4096, 3, 64, C.byref(h), 1, 0)


@pytest.mark.gpu
def test_read_and_attention_refuse(rt):
    print("result strides", flush=True)
    c = rt.cache(pages=4, kv_heads=2, head_dim=32, seqs=2, table_pages=2, page_tokens=16)
    off = rt.to_device(np.array([0, 3], np.int32))
    x = rt.to_device(np.zeros((3, 2, 32), np.float32))
    buf = rt.to_device(np.zeros(512, np.float32))
    bad = rocm.View(buf, (3, 2, 32), (32, 32, 1))
    for k, v in ((bad, x), (x, bad)):
        with pytest.raises(_lib.MantaRocmError, match="cache_read: rows of the result run into each other"):
            c.read(0, off, k, v)
    c.append(0, bad, bad, off)  # (what is only read may)
    q = rt.to_device(np.zeros((3, 2, 32), np.uint16))
    out = rocm.View(rt.to_device(np.zeros(512, np.uint16)), (3, 2, 32), (48, 32, 1))
    with pytest.raises(_lib.MantaRocmError, match="cache_attention: rows of the result run into each other"):
        c.attention(0, q, off, out=out)
    rt.synchronize()
    c.close()
