"""Batches whose offsets descend: how many tiles the evenly cut attention would
lay out for them (plain C++), and that the kernel refuses them."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TICKETS = 65536  # cache.cpp's

SHIM = r"""
#include "cache_layout.hpp"
using namespace manta;
extern "C" {
long long slots(long long t, long long n, long long group, int rows) { return tile_slots(t, n, group, rows); }
int count(int from, int to, long long group, int rows) { return tile_count(from, to, group, rows); }
int fit(long long tiles, long long kv, long long tickets) { return tiles_fit(tiles, kv, tickets); }
void describe(int kind, long long a, long long b, char* out) { describe_cache_error(cache_error(kind, a, b), out, 160); }
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("cache_offsets")
    src, so = d / "shim.cpp", d / "libshim.so"
    src.write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I" + os.path.join(ROOT, "include"),
                    "-I" + os.path.join(ROOT, "manta_amd", "csrc"), str(src), "-o", str(so)], check=True)
    L = C.CDLL(str(so))
    L.slots.restype = C.c_longlong
    L.slots.argtypes = [C.c_longlong, C.c_longlong, C.c_longlong, C.c_int]
    L.count.argtypes = [C.c_int, C.c_int, C.c_longlong, C.c_int]
    L.fit.argtypes = [C.c_longlong] * 3
    L.describe.argtypes = [C.c_int, C.c_longlong, C.c_longlong, C.c_char_p]
    return L


@pytest.mark.parametrize("rows", [16, 32])
def test_tiles_of_ascending_offsets_have_their_tickets(lib, rows):
    """What the host checks (the batch's slots) bounds what the device counts."""
    rng = np.random.default_rng(rows)
    for _ in range(300):
        n, group = int(rng.integers(1, 65)), int(rng.choice([1, 2, 3, 7, 16, 31, 40]))
        off = np.sort(rng.integers(0, int(rng.choice([2, 40, 3000])), n + 1))
        tiles = sum(lib.count(int(a), int(b), group, rows) for a, b in zip(off, off[1:]))
        slots = lib.slots(int(off[-1]), n, group, rows)
        assert tiles <= slots
        kv = max(1, TICKETS // slots)
        assert not lib.fit(slots, kv, TICKETS) or lib.fit(tiles, kv, TICKETS)


def test_tiles_of_descending_offsets_do_not(lib):
    """64 entries of 0, 1024, 0, 1024, ... and 64 kv heads: 1024 rows in all,
    which the host finds to fit, and twice as many tiles as tickets."""
    off = [0 if i % 2 == 0 else 1024 for i in range(65)]
    tiles = sum(lib.count(a, b, 1, 16) for a, b in zip(off, off[1:]))
    assert lib.fit(lib.slots(1024, 64, 1, 16), 64, TICKETS)
    assert tiles * 64 == 2 * TICKETS and not lib.fit(tiles, 64, TICKETS)
    assert lib.count(1024, 0, 1, 16) == 0 and lib.count(5, 5, 1, 16) == 0


def test_error_words(lib):
    buf = C.create_string_buffer(160)
    lib.describe(6, 17, 0, buf)
    assert buf.value.decode() == "cache offsets descend at entry 17 of the batch"
    lib.describe(7, 40000, 0, buf)
    assert buf.value.decode() == "cache page 40000 is shared: extend copies it before an append"


@pytest.mark.gpu
def test_attention_refuses_descending_offsets(rt):
    """Reported, no row written, and the calls after it as ever (the tickets
    are zero)."""
    from cache_oracle import filled, to_bits
    from manta_amd import _lib

    print("descending offsets", flush=True)
    rng = np.random.default_rng(41)
    n, kv, d, many = 64, 2, 64, 1 << 22
    m = filled(rng, [40] * n, 16, kv, d)
    c = m.upload(rt)
    t = 64
    q = rt.to_device(to_bits(rng.standard_normal((t, kv, d)), "f16"))
    ascending = rt.to_device(np.arange(n + 1, dtype=np.int32))
    want = c.attention(0, q, ascending, longest=many).download()
    for bad in ([0 if i % 2 == 0 else t for i in range(n + 1)], list(range(n, -1, -1)),
                [0, 9, 8] + [64] * (n - 2)):
        out = rt.to_device(np.full((t, kv, d), 0x5555, np.uint16))
        c.attention(0, q, rt.to_device(np.asarray(bad, np.int32)), out=out, longest=many)
        with pytest.raises(_lib.MantaRocmError, match="offsets descend at entry"):
            rt.synchronize()
        np.testing.assert_array_equal(out.download(), 0x5555)
    np.testing.assert_array_equal(c.attention(0, q, ascending, longest=many).download(), want)
    c.close()
