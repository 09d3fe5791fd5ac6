"""The mapping of a ragged batch's query rows to tiles (plain C++), against a
loop: every row of every sequence and kv head lies in one slot's tile."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SHIM = r"""
#include "cache_layout.hpp"
using namespace manta;
extern "C" {
long long slots(long long t, long long n, long long group, int rows) { return tile_slots(t, n, group, rows); }
long long base(int off, long long i, long long group, int rows) { return tile_base(off, i, group, rows); }
const char* batch(long long n, long long t, long long s) { return check_batch(n, t, s, 1); }
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("cache_tiles")
    src, so = d / "shim.cpp", d / "libshim.so"
    src.write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I" + os.path.join(ROOT, "include"),
                    "-I" + os.path.join(ROOT, "manta_amd", "csrc"), str(src), "-o", str(so)], check=True)
    L = C.CDLL(str(so))
    L.slots.restype = L.base.restype = C.c_longlong
    L.slots.argtypes = [C.c_longlong, C.c_longlong, C.c_longlong, C.c_int]
    L.base.argtypes = [C.c_int, C.c_longlong, C.c_longlong, C.c_int]
    L.batch.restype = C.c_char_p
    L.batch.argtypes = [C.c_longlong] * 3
    return L


@pytest.mark.parametrize("rows", [16, 32, 128, 256])
@pytest.mark.parametrize("group", [1, 3, 4, 17, 40, 300])
def test_every_row_lies_in_one_tile(lib, rows, group):
    rng = np.random.default_rng(rows + group)
    for _ in range(50):
        n = int(rng.integers(1, 7))
        counts = [int(x) for x in rng.choice([0, 1, 2, 15, 16, 17, 33, 100], n)]
        off = np.concatenate([[0], np.cumsum(counts)]).astype(int) + int(rng.integers(0, 3))
        slots = lib.slots(int(off[-1]), n, group, rows)
        seen = set()
        for slot in range(slots):
            # as the kernels find it: the last sequence whose base is at or below the slot
            i = max(j for j in range(n) if j == 0 or lib.base(int(off[j]), j, group, rows) <= slot)
            r0 = (slot - lib.base(int(off[i]), i, group, rows)) * rows
            total = counts[i] * group
            if r0 < 0 or r0 >= total:
                continue
            for r in range(r0, min(r0 + rows, total)):
                assert (i, r) not in seen
                seen.add((i, r))
        assert len(seen) == sum(counts) * group


def test_batches_that_no_launch_holds(lib):
    assert lib.batch(1 << 21, 1 << 25, 1) is None
    assert b"too many" in lib.batch((1 << 21) + 1, 1, 1)
    assert b"too many" in lib.batch(1, (1 << 25) + 1, 1)
