"""The decoding calls' layout header (plain C++): where codes lie, how rows of
logits and tables are cut, against what the kernels take for granted."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from manta_amd import decode

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SHIM = r"""
#include "decode_layout.hpp"
using namespace manta;
extern "C" {
long long pitch(long long w) { return product_pitch(w); }
long long at(long long p, long long r, long long c) { return product_at(p, r, c); }
long long rows(long long n, int gated) { return weight_rows(n, gated); }
int parts(long long rows, long long vocab) { return beam_parts(rows, vocab); }
long long all_parts(long long rows) { return beam_parts_in_all(rows); }
int columns(long long group) { return reorder_columns(group); }
int ints() { return kReorderInts; }
int piece() { return kBeamPiece; }
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("decode_layout")
    src, so = d / "shim.cpp", d / "libshim.so"
    src.write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I" + os.path.join(ROOT, "include"),
                    "-I" + os.path.join(ROOT, "manta_amd", "csrc"), str(src), "-o", str(so)], check=True)
    L = C.CDLL(str(so))
    for f in ("pitch", "at", "rows"):
        getattr(L, f).restype = C.c_longlong
    L.pitch.argtypes = [C.c_longlong]
    L.at.argtypes = [C.c_longlong] * 3
    L.rows.argtypes = [C.c_longlong, C.c_int]
    L.parts.argtypes = [C.c_longlong] * 2
    L.all_parts.argtypes, L.all_parts.restype = [C.c_longlong], C.c_longlong
    L.columns.argtypes = [C.c_longlong]
    return L


@pytest.mark.parametrize("rows,width", [(1, 1), (16, 64), (17, 65), (33, 130), (5, 300)])
def test_codes_lie_apart_and_come_back(lib, rows, width):
    p = lib.pitch(width)
    full = (rows + 15) // 16 * 16
    at = np.array([[lib.at(p, r, c) for c in range(p)] for r in range(full)])
    assert p % 128 == 0 and p - width < 128
    np.testing.assert_array_equal(np.sort(at.ravel()), np.arange(full * p))
    # 16 columns of a row are 16 bytes in a row, and a wave's 64 runs a KB in order
    assert (at[:, 1::16] - at[:, ::16] == 1).all()
    for lane in range(64):
        assert at[lane % 16, 16 * (lane // 16)] == 16 * lane
    # Quantized.values finds them
    values = np.arange(full * p, dtype=np.int64) % 251 - 125
    buf = np.zeros(full * p, np.int8)
    buf[at.ravel()] = values
    q = decode.Quantized.__new__(decode.Quantized)
    q.rows, q.width = rows, width
    q.codes = type("A", (), {"download": lambda self: buf})()
    q.scales = type("A", (), {"download": lambda self: None})()
    np.testing.assert_array_equal(q.values()[0], values.reshape(full, p)[:rows, :width])


def test_gated_weights_have_both_halves_in_whole_blocks(lib):
    for n in (1, 15, 16, 17, 1000):
        assert lib.rows(n, 0) == (n + 15) // 16 * 16 and lib.rows(n, 1) == 2 * lib.rows(n, 0)


def test_parts_of_rows(lib):
    piece = lib.piece()
    for rows in (1, 2, 7, 64, 512, 1024, 100000):
        for vocab in (1, 17, piece - 1, piece, piece + 1, 32000, 130001, 10 ** 6, 2 ** 31 - 17):
            n = lib.parts(rows, vocab)
            pieces = (vocab + piece - 1) // piece
            assert 1 <= n <= min(64, pieces)
            cuts = [pieces * k // n for k in range(n + 1)]  # as the workgroups take them
            assert cuts[0] == 0 and cuts[-1] == pieces and all(a < b for a, b in zip(cuts, cuts[1:]))
            assert rows * n <= max(1024, rows)
            assert n == 1 or n == min(64, pieces) or rows * (n + 1) > 1024


def test_scratch_holds_every_smaller_call(lib):
    for made in (1, 2, 15, 16, 17, 100, 512, 1023, 1024, 1025, 5000):
        have = lib.all_parts(made)
        for rows in range(1, made + 1):
            for vocab in (1, 5000, 100000, 2 ** 31 - 17):
                assert rows * lib.parts(rows, vocab) <= have


def test_columns_of_tables(lib):
    for group in list(range(1, 1025)):
        c = lib.columns(group)
        assert c in (8, 16, 32, 64) and c * group <= lib.ints()
