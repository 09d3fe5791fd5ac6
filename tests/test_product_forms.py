"""The rule that chooses a product's kernel (decode_layout.hpp, plain C++): the
GPU tests' shapes take every form, and every form covers its results."""
import ctypes as C
import os
import subprocess

import pytest

import test_gpu_product
import test_gpu_product_forms as forms

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NAMES = ["few16x16", "few16x32", "few32x32", "few64x32", "tile64deep", "tile64row", "tile64", "tile128", "tile256"]
UNITS = 256  # compute units

SHIM = r"""
#include "decode_layout.hpp"
using namespace manta;
extern "C" int form(long long rows, long long n, int gated, long long cus) {
    return product_form(rows, weight_rows(n, gated) / 16, gated, cus);
}
"""


@pytest.fixture(scope="module")
def form(tmp_path_factory):
    d = tmp_path_factory.mktemp("product_forms")
    src, so = d / "shim.cpp", d / "libshim.so"
    src.write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I" + os.path.join(ROOT, "include"),
                    "-I" + os.path.join(ROOT, "manta_amd", "csrc"), str(src), "-o", str(so)], check=True)
    f = C.CDLL(str(so)).form
    f.argtypes = [C.c_longlong, C.c_longlong, C.c_int, C.c_longlong]
    return lambda rows, n, gated: NAMES[f(rows, n, gated, UNITS)]


def test_the_tested_shapes_take_every_form(form):
    for gated, few, tiles in ((0, test_gpu_product.SHAPES, forms.PLAIN),
                              (1, [s for s in test_gpu_product.SHAPES if s[0] * s[2] < 600000], forms.GATED)):
        assert {form(r, n, gated) for r, _, n in few + tiles} == set(NAMES[gated:])
        # ... and more columns than make a strip a unit
        assert {form(r, n, gated) for r, _, n in tiles if r <= 32} == {"few16x32", "few32x32"}
        stages, edges = {}, {}
        for r, width, n in tiles:
            name = form(r, n, gated)
            if name not in NAMES[4:]:
                continue
            per = 2 if name in ("tile64deep", "tile64") else 1  # steps of 64 columns a stage
            stages.setdefault(name, set()).add((width + 127) // 128 * 2 // per)
            edges.setdefault(name, set()).add((r % 64 != 0, n % 8 != 0))
        assert set(stages) == set(NAMES[4:]), stages
        assert stages["tile64deep"] == {1, 2, 3, 5} and stages["tile64"] == {1, 2, 3, 5}
        for name in ("tile64row", "tile128", "tile256"):
            assert stages[name] == {2, 4, 6}
        # ragged rows and columns, and results that are whole tiles or pieces
        assert all((True, True) in e and any(not ragged for _, ragged in e) for e in edges.values()), edges


def test_gated_weights_are_never_split_between_tiles_of_one_block(form):
    for rows in (1, 16, 33, 100, 1000, 30000):
        for n in (1, 16, 17, 300, 4096, 50000):
            assert form(rows, n, 1) != "few16x16"
