"""The key/value cache's layout header (plain C++): what shapes and batches it
refuses, the mapping of a ragged batch's rows to page pieces against a loop,
and the words its kernels report errors in; and the refusals of the C entry
points that need no device."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from manta_amd import _lib, cache, rocm

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SHIM = r"""
#include "cache_layout.hpp"
using namespace manta;
extern "C" {
const char* shape(long long a, long long b, long long c, long long d, long long e, long long f, long long g) {
    MantaRocmCacheShape s{a, b, c, d, e, f, g};
    return check_cache_shape(s);
}
const char* strides(long long t, long long h, long long d, long long ts, long long hs) {
    return check_strides(t, h, d, ts, hs);
}
const char* batch(long long n, long long t, long long s, int listed) { return check_batch(n, t, s, listed); }
long long slots(long long t, long long n, int shift) { return ragged_slots(t, n, shift); }
long long base(int off, long long i, int shift) { return ragged_base(off, i, shift); }
int piece(int a, int b, int len, long long local, int shift, int* out) {
    Piece p;
    if (!ragged_piece(a, b, len, local, shift, &p)) return 0;
    out[0] = p.index; out[1] = p.from; out[2] = p.to; out[3] = p.row;
    return 1;
}
void describe(int kind, long long a, long long b, char* out) { describe_cache_error(cache_error(kind, a, b), out, 160); }
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("cache_layout")
    src, so = d / "shim.cpp", d / "libshim.so"
    src.write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I" + os.path.join(ROOT, "include"),
                    "-I" + os.path.join(ROOT, "manta_amd", "csrc"), str(src), "-o", str(so)], check=True)
    L = C.CDLL(str(so))
    for f in ("shape", "strides", "batch"):
        getattr(L, f).restype = C.c_char_p
    L.shape.argtypes = [C.c_longlong] * 7
    L.strides.argtypes = [C.c_longlong] * 5
    L.batch.argtypes = [C.c_longlong] * 3 + [C.c_int]
    L.slots.restype = L.base.restype = C.c_longlong
    L.slots.argtypes = [C.c_longlong, C.c_longlong, C.c_int]
    L.base.argtypes = [C.c_int, C.c_longlong, C.c_int]
    L.piece.argtypes = [C.c_int, C.c_int, C.c_int, C.c_longlong, C.c_int, C.POINTER(C.c_int)]
    L.describe.argtypes = [C.c_int, C.c_longlong, C.c_longlong, C.c_char_p]
    return L


GOOD = dict(layers=2, pages=10, page=16, kv=2, d=64, seqs=3, table=5)


@pytest.mark.parametrize("change,text", [
    (dict(), None), (dict(layers=0), "must be positive"), (dict(pages=0), "must be positive"),
    (dict(pages=-4), "must be positive"), (dict(seqs=0), "must be positive"), (dict(table=0), "must be positive"),
    (dict(kv=0), "must be positive"), (dict(page=8), "page_tokens"), (dict(page=48), "page_tokens"),
    (dict(page=256), "page_tokens"), (dict(d=0), "head_dim"), (dict(d=257), "head_dim"), (dict(d=256), None),
    (dict(d=1), None), (dict(table=1 << 30), "int32 lengths"), (dict(kv=70000), "65535"),
    (dict(pages=1 << 40), "too many"), (dict(seqs=1 << 20, table=1 << 14), "book"),
])
def test_shapes(lib, change, text):
    s = dict(GOOD, **change)
    got = lib.shape(s["layers"], s["pages"], s["page"], s["kv"], s["d"], s["seqs"], s["table"])
    assert (got is None) if text is None else (got is not None and text in got.decode())


@pytest.mark.parametrize("args,text", [
    ((4, 2, 64, 128, 64), None), ((4, 2, 64, 64, 256), None), ((4, 2, 64, -128, 64), "negative"),
    ((4, 2, 64, 128, 63), "head stride"), ((4, 2, 64, 63, 512), "token stride"), ((1, 1, 64, 0, 0), None),
])
def test_strides(lib, args, text):
    got = lib.strides(*args)
    assert (got is None) if text is None else (got is not None and text in got.decode())


@pytest.mark.parametrize("args,text", [
    ((3, 7, 3, 0), None), ((4, 7, 3, 0), "more sequences"), ((4, 7, 3, 1), None), ((-1, 7, 3, 1), "negative"),
    ((1, -1, 3, 1), "negative"), ((1 << 40, 1, 3, 1), "too many"), ((1, 1 << 40, 3, 1), "too many"),
])
def test_batches(lib, args, text):
    got = lib.batch(*args)
    assert (got is None) if text is None else (got is not None and text in got.decode())


@pytest.mark.parametrize("shift", [4, 5, 6, 7])
def test_every_row_lies_in_one_piece(lib, shift):
    """Random batches, with lengths of 0, counts of 0 and counts beyond the
    length: the slots' pieces cover each row of position >= 0 once, at its
    page and place, and nothing else."""
    rng = np.random.default_rng(shift)
    page = 1 << shift
    out = (C.c_int * 4)()
    for _ in range(200):
        n = int(rng.integers(1, 6))
        counts = [int(x) for x in rng.choice([0, 1, 2, page - 1, page, page + 1, 3 * page + 5], n)]
        lens = [max(0, c + int(rng.choice([-3, 0, 1, page - 1, page, 2 * page + 3]))) for c in counts]
        off = np.concatenate([[0], np.cumsum(counts)]).astype(int) + int(rng.integers(0, 3))
        total = int(off[-1])
        seen = {}
        slots = lib.slots(total, n, shift)
        for i in range(n):
            lo, hi = lib.base(int(off[i]), i, shift), lib.base(int(off[i + 1]), i + 1, shift)
            assert 0 <= lo <= hi <= slots
            for slot in range(lo, hi):
                if not lib.piece(int(off[i]), int(off[i + 1]), lens[i], slot - lo, shift, out):
                    continue
                index, a, b, row = out
                assert 0 <= a < b <= page
                for t in range(a, b):
                    assert row + t - a not in seen
                    seen[row + t - a] = (i, index * page + t)
            # a slot past the sequence's own is never one of its pieces
            assert not lib.piece(int(off[i]), int(off[i + 1]), lens[i], hi - lo, shift, out)
            assert not lib.piece(int(off[i]), int(off[i + 1]), lens[i], -1, shift, out)
        want = {}
        for i in range(n):
            for j in range(counts[i]):
                pos = lens[i] - counts[i] + j
                if pos >= 0:
                    want[int(off[i]) + j] = (i, pos)
        assert seen == want


@pytest.mark.parametrize("kind,a,b,text", [
    (1, -1, 0, "cache sequence -1 out of range"), (1, 70000, 0, "cache sequence 70000 out of range"),
    (2, 12345, 0, "cache page 12345 out of range"), (2, -1, 0, "cache page -1 out of range"),
    (3, 900000000, 5, "cache is out of pages: 900000000 needed, 5 free"), (4, 3, 0, "cache sequence 3 is not empty"),
    (5, 2, -7, "cache sequence 2: count -7 out of range"),
])
def test_error_words(lib, kind, a, b, text):
    buf = C.create_string_buffer(160)
    lib.describe(kind, a, b, buf)
    assert buf.value.decode() == text


def test_frequencies_are_their_formulas():
    p = np.arange(32)
    f = 10000.0 ** (-2.0 * p / 64)
    np.testing.assert_allclose(rocm.rotary_freqs(64), f, rtol=1e-14)
    np.testing.assert_allclose(rocm.rotary_freqs(64, scaling="linear", factor=4.0), f / 4, rtol=1e-14)
    np.testing.assert_allclose(rocm.rotary_freqs(64, base=500.0, scaling="base", factor=8.0),
                               (500.0 * 8.0 ** (64 / 62)) ** (-2.0 * p / 64), rtol=1e-13)
    got = rocm.rotary_freqs(64, scaling="blend", factor=8.0, low=1.0, high=4.0, original=8192.0)
    turns = 8192.0 * f / (2 * np.pi)
    np.testing.assert_allclose(got[turns >= 4.0], f[turns >= 4.0], rtol=1e-14)
    np.testing.assert_allclose(got[turns <= 1.0], f[turns <= 1.0] / 8, rtol=1e-14)
    between = (turns > 1) & (turns < 4)
    g = (turns[between] - 1) / 3
    assert between.any()
    np.testing.assert_allclose(got[between], f[between] * ((1 - g) / 8 + g), rtol=1e-13)
    np.testing.assert_allclose(rocm.rotary_freqs(2, scaling="base", factor=8.0), [1.0])


@pytest.mark.parametrize("kw,text", [
    (dict(rot=63), "even"), (dict(rot=0), "even"), (dict(rot=258), "even"), (dict(rot=64, base=0.0), "base"),
    (dict(rot=64, base=float("inf")), "base"), (dict(rot=64, scaling="linear", factor=0.0), "factor"),
    (dict(rot=64, scaling="blend", factor=2.0, low=4.0, high=4.0), "blend"),
    (dict(rot=64, scaling="blend", factor=2.0, original=float("nan")), "blend"),
])
def test_frequencies_refused(kw, text):
    with pytest.raises(_lib.MantaRocmError, match=text):
        rocm.rotary_freqs(**kw)


class _Array:
    """Stands in for a device array: shape, type and address only."""

    def __init__(self, shape, dtype, addr=4096):
        self.shape, self.dtype, self.addr = tuple(shape), np.dtype(dtype), addr
        self.nbytes = int(np.prod(shape)) * self.dtype.itemsize


class _Nothing:
    handle = None
    rot = 64


def test_wrapper_refuses_what_the_entry_points_cannot_see():
    x, pos = _Array((5, 2, 64), np.uint16), _Array((5,), np.int32)
    bad = [
        ([], pos, None, ValueError, "at least one"),
        ([(x, _Array((5, 2, 32), np.uint16))], pos, None, ValueError, "out must be"),
        ([(x, x), (_Array((4, 2, 64), np.uint16),) * 2], pos, None, ValueError, "agree"),
        ([(x, x)], _Array((4,), np.int32), None, ValueError, "positions"),
        ([(x, x)], _Array((5,), np.int64), None, ValueError, "positions"),
        ([(x, x)], pos, "f32", TypeError, "does not hold"),
        ([(x, x)], pos, "f64", TypeError, "f32, f16 or bf16"),
        ([(_Array((5, 2, 64), np.int16),) * 2], pos, None, TypeError, "f32, f16 or bf16"),
        ([(_Array((5, 128), np.uint16),) * 2], pos, None, ValueError, "tokens, heads"),
    ]
    for parts, p, dtype, error, text in bad:
        with pytest.raises(error, match=text):
            cache.rotary(_Nothing, _Nothing, p, parts, False, dtype)


def test_views_stay_in_their_array():
    a = _Array((10, 96), np.uint16)
    a.rt = None
    v = rocm.View(a, (10, 2, 16), (96, 16, 1), 64)
    assert v.addr == 4096 + 128
    for shape, strides, offset in (((10, 2, 17), (96, 16, 1), 64), ((11, 2, 16), (96, 16, 1), 0),
                                   ((10, 2, 16), (96, 16, 2), 0), ((10, 2, 16), (96, 16, 1), -1),
                                   ((10, 2, 16), (96, -16, 1), 32), ((10, 16), (96, 16, 1), 0)):
        with pytest.raises(ValueError, match="view"):
            rocm.View(a, shape, strides, offset)


def _heads(**kw):
    h = _lib.Heads(4096, 8192, 2, 128, 64, 128, 64)
    for k, v in kw.items():
        setattr(h, k, v)
    return h


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=64), "element type"), (dict(tokens=-1), "token count"), (dict(nparts=0), "1 to 4 tensors"),
    (dict(nparts=5), "1 to 4 tensors"), (dict(h=dict(heads=0)), "heads"), (dict(h=dict(x_dev=None)), "nil pointer"),
    (dict(h=dict(out_dev=None)), "nil pointer"), (dict(h=dict(x_head=32)), "head stride"),
    (dict(h=dict(out_token=-1)), "negative"), (dict(h=dict(out_dev=4096, out_token=256)), "equal strides"),
    (dict(), "nil frequencies"),
])
def test_rotary_entry_refuses_before_it_needs_a_device(kw, text):
    parts = (_lib.Heads * 5)(*[_heads(**kw.get("h", {})) for _ in range(5)])
    with pytest.raises(_lib.MantaRocmError, match=text):
        _lib.call("manta_rocm_rotary", None, None, kw.get("dtype", _lib.F16), 4096, kw.get("tokens", 3), 64, parts,
                  kw.get("nparts", 1), 0)


def test_cache_entries_without_a_cache_or_runtime():
    h = C.c_void_p()
    shape = _lib.CacheShape(1, 4, 16, 1, 64, 2, 2)
    with pytest.raises(_lib.MantaRocmError, match="nil rocm runtime"):
        _lib.call("manta_rocm_cache_create", None, C.byref(shape), C.byref(h))
    shape.page_tokens = 17
    with pytest.raises(_lib.MantaRocmError, match="page_tokens"):
        _lib.call("manta_rocm_cache_create", None, C.byref(shape), C.byref(h))
    with pytest.raises(_lib.MantaRocmError, match="nil shape"):
        _lib.call("manta_rocm_cache_create", None, None, C.byref(h))
    nil = [("extend", (1, 1, 1)), ("fork", (1, 1, None, 1)), ("release", (1, None, 1)), ("compact", (None,)),
           ("copy_pages", (1, 1, 1)), ("append", (0, 16, 1, 1, 1, 1, 1, 1, 1, None, 1, 1)),
           ("read", (0, 16, 1, 1, 1, 1, 1, 1, 1, None, 1, 1)),
           ("attention", (0, 16, C.byref(_heads()), None, 1, None, 1, 1, 1.0, 1, 0, 1))]
    for name, args in nil:
        with pytest.raises(_lib.MantaRocmError, match="cache_%s: nil cache" % name):
            _lib.call("manta_rocm_cache_" + name, None, None, *args)
    assert _lib.load().manta_rocm_cache_buffers(None, C.byref(_lib.CacheBuffers())) == _lib.ERROR
    _lib.load().manta_rocm_cache_destroy(None)
    _lib.load().manta_rocm_rotary_unbind(None)
    with pytest.raises(_lib.MantaRocmError, match="nil rocm runtime"):
        _lib.call("manta_rocm_copy", None, 1, 2, 3)
    f = np.ones(4)
    r = C.c_void_p()
    for rot, layout, mag, text in ((7, 0, 1.0, "even"), (8, 5, 1.0, "layout"), (8, 0, float("nan"), "magnitude"),
                                   (8, 0, 1.0, "nil rocm runtime")):
        with pytest.raises(_lib.MantaRocmError, match=text):
            _lib.call("manta_rocm_rotary_bind", None, f.ctypes.data, rot, layout, mag, C.byref(r))
    f[2] = np.inf
    with pytest.raises(_lib.MantaRocmError, match="frequency 2"):
        _lib.call("manta_rocm_rotary_bind", None, f.ctypes.data, 8, 0, 1.0, C.byref(r))
