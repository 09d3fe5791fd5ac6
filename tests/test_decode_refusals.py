"""What the decoding calls refuse before they look at a device."""
import ctypes as C

import numpy as np
import pytest

from manta_amd import _lib, cache, decode
from manta_amd._lib import call

BYTES = np.zeros(4096, np.int8)
P = BYTES.ctypes.data // 16 * 16 + 16


class _Array:
    def __init__(self, shape, dtype=np.float32, strides=None):
        self.shape, self.dtype, self.strides, self.addr = shape, np.dtype(dtype), strides, P


class _Rows:
    def __init__(self, rows, width):
        self.rows, self.width, self.codes, self.scales = rows, width, _Array((1,), np.int8), _Array((rows,))


@pytest.mark.parametrize("width,n,gate,message", [
    (0, 4, 0, "width"), (131073, 4, 0, "width"), (4, 0, 0, "columns"), (4, (1 << 24) + 1, 0, "columns"),
    (4, 4, 3, "gate"), (4, 4, -1, "gate")])
def test_weights(width, n, gate, message):
    out = C.c_void_p()
    with pytest.raises(_lib.MantaRocmError, match=message):
        call("manta_rocm_weight_bind", None, P, P, width, n, gate, C.byref(out))
    assert not out.value


def test_weights_need_their_arrays():
    out = C.c_void_p()
    for a, b in ((None, P), (P, None)):
        with pytest.raises(_lib.MantaRocmError, match="nil pointer"):
            call("manta_rocm_weight_bind", None, a, b, 4, 4, 0, C.byref(out))
    with pytest.raises(ValueError, match="int8"):
        decode.Weight(None, np.zeros((3, 4), np.float32), np.zeros(4), None)
    with pytest.raises(ValueError, match="scales"):
        decode.Weight(None, np.zeros((3, 4), np.int8), np.zeros(3), None)
    with pytest.raises(ValueError, match="as many columns"):
        decode.Weight(None, np.zeros((3, 5), np.int8), np.zeros(5), "silu")
    with pytest.raises(ValueError, match="unknown gate"):
        decode.Weight(None, np.zeros((3, 4), np.int8), np.zeros(4), "relu")


def test_quantised_bytes():
    f = _lib.load().manta_rocm_quantized_bytes
    assert [f(r, w) for r, w in ((0, 1), (1, 1), (16, 128), (17, 129))] == [0, 16 * 128, 16 * 128, 32 * 256]
    assert f(1 << 25, 131072) == (1 << 25) * 131072
    assert [f(r, w) for r, w in ((-1, 1), (1, 0), (1, 131073), ((1 << 25) + 1, 1))] == [-1] * 4


@pytest.mark.parametrize("args,message", [
    ((9, P, 8, 2, 8, None, 0.0, P, P), "element type"), ((32, P, 7, 2, 8, None, 0.0, P, P), "7 elements apart"),
    ((32, P, -1, 1, 8, None, 0.0, P, P), "elements apart"), ((32, P, 8, -2, 8, None, 0.0, P, P), "bad shape"),
    ((32, P, 8, 2, 8, P, 0.0, P, P), "eps"), ((32, P, 8, 2, 8, P, float("nan"), P, P), "eps"),
    ((32, P, 8, 2, 8, P, 1e300, P, P), "eps"), ((32, None, 8, 2, 8, None, 0.0, P, P), "nil pointer"),
    ((32, P, 8, 2, 8, None, 0.0, P + 4, P), "16 bytes"), ((32, P, 8, 2, 8, None, 0.0, P, None), "nil pointer"),
    ((32, P, 8, 2, 8, None, 0.0, P, P), "nil rocm runtime")])
def test_quantising(args, message):
    with pytest.raises(_lib.MantaRocmError, match=message):
        call("manta_rocm_quantize_rows", None, *args)


def test_products_without_a_weight():
    with pytest.raises(_lib.MantaRocmError, match="nil weight"):
        call("manta_rocm_matmul_q8", None, None, P, P, 1, 32, None, 0, P, 8)


def test_shapes_of_products():
    w = decode.Weight.__new__(decode.Weight)
    w.width, w.n, w.handle = 8, 6, None
    with pytest.raises(ValueError, match="mismatch"):
        decode.matmul_q8(None, w, _Rows(2, 9), None, None, "f32")
    with pytest.raises(ValueError, match=r"out must be \[2, 6\]"):
        decode.matmul_q8(None, w, _Rows(2, 8), _Array((2, 7)), None, None)
    with pytest.raises(ValueError, match="add must be"):
        decode.matmul_q8(None, w, _Rows(2, 8), _Array((2, 6)), _Array((3, 6)), None)
    with pytest.raises(TypeError, match="one element type"):
        decode.matmul_q8(None, w, _Rows(2, 8), _Array((2, 6)), _Array((2, 6), np.uint16), None)
    with pytest.raises(TypeError, match="elements"):
        decode.matmul_q8(None, w, _Rows(2, 8), None, None, "f64")
    with pytest.raises(ValueError, match="norm must be"):
        decode.quantize_rows(None, _Array((2, 8)), _Rows(2, 8), _Array((7,)), 1e-6, None)
    with pytest.raises(ValueError, match="quantized rows"):
        decode.quantize_rows(None, _Array((2, 8)), _Rows(3, 8), None, 1e-6, None)


def test_normed_rotation():
    for eps in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(_lib.MantaRocmError, match="eps"):
            call("manta_rocm_rotary_normed", None, None, 32, P, 1, 8, b"", P, 1, eps)
    with pytest.raises(_lib.MantaRocmError, match="nil norms"):
        call("manta_rocm_rotary_normed", None, None, 32, P, 1, 8, b"", None, 1, 1e-6)
    x = _Array((2, 3, 8))
    with pytest.raises(ValueError, match="a norm .* for each"):
        cache.rotary_normed(None, None, _Array((2,), np.int32), [(x, x)], [], 1e-6, None)
    with pytest.raises(ValueError, match=r"a norm must be f32 \[8\]"):
        cache.rotary_normed(None, None, _Array((2,), np.int32), [(x, x)], [_Array((7,))], 1e-6, None)


@pytest.mark.parametrize("groups,beams,best,message", [
    (0, 4, 4, "no groups"), (1, 0, 4, "64 beams"), (1, 65, 4, "64 beams"), (1, 4, 0, "64 results"),
    (1, 4, 65, "64 results"), (1 << 20, 2, 4, "1048576"), (-1, 4, 4, "64 beams")])
def test_beams(groups, beams, best, message):
    out = C.c_void_p()
    with pytest.raises(_lib.MantaRocmError, match=message):
        call("manta_rocm_beams_create", None, groups, beams, best, C.byref(out))


def test_shapes_of_beams():
    b = decode.Beams.__new__(decode.Beams)
    b.handle = None
    i32 = np.int32
    good = [_Array((2, 4, 9)), _Array((2, 4)), _Array((2, 8), i32), _Array((2, 8), i32), _Array((2, 8))]
    for k, bad, message in ((0, _Array((8, 9)), "logits"), (1, _Array((2, 5)), "scores"), (2, _Array((3, 8), i32), "parents"),
                            (3, _Array((2, 7), i32), "tokens"), (4, _Array((2, 8), i32), "totals"),
                            (0, _Array((2, 4, 9), strides=(50, 9, 1)), "follow")):
        with pytest.raises(ValueError, match=message):
            b.select(*[bad if j == k else a for j, a in enumerate(good)])
    with pytest.raises(ValueError, match="ended"):
        b.select(*good, ended=_Array((2, 8), i32))


def test_no_more_beams_than_tokens():
    from manta_amd import answer

    model = type("Model", (), {"vocab": 3})()
    with pytest.raises(ValueError, match="4 beams of a vocabulary of 3"):
        answer.Answerer(None, model, 1, 4, 16, 0)


def test_reorder_without_a_cache():
    with pytest.raises(_lib.MantaRocmError, match="nil cache"):
        call("manta_rocm_cache_reorder", None, None, P, P, 4, 2)
