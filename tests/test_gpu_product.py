"""Products in 8 bits on the device.  Codes are compared bit for bit, results
with the bound of decode_oracle.product."""
import numpy as np
import pytest

from cache_oracle import from_bits, to_bits
from decode_oracle import U, product, quantise
from manta_amd import rocm

pytestmark = pytest.mark.gpu


def _weight(rng, width, columns):
    return (rng.integers(-127, 128, (width, columns)).astype(np.int8),
            (rng.uniform(0.5, 1.5, columns) / (73 * np.sqrt(width))).astype(np.float32))


def _check(got, want, tol):
    assert got.shape == want.shape
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], tol[bad][:4])


def _quantised(rt, x, dtype, norm=None, eps=1e-6, stride=None, offset=0):
    rows, width = x.shape
    stride = stride or width
    host = to_bits(np.full((offset + rows * stride,), 3.0), dtype)
    bits = to_bits(x, dtype)
    for r in range(rows):
        host[offset + r * stride:offset + r * stride + width] = bits[r]
    a = rt.to_device(host)
    view = rocm.View(a, (rows, width), (stride, 1), offset)
    q = rt.quantize_rows(view, norm=None if norm is None else rt.to_device(norm), eps=eps, dtype=dtype)
    codes, scales = q.values()
    want, want_scales = quantise(from_bits(bits, dtype), norm, eps)
    np.testing.assert_array_equal(codes, want)
    # one rounding, or that of f64 steps before it
    np.testing.assert_allclose(scales, want_scales, rtol=U * 1.0001, atol=2.0 ** -150)
    # padding columns are 0
    pitch = (width + 127) // 128 * 128
    c = q.codes.download().reshape(-1, pitch // 64, 4, 16, 16).transpose(0, 3, 1, 2, 4).reshape(-1, pitch)
    assert not c[:rows, width:].any()
    return q, codes, scales


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("rows,width,stride,offset", [
    (1, 1, 1, 0), (1, 128, 128, 0), (3, 64, 64, 0), (5, 100, 107, 3), (16, 384, 384, 0), (17, 129, 136, 8),
    (40, 1000, 1000, 0), (2, 4096, 4100, 4), (1, 16383, 16383, 1), (3, 20000, 20000, 0), (33, 8192, 8200, 0),
    (2, 131072, 131072, 0)])
def test_quantised_rows(rt, dtype, normed, rows, width, stride, offset):
    print("quantize", dtype, normed, rows, width, stride, offset, flush=True)
    rng = np.random.default_rng(rows * 7 + width)
    x = (rng.standard_normal((rows, width)) * 10.0 ** rng.integers(-3, 3, (rows, 1))).astype(np.float32)
    norm = rng.uniform(-1.5, 1.5, width).astype(np.float32) if normed else None
    _quantised(rt, x, dtype, norm, 1e-5, stride, offset)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("normed", [False, True])
def test_rows_at_the_ends_of_the_range(rt, dtype, normed):
    """Zeros, numbers below the smallest normal, the largest, infinities, NaN."""
    print("quantize ends", dtype, normed, flush=True)
    x = np.ones((9, 70), np.float32)
    x[0] = 0.0
    x[1] = 2.0 ** -130
    x[2, 5] = np.inf
    x[3, 69] = np.nan
    x[4, :] = -0.0
    x[5] *= 2.0 ** -126
    x[6, 3] = -np.inf
    x[7, 10] = 3.0e38
    x[8] *= 1.0e25
    norm = np.full(70, 0.5, np.float32) if normed else None
    q, codes, scales = _quantised(rt, x, dtype, norm, 1e-6)
    w, ws = np.ones((70, 20), np.int8), np.ones(20, np.float32)
    y = rt.matmul_q8(rt.weight(w, ws), q, dtype="f32").download()
    assert np.isnan(y[[2, 3, 6]]).all() and not np.isnan(y[[0, 1, 4, 5]]).any()
    assert (y[[0, 1, 4]] == 0).all()


SHAPES = [(1, 1, 1), (1, 64, 16), (2, 100, 17), (12, 384, 1152), (15, 63, 40), (16, 128, 33), (17, 200, 100),
          (31, 1000, 24), (32, 384, 384), (33, 512, 65), (48, 4096, 96), (49, 640, 272), (64, 130, 48), (65, 384, 130),
          (100, 256, 128), (129, 1111, 257), (200, 384, 768), (257, 64, 512), (300, 2000, 300), (513, 448, 129),
          (1000, 128, 40), (1, 16384, 50), (3, 5000, 3000), (256, 1024, 1024), (700, 768, 1536), (2049, 320, 1000)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,width,n", SHAPES)
def test_products(rt, dtype, rows, width, n):
    print("matmul_q8", dtype, rows, width, n, flush=True)
    rng = np.random.default_rng(rows + 3 * width + 5 * n)
    w, ws = _weight(rng, width, n)
    q, codes, scales = _quantised(rt, rng.standard_normal((rows, width)).astype(np.float32), dtype)
    weight = rt.weight(w, ws)
    want, tol = product(codes, scales.astype(np.float64), w, ws, dtype)
    _check(from_bits(rt.matmul_q8(weight, q, dtype=dtype).download(), dtype), want, tol)
    # onto something, in place, inside a wider buffer whose other columns stay
    add = rng.standard_normal((rows, n)).astype(np.float32)
    wide = to_bits(np.full((rows, n + 5), 7.0), dtype)
    wide[:, 2:2 + n] = to_bits(add, dtype)
    a = rt.to_device(wide)
    view = rocm.View(a, (rows, n), (n + 5, 1), 2)
    rt.matmul_q8(weight, q, out=view, add=view, dtype=dtype)
    want, tol = product(codes, scales.astype(np.float64), w, ws, dtype, from_bits(to_bits(add, dtype), dtype))
    got = from_bits(a.download(), dtype)
    _check(got[:, 2:2 + n], want, tol)
    assert (got[:, :2] == 7.0).all() and (got[:, 2 + n:] == 7.0).all()
    # ... and from another, whole rows aligned
    b = rt.to_device(to_bits(add, dtype))
    _check(from_bits(rt.matmul_q8(weight, q, add=b, dtype=dtype).download(), dtype), want, tol)


@pytest.mark.parametrize("gate", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,width,n", [s for s in SHAPES if s[0] * s[2] < 600000])
def test_gated_products(rt, gate, dtype, rows, width, n):
    print("matmul_q8 gated", gate, dtype, rows, width, n, flush=True)
    rng = np.random.default_rng(rows + 3 * width + 5 * n + 1)
    w, ws = _weight(rng, width, 2 * n)
    ws[:n] *= rng.uniform(0, 8, n).astype(np.float32)  # gates far out on both sides
    q, codes, scales = _quantised(rt, rng.standard_normal((rows, width)).astype(np.float32), dtype)
    want, tol = product(codes, scales.astype(np.float64), w, ws, dtype, gate=gate)
    _check(from_bits(rt.matmul_q8(rt.weight(w, ws, gate=gate), q, dtype=dtype).download(), dtype), want, tol)


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_the_widest_sums_are_exact(rt, rows):
    """131072 columns of codes of one sign: sums near 2^31, right to the last
    unit before their one rounding."""
    print("matmul_q8 widest", rows, flush=True)
    width = 131072
    x = np.ones((rows, width), np.float32)
    x[:, ::2] = 0.9921875  # 126 / 127
    w = np.full((width, 18), 127, np.int8)
    w[:, 3] = -128
    w[::3, 4] = -127
    q, codes, scales = _quantised(rt, x, "f32")
    want, tol = product(codes, scales.astype(np.float64), w, np.ones(18, np.float32), "f32")
    _check(rt.matmul_q8(rt.weight(w, np.ones(18, np.float32)), q, dtype="f32").download(), want, tol)


def test_one_row_does_not_touch_another(rt):
    """A row that is not finite is NaN, the others are as without it; rows do
    not depend on how many there are."""
    print("matmul_q8 rows", flush=True)
    rng = np.random.default_rng(4)
    x = rng.standard_normal((300, 256)).astype(np.float32)
    w, ws = _weight(rng, 256, 160)
    weight = rt.weight(w, ws)
    whole = rt.matmul_q8(weight, rt.quantize_rows(rt.to_device(x)), dtype="f32").download()
    for a, b in ((0, 1), (5, 21), (0, 64), (100, 300)):
        part = rt.matmul_q8(weight, rt.quantize_rows(rt.to_device(x[a:b])), dtype="f32").download()
        np.testing.assert_array_equal(part, whole[a:b])
    x[17, 3] = np.nan
    y = rt.matmul_q8(weight, rt.quantize_rows(rt.to_device(x)), dtype="f32").download()
    assert np.isnan(y[17]).all()
    np.testing.assert_array_equal(np.delete(y, 17, 0), np.delete(whole, 17, 0))


def test_no_rows(rt):
    print("matmul_q8 empty", flush=True)
    w = rt.weight(np.ones((5, 3), np.int8), np.ones(3, np.float32))
    q = rt.quantize_rows(rt.empty((0, 5), np.float32))
    assert rt.matmul_q8(w, q, dtype="f32").download().shape == (0, 3)
