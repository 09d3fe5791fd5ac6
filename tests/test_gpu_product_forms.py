"""Products in 8 bits in every form that the rule on sizes takes (tiles of 64,
128 and 256, one stage of summed columns to several, ragged edges on both
sides), with the bound of decode_oracle.product."""
import numpy as np
import pytest

from cache_oracle import from_bits, to_bits
from decode_oracle import U, activate, quantise, rounding
from manta_amd import rocm

pytestmark = pytest.mark.gpu

# (rows, summed columns, result columns): tests/test_product_forms.py says which form each takes
PLAIN = [(16, 130, 8501), (31, 130, 8501), (64, 300, 5001), (200, 130, 1504),
         (500, 60, 1101), (500, 130, 1104), (449, 300, 1101), (500, 640, 1030), (60, 200, 8301),
         (50, 60, 16501), (64, 130, 16512), (33, 300, 16501),
         (700, 60, 1543), (700, 130, 1536), (641, 300, 1603), (700, 640, 1543),
         (2049, 60, 2101), (2048, 130, 2112), (2100, 300, 2101),
         (2900, 60, 2931), (2816, 130, 2960), (2818, 300, 2931)]
GATED = [(16, 130, 4251), (31, 130, 4251), (64, 300, 2501), (200, 130, 752),
         (500, 60, 521), (500, 130, 528), (449, 300, 521), (500, 640, 515), (60, 200, 4151),
         (50, 60, 8261), (64, 130, 8256), (33, 300, 8261),
         (700, 60, 783), (700, 130, 784), (641, 300, 801), (700, 640, 783),
         (2049, 60, 1051), (2048, 130, 1056), (2100, 300, 1051),
         (2900, 60, 1467), (2816, 130, 1480), (2818, 300, 1467)]


def _case(rt, rows, width, columns, dtype, seed):
    rng = np.random.default_rng(seed)
    w = rng.integers(-127, 128, (width, columns)).astype(np.int8)
    ws = (rng.uniform(0.5, 1.5, columns) / (73 * np.sqrt(width))).astype(np.float32)
    bits = to_bits(rng.standard_normal((rows, width)), dtype)
    q = rt.quantize_rows(rt.to_device(bits), dtype=dtype)
    codes, scales = q.values()
    np.testing.assert_array_equal(codes, quantise(from_bits(bits, dtype))[0])
    # whole numbers below 2^53: exact
    y = (codes.astype(np.float64) @ w.astype(np.float64)) * np.outer(scales.astype(np.float64), ws.astype(np.float64))
    return rng, w, ws, q, y


def _check(got, want, off, dtype):
    bad = ~(np.abs(got - want) <= off * 1.001 + rounding(np.abs(want) + off, dtype))
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])


class _Wide:
    """Room for [rows, n] inside a larger buffer, of which all else stays."""

    def __init__(self, rt, host, dtype):
        rows, n = host.shape
        self.dtype, self.rows, self.n = dtype, rows, n
        whole = to_bits(np.full((rows + 3, n + 5), 7.0), dtype)
        whole[:rows, 2:2 + n] = host
        self.array = rt.to_device(whole)
        self.view = rocm.View(self.array, (rows, n), (n + 5, 1), 2)

    def result(self):
        x = from_bits(self.array.download(), self.dtype)
        assert (x[:, :2] == 7.0).all() and (x[:, 2 + self.n:] == 7.0).all() and (x[self.rows:] == 7.0).all()
        return x[:self.rows, 2:2 + self.n]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,width,n", PLAIN)
def test_products(rt, dtype, rows, width, n):
    print("matmul_q8 forms", dtype, rows, width, n, flush=True)
    rng, w, ws, q, y = _case(rt, rows, width, n, dtype, rows + width + n)
    weight = rt.weight(w, ws)
    _check(from_bits(rt.matmul_q8(weight, q, dtype=dtype).download(), dtype), y, 3 * U * np.abs(y), dtype)
    host = to_bits(rng.standard_normal((rows, n)), dtype)
    want = y + from_bits(host, dtype)
    off = 3 * U * np.abs(y) + U * np.abs(want)
    wide = _Wide(rt, host, dtype)
    rt.matmul_q8(weight, q, out=wide.view, add=wide.view, dtype=dtype)  # in place
    _check(wide.result(), want, off, dtype)
    whole = rt.matmul_q8(weight, q, add=rt.to_device(host), dtype=dtype)
    _check(from_bits(whole.download(), dtype), want, off, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,width,n", GATED)
def test_gated_products(rt, dtype, rows, width, n):
    gate = "silu" if (rows + width + n) % 2 else "gelu"
    print("matmul_q8 gated forms", gate, dtype, rows, width, n, flush=True)
    _, w, ws, q, y = _case(rt, rows, width, 2 * n, dtype, rows + width + n + 1)
    weight = rt.weight(w, ws, gate=gate)
    v, u = y[:, :n], y[:, n:]
    want = activate(v, gate) * u
    off = np.abs(u) * np.abs(v) * (1.13 * 3 + 2 * 0.28 * 6) * U + 8 * U * np.abs(want)
    _check(from_bits(rt.matmul_q8(weight, q, dtype=dtype).download(), dtype), want, off, dtype)
    wide = _Wide(rt, to_bits(np.zeros((rows, n)), dtype), dtype)
    rt.matmul_q8(weight, q, out=wide.view, dtype=dtype)
    _check(wide.result(), want, off, dtype)
