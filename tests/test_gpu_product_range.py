"""Quantised rows whose largest value times 127 is past f32's range."""
import numpy as np
import pytest

from cache_oracle import from_bits, to_bits

pytestmark = pytest.mark.gpu


def _codes(z):
    """The definition in f32 of z and its largest 2^-7 times as large: what is
    in range then, and the same quotients (of z above 2^-119; codes 0 below)."""
    f32 = np.float32
    z = z * f32(2.0 ** -7)
    return np.rint((z * f32(127)) / np.abs(z).max(1, keepdims=True)).astype(np.int8)


@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("width", [3, 40, 3000, 20000, 40000])
def test_codes_of_the_largest_numbers(rt, width, dtype, normed):
    print("quantize largest", width, dtype, normed, flush=True)
    rng = np.random.default_rng(width)
    x = np.zeros((5, width), np.float32)
    x[0, :3] = [3.3e38, 3.0e36, 1.0e36]
    x[1, :3] = [-2.0e37, 2.0e37, 1.0e35]
    x[2, :3] = [2.6e36, -2.7e36, 1.0e30]  # on both sides of 2^121
    x[3] = rng.standard_normal(width) * 5e37
    x[4] = rng.standard_normal(width)
    x = from_bits(to_bits(np.clip(x, -3.3e38, 3.3e38), dtype), dtype)
    norm = rng.uniform(0.5, 1.0, width).astype(np.float32) if normed else None
    if normed:
        norm[:3] = 1.0
    q = rt.quantize_rows(rt.to_device(to_bits(x, dtype)), norm=None if norm is None else rt.to_device(norm), dtype=dtype)
    codes, scales = q.values()
    assert codes[0, :3].tolist() == [127, 1, 0]
    assert codes[1, :3].tolist() == [-127, 127, 1]
    assert abs(int(codes[2, 0])) == round(127 * float(x[2, 0]) / float(-x[2, 1])) and codes[2, 1] == -127
    z = x if norm is None else x * norm
    np.testing.assert_array_equal(codes, _codes(z))
    want = np.abs(z).max(1).astype(np.float64) / 127
    if normed:
        want = want / np.sqrt((x.astype(np.float64) ** 2).mean(1) + 1e-6)
    np.testing.assert_allclose(scales, want, rtol=2.0 ** -24 * 1.0001)
