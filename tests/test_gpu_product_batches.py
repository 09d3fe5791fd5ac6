"""Batches of fewer rows in the memory of a larger one."""
import numpy as np
import pytest

from decode_oracle import quantise

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width", [70, 2000])
def test_ragged_batches_share_memory(rt, width):
    print("quantized first", width, flush=True)
    rng = np.random.default_rng(width)
    whole = rt.quantized(100, width)
    w, ws = rng.integers(-127, 128, (width, 40)).astype(np.int8), np.full(40, 0.01, np.float32)
    weight = rt.weight(w, ws)
    for rows in (100, 1, 33, 16, 0, 99):
        x = rng.standard_normal((rows, width)).astype(np.float32)
        q = whole.first(rows)
        assert rt.quantize_rows(rt.to_device(x), q) is q and q.codes is whole.codes
        codes, scales = q.values()
        if rows:
            want, _ = quantise(x)
            np.testing.assert_array_equal(codes, want)
        assert codes.shape == (rows, width) and scales.shape == (rows,)
        alone = rt.matmul_q8(weight, rt.quantize_rows(rt.to_device(x)), dtype="f32").download()
        np.testing.assert_array_equal(rt.matmul_q8(weight, q, dtype="f32").download(), alone)
        assert q.first(rows).rows == rows
    for rows in (-1, 34):
        with pytest.raises(ValueError, match="of 33"):
            whole.first(33).first(rows)
