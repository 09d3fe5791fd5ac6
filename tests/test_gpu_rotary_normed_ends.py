"""Normed rotation of heads that are not finite."""
import numpy as np
import pytest

from cache_oracle import from_bits, to_bits
from decode_oracle import rotary_normed
from manta_amd import rocm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d,rot", [(64, 64), (64, 32), (80, 50), (20, 4), (256, 2)])
def test_infinities_as_the_formula_has_them(rt, dtype, layout, d, rot):
    print("rotary_normed infinities", dtype, layout, d, rot, flush=True)
    rng = np.random.default_rng(d)
    x = rng.standard_normal((4, 2, d)).astype(np.float32)
    x[0, 0, 1] = np.inf
    x[1, 1, d - 1] = -np.inf
    x[2, 0, [0, d // 2]] = np.inf
    x[3, 1, 3] = np.nan
    w, freqs, pos = rng.uniform(0.5, 2.0, d).astype(np.float32), rocm.rotary_freqs(rot), np.arange(4) * 7
    with np.errstate(invalid="ignore"):
        want, off = rotary_normed(x, w, 1e-6, pos, freqs, layout, 1.0)
    out = rt.to_device(np.zeros_like(to_bits(x, dtype)))
    rt.rotary_normed(rt.rotary_bind(freqs, layout=layout), rt.to_device(pos.astype(np.int32)),
                     [(rt.to_device(to_bits(x, dtype)), out)], [rt.to_device(w)], dtype=dtype)
    got = from_bits(out.download(), dtype)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    for t, h in ((0, 0), (1, 1), (2, 0)):
        live = ~np.isnan(want[t, h])
        assert 0 < live.sum() < d and (got[t, h][live] == 0).all()
    assert np.isnan(got[3, 1]).all()
