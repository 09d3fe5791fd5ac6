"""Attention whose keys are split over workgroups, with values that the joining
of the parts must not take past the largest number: the bounds of
Model.attend, as test_gpu_cache_attention.py has them."""
import numpy as np
import pytest

from cache_oracle import filled
from test_gpu_cache_attention import _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("counts,longest", [([1], None), ([8], None), ([1, 1], 1 << 22), ([7, 8], 1 << 22), ([60], None)])
def test_large_values_in_parts(rt, counts, longest):
    """Means of several thousand values of up to 5e37: the parts' sums of
    weights are in the hundreds."""
    print("large parts", counts, longest, flush=True)
    rng = np.random.default_rng(sum(counts))
    m = filled(rng, [6000, 3000][:len(counts)], 64, 1, 64)
    rows = m.tables[m.tables >= 0]
    m.vm[:, rows] = 5e37
    m.v[0, rows] = np.abs(m.v[0, rows])  # (-128 does not occur)
    _check(rt, m, rng, "bf16", 2, counts, longest=longest, q_scale=0.3)
