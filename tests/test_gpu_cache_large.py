"""The 8-bit cache near the largest f32 numbers, where x * 127 and code * max
are no f32 numbers any more: append's two kernels against the definition, bit
for bit."""
import numpy as np
import pytest

from cache_oracle import Model, from_bits, to_bits

pytestmark = pytest.mark.gpu

MAXIMA = [1e36, 2.6e36, 3e36, 1e37, 4e37, 5e37, 3e38]


def _dev(rt, x):
    return rt.to_device(np.asarray(x, np.int32))


def _offsets(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tokens", [1, 16])
def test_new_values(rt, dtype, tokens):
    """A page a sequence and magnitude; one token each goes to the plain kernel,
    16 to the one of 16-byte pieces."""
    print("append large", dtype, tokens, flush=True)
    rng = np.random.default_rng(tokens)
    n, d = len(MAXIMA), 64
    x = rng.uniform(-1, 1, (n, tokens, 2, d)) * rng.choice([1e-3, 0.05, 0.5, 1.0], (n, tokens, 2, d))
    x[:, 0, :, 5], x[:, -1, :, 6] = 1.0, -1.0
    x = to_bits((x * np.array(MAXIMA)[:, None, None, None]).reshape(n * tokens, 2, d), dtype)
    m = Model(1, n, 16, 2, d, n, 1)
    assert m.extend(range(n), [tokens] * n)
    c = m.upload(rt)
    off = _offsets([tokens] * n)
    xd = rt.to_device(x)
    c.append(0, xd, xd, _dev(rt, off), dtype=dtype)
    y = from_bits(x, dtype)
    with np.errstate(all="ignore"):
        m.append(0, y, y, off)
    assert (np.abs(m.k).max((3, 4)) == 127).all()  # the largest element has the largest code
    m.check_pages(c)
    c.close()
