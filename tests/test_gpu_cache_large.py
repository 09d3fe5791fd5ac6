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


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tokens", [1, 14])
def test_values_that_were_there(rt, dtype, tokens):
    """A page of two tokens goes on with larger ones: round_half_even(code * old
    / max), each of its f32 steps on numbers 2^-8 as large, which changes no
    rounding."""
    print("append raises", dtype, tokens, flush=True)
    rng = np.random.default_rng(tokens + 50)
    pairs = [(1e35, 2e35), (2e36, 2.6e36), (3e36, 3.5e36), (1e37, 2e37), (1e37, 3e38), (4e37, 5e37), (3e38, 3.3e38),
             (1.0, 3e38), (1e-38, 1e38)]
    n, d = len(pairs), 64
    m = Model(1, n, 16, 2, d, n, 1)
    assert m.extend(range(n), [2 + tokens] * n)
    rows = m.tables[:, 0]
    old, new = (np.array(x, np.float32) for x in zip(*pairs))
    m.k[0, rows, :, :2] = rng.integers(-127, 128, (n, 2, 2, d))
    m.v[0, rows, :, :, :2] = rng.integers(-127, 128, (n, 2, d, 2))
    m.k[0, rows, :, 0, :2] = 127, -127
    m.km[0, rows], m.vm[0, rows] = old[:, None], old[:, None]
    c = m.upload(rt)
    x = rng.uniform(-0.5, 0.5, (n, tokens, 2, d)) * new[:, None, None, None]
    x[:, -1, :, 3] = new[:, None]
    x = to_bits(x.reshape(n * tokens, 2, d), dtype)
    xd = rt.to_device(x)
    c.append(0, xd, xd, _dev(rt, _offsets([tokens] * n)), dtype=dtype)
    big = np.abs(from_bits(x, dtype)).reshape(n, -1).max(1)
    h = np.float32(2.0 ** -8)

    def again(codes):  # [n, ...]
        codes = codes.astype(np.float32)
        at = (slice(None),) + (None,) * (codes.ndim - 1)
        return np.rint(codes * (old * h)[at] / (big * h)[at])

    np.testing.assert_array_equal(c.k_max.download()[0, rows], np.stack([big, big], 1))
    np.testing.assert_array_equal(c.k_codes.download()[0, rows, :, :2], again(m.k[0, rows, :, :2]))
    np.testing.assert_array_equal(c.v_codes.download()[0, rows, :, :, :2], again(m.v[0, rows, :, :, :2]))
    c.close()


@pytest.mark.parametrize("d", [64, 33])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_values_read_back(rt, dtype, d):
    """code * max / 127 with maxima up to the largest number: two roundings, and
    the result's; the plain kernel (33 columns) and that of 16-byte pieces."""
    print("read large", dtype, d, flush=True)
    rng = np.random.default_rng(d)
    maxima = np.array(MAXIMA + [1.0, np.finfo(np.float32).max], np.float32)
    n = len(maxima)
    m = Model(1, n, 16, 1, d, n, 1)
    assert m.extend(range(n), [16] * n)
    rows = m.tables[:, 0]
    m.k[0, rows, :, :, :d] = rng.integers(-127, 128, (n, 1, 16, d))
    m.v[0, rows, :, :d] = rng.integers(-127, 128, (n, 1, d, 16))
    m.k[0, rows, :, 3, :2], m.v[0, rows, :, 2, :2] = (127, -127), (127, -127)
    m.km[0, rows], m.vm[0, rows] = maxima[:, None], maxima[::-1, None]
    c = m.upload(rt)
    outs = [rt.empty((16 * n, 1, d), np.float32 if dtype == "f32" else np.uint16) for _ in range(2)]
    c.read(0, _dev(rt, _offsets([16] * n)), outs[0], outs[1], dtype=dtype)
    for j, o in enumerate(outs):
        got = from_bits(o.download(), dtype).astype(np.float64)
        want = np.concatenate([m.values(0, i)[j] for i in range(n)])
        top = np.float64(3.3895313892515355e38)  # bf16's largest; beyond its half step a result is infinite
        seen = np.abs(want) <= (top if dtype == "bf16" else np.inf)
        assert np.isfinite(got[seen]).all()
        tol = np.abs(want) * (2.0 ** -23 + (2.0 ** -8 if dtype == "bf16" else 0)) * 1.01
        assert (np.abs(got - want)[seen] <= tol[seen]).all()
    c.close()
