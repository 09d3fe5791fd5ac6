"""Norms of queries and keys with their rotation, against 64 bits with the
bound of decode_oracle.rotary_normed."""
import numpy as np
import pytest

from cache_oracle import from_bits, to_bits
from decode_oracle import rotary_normed, rounding
from manta_amd import rocm

pytestmark = pytest.mark.gpu


def _check(got, x, norm, eps, pos, freqs, layout, magnitude, dtype):
    want, off = rotary_normed(x, norm, eps, pos, freqs, layout, magnitude)
    bad = ~(np.abs(got - want) <= off + rounding(np.abs(want) + off, dtype))
    assert not bad.any(), (int(bad.sum()), got[bad][:4], want[bad][:4])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,d,rot", [
    (1, (1,), 2, 2), (1, (6, 6), 64, 64), (3, (32, 8), 128, 128), (7, (5, 1), 96, 32), (600, (4, 2), 64, 16),
    (2, (3,), 80, 80), (5, (2, 1, 1, 3), 33, 22), (4, (12, 2), 256, 256), (9, (7,), 192, 50), (1, (3, 1), 255, 2), (3, (2, 1), 256, 2), (70, (3, 3), 80, 50), (5, (4,), 77, 44),
    (1100, (9, 3), 128, 64), (2, (70, 5), 128, 96), (6, (3, 2), 128, 126), (3, (2, 1), 80, 8), (2, (1,), 20, 4),
    (65, (7, 2), 47, 40), (4, (3,), 24, 16)])
def test_sizes_layouts_types(rt, dtype, layout, tokens, heads, d, rot):
    print("rotary_normed", dtype, layout, tokens, heads, d, rot, flush=True)
    rng = np.random.default_rng(tokens + 10 * d + rot)
    freqs = rocm.rotary_freqs(rot)
    pos = rng.integers(0, 1000000, tokens)
    r = rt.rotary_bind(freqs, layout=layout, magnitude=1.25)
    p = rt.to_device(pos.astype(np.int32))
    parts, norms, hosts = [], [], []
    for i, h in enumerate(heads):
        bits = to_bits(rng.standard_normal((tokens, h, d)) * 10.0 ** rng.integers(-2, 3, (tokens, h, 1)), dtype)
        a = rt.to_device(bits)
        parts.append((a, a if i % 2 else rt.to_device(np.zeros_like(bits))))  # every second in place
        w = rng.uniform(-2, 2, d).astype(np.float32) if i != 2 else None
        norms.append(w)
        hosts.append(from_bits(bits, dtype))
    rt.rotary_normed(r, p, parts, [None if w is None else rt.to_device(w) for w in norms], eps=1e-5, dtype=dtype)
    for x, w, (_, out) in zip(hosts, norms, parts):
        got = from_bits(out.download(), dtype)
        _check(got, x, w, 1e-5, pos, freqs, layout, 1.25, dtype)
        if w is None:  # what is not normed is rotary's, bit for bit
            b = rt.to_device(to_bits(x, dtype))
            rt.rotary(r, p, [(b, b)], dtype=dtype)
            np.testing.assert_array_equal(from_bits(b.download(), dtype), got)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_strided_views(rt, dtype):
    """q and k inside one [tokens, columns] buffer, at any alignment; what lies
    beside them stays."""
    print("rotary_normed strided", dtype, flush=True)
    rng = np.random.default_rng(3)
    t, d = 13, 32
    f = rocm.rotary_freqs(d)
    r = rt.rotary_bind(f)
    pos = rng.integers(0, 1000, t)
    p = rt.to_device(pos.astype(np.int32))
    w = [rng.uniform(0.5, 2, d).astype(np.float32) for _ in range(2)]
    for offset, width in ((0, 5 * d), (1, 5 * d + 3), (8, 5 * d + 8)):
        bits = to_bits(rng.standard_normal((t, width)), dtype)
        a = rt.to_device(bits)
        q = rocm.View(a, (t, 2, d), (width, d, 1), offset)
        k = rocm.View(a, (t, 1, d), (width, d, 1), offset + 2 * d)
        rt.rotary_normed(r, p, [(q, q), (k, k)], [rt.to_device(x) for x in w], dtype=dtype)
        x, got = from_bits(bits, dtype), from_bits(a.download(), dtype)
        for view, norm, c0, h in ((q, w[0], offset, 2), (k, w[1], offset + 2 * d, 1)):
            part = x[:, c0:c0 + h * d].reshape(t, h, d)
            _check(got[:, c0:c0 + h * d].reshape(t, h, d), part, norm, 1e-6, pos, f, "half", 1.0, dtype)
        np.testing.assert_array_equal(got[:, :offset], x[:, :offset])
        np.testing.assert_array_equal(got[:, offset + 3 * d:], x[:, offset + 3 * d:])


def test_heads_at_the_ends_of_the_range(rt):
    """A head of zeros stays zero, one of large or small numbers is normed, one
    that is not finite does not touch another."""
    print("rotary_normed ends", flush=True)
    rng = np.random.default_rng(1)
    x = rng.standard_normal((6, 2, 64)).astype(np.float32)
    x[0, 0] = 0.0
    x[1, 1] *= 1e30
    x[2, 0] *= 1e-30
    x[3, 1, 7] = np.nan
    x[4, 0, 7] = np.inf
    f = rocm.rotary_freqs(64)
    r = rt.rotary_bind(f)
    pos = np.arange(6)
    a = rt.to_device(x)
    w = np.ones(64, np.float32)
    rt.rotary_normed(r, rt.to_device(pos.astype(np.int32)), [(a, a)], [rt.to_device(w)], eps=1e-6)
    got = a.download()
    assert (got[0, 0] == 0).all() and np.isnan(got[3, 1]).all() and np.isnan(got[4, 0]).any()
    fine = [(t, h) for t in range(6) for h in range(2) if (t, h) not in ((3, 1), (4, 0))]
    for t, h in fine:
        _check(got[t:t + 1, h:h + 1], x[t:t + 1, h:h + 1], w, 1e-6, pos[t:t + 1], f, "half", 1.0, "f32")
    # eps counts: the small head is not blown up to 1
    assert np.abs(got[2, 0]).max() < 1e-25
