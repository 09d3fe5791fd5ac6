"""Rotary positions on the device against cos and sin in 64 bits.

Tolerance: a turn is reduced in f64 and rounded to f32 (2^-25 of a turn,
2 pi 2^-25 radians), sincospi is within 4 units in the last place, and each
result is two products and a sum: (|x1| + |x2|) * magnitude * 12 * 2^-24, and
the element type's rounding of the result."""
import numpy as np
import pytest

from cache_oracle import EPS, from_bits, rotate, to_bits
from manta_amd import _lib, rocm

pytestmark = pytest.mark.gpu


def _close(got, want, x, dtype, magnitude):
    # |x1| + |x2| <= 2 max of the head's columns, and the type's smallest step
    # (f16 2^-24: half of it)
    scale = 2 * np.abs(x).max(axis=-1, keepdims=True) * abs(magnitude)
    tol = scale * 12 * 2.0 ** -24 + np.abs(want) * EPS[dtype] * 1.001 + (2.0 ** -25 if dtype == "f16" else 1e-38)
    bad = np.abs(got - want) > tol
    assert not bad.any(), (np.abs(got - want)[bad].max(), int(bad.sum()))


def _run(rt, rng, dtype, layout, tokens, heads, d, rot, pos, inverse=False, magnitude=1.0, in_place=False, freqs=None):
    freqs = rocm.rotary_freqs(rot) if freqs is None else freqs
    r = rt.rotary_bind(freqs, layout=layout, magnitude=magnitude)
    p = rt.to_device(np.asarray(pos, np.int32))
    xs, parts = [], []
    for h in heads:
        x = to_bits(rng.standard_normal((tokens, h, d)), dtype)
        a = rt.to_device(x)
        parts.append((a, a if in_place else rt.to_device(np.zeros_like(x))))
        xs.append(from_bits(x, dtype))
    rt.rotary(r, p, parts, inverse=inverse, dtype=dtype)
    for x, (_, out) in zip(xs, parts):
        want = rotate(x, pos, freqs, layout, magnitude, inverse)
        got = from_bits(out.download(), dtype)
        _close(got, want, x, dtype, magnitude)
        np.testing.assert_array_equal(got[..., rot:], x[..., rot:])  # columns past the rotated ones
    r.close()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,d,rot", [
    (1, (1,), 2, 2), (1, (6, 6), 64, 64), (3, (32, 8), 128, 128), (7, (5, 1), 96, 32), (600, (4, 2), 64, 16),
    (2, (3,), 80, 80), (5, (2, 1, 1, 3), 33, 22), (4, (12, 2), 256, 256), (9, (7,), 192, 50), (1, (3, 1), 100, 4),
])
def test_sizes_layouts_types(rt, dtype, layout, tokens, heads, d, rot):
    print("rotary", dtype, layout, tokens, heads, d, rot, flush=True)
    rng = np.random.default_rng(tokens * 1000 + d + rot)
    _run(rt, rng, dtype, layout, tokens, heads, d, rot, rng.integers(0, 100000, tokens))


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_in_place_gradient_magnitude(rt, dtype, layout, in_place, inverse):
    print("rotary in place", dtype, layout, in_place, inverse, flush=True)
    rng = np.random.default_rng(9)
    _run(rt, rng, dtype, layout, 11, (4, 2), 64, 48, rng.integers(0, 4096, 11), inverse, 1.25, in_place)


def test_far_and_negative_positions(rt):
    print("rotary far", flush=True)
    rng = np.random.default_rng(2)
    pos = [0, 1, -1, 2 ** 31 - 1, -2 ** 31, 123456789, -7654321, 1 << 24]
    # a turn of a position of 2^31 in f64: 2^31 * 2^-53 of it is lost
    _run(rt, rng, "f32", "half", len(pos), (2,), 64, 64, pos)
    f = rocm.rotary_freqs(64, scaling="blend", factor=16.0, low=1.0, high=32.0, original=4096.0)
    _run(rt, rng, "f32", "interleaved", len(pos), (2,), 64, 64, pos, freqs=f)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_gradient_is_the_adjoint_and_matches_differences(rt, layout):
    """<rotate(x), g> = <x, gradient(g)>, and the change of a loss along a
    direction."""
    print("rotary gradient", layout, flush=True)
    rng = np.random.default_rng(5)
    x, g, u = (rng.standard_normal((6, 3, 32)).astype(np.float32) for _ in range(3))
    pos = rng.integers(0, 5000, 6)
    f = rocm.rotary_freqs(24)
    r = rt.rotary_bind(f, layout=layout, magnitude=1.5)
    p = rt.to_device(pos.astype(np.int32))

    def turn(a, inverse=False):
        d = rt.to_device(np.ascontiguousarray(a, np.float32))
        rt.rotary(r, p, [(d, d)], inverse=inverse)
        return d.download().astype(np.float64)

    y, dx = turn(x), turn(g, True)
    size = np.abs(g).astype(np.float64).sum() * 6
    assert abs((y * g).sum() - (x * dx).sum()) <= 24 * 2.0 ** -24 * 1.5 * size
    step = 0.25  # the loss <rotate(x), g> is linear: any step will do
    difference = ((turn(x + step * u) - turn(x - step * u)) * g).sum() / (2 * step)
    assert abs(difference - (u * dx).sum()) <= 24 * 2.0 ** -24 * 1.5 * size / step


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_strided_views(rt, dtype):
    """q and k inside one [tokens, columns] buffer, rows that do not start on
    16 bytes, heads before tokens."""
    print("rotary strided", dtype, flush=True)
    rng = np.random.default_rng(3)
    t, d = 13, 32
    f = rocm.rotary_freqs(d)
    r = rt.rotary_bind(f)
    pos = rng.integers(0, 1000, t)
    p = rt.to_device(pos.astype(np.int32))
    for offset, width in ((0, 5 * d), (1, 5 * d + 3), (8, 5 * d + 8)):
        buf = to_bits(rng.standard_normal((t, width)), dtype)
        a = rt.to_device(buf)
        q = rocm.View(a, (t, 2, d), (width, d, 1), offset)
        k = rocm.View(a, (t, 1, d), (width, d, 1), offset + 2 * d)
        rt.rotary(r, p, [(q, q), (k, k)], dtype=dtype)
        x, got = from_bits(buf, dtype), from_bits(a.download(), dtype)
        part = x[:, offset:offset + 3 * d].reshape(t, 3, d)
        _close(got[:, offset:offset + 3 * d].reshape(t, 3, d), rotate(part, pos, f, "half"), part, dtype, 1.0)
        keep = np.ones(width, bool)
        keep[offset:offset + 3 * d] = False
        np.testing.assert_array_equal(got[:, keep], x[:, keep])
    x = to_bits(rng.standard_normal((3, t, d)), dtype)
    a, o = rt.to_device(x), rt.to_device(np.zeros((t, 3, d), x.dtype))
    rt.rotary(r, p, [(rocm.View(a, (t, 3, d), (d, t * d, 1)), o)], dtype=dtype)
    x = from_bits(x, dtype).transpose(1, 0, 2)
    _close(from_bits(o.download(), dtype), rotate(x, pos, f, "half"), x, dtype, 1.0)


def test_no_tokens_and_refusals(rt):
    print("rotary refusals", flush=True)
    r = rt.rotary_bind(rocm.rotary_freqs(64))
    e = rt.empty((0, 2, 64), np.float32)
    rt.rotary(r, rt.empty((0,), np.int32), [(e, e)])
    x, p = rt.to_device(np.ones((2, 2, 32), np.float32)), rt.to_device(np.zeros(2, np.int32))
    with pytest.raises(_lib.MantaRocmError, match="rotated columns"):
        rt.rotary(r, p, [(x, x)])
    big = rt.to_device(np.ones((2, 1, 257), np.float32))
    with pytest.raises(_lib.MantaRocmError, match="to 256"):
        rt.rotary(r, p, [(big, big)])
    with rocm.Runtime(0) as other:
        o = other.rotary_bind(rocm.rotary_freqs(32))
        with pytest.raises(_lib.MantaRocmError, match="another runtime"):
            rt.rotary(o, p, [(x, x)])
    with pytest.raises(_lib.MantaRocmError, match="runtime is destroyed"):
        rt.rotary(o, p, [(x, x)])
    o.close()
    np.testing.assert_array_equal(x.download(), np.ones((2, 2, 32), np.float32))
