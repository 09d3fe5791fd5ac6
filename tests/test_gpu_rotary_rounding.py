"""Where rotary rounds: an angle comes from the exact product of position and
turns, and a pair's two results are a product and a fused one each."""
from fractions import Fraction

import numpy as np
import pytest

from cache_oracle import from_bits, to_bits

pytestmark = pytest.mark.gpu


def _fused(a, b, c):
    """f32 a * b + c, rounded once.  The product is exact in f64; a sum that is
    not is made odd in its last place, so that rounding it again is right."""
    p, c = a.astype(np.float64) * b.astype(np.float64), c.astype(np.float64)
    s = p + c
    t = s - p
    left = (p - (s - t)) + (c - t)
    bits = s.view(np.int64).copy()
    towards = np.where((left > 0) == (s > 0), 1, -1)
    bits += np.where((left != 0) & (bits & 1 == 0), towards, 0)
    return bits.view(np.float64).astype(np.float32)


def test_the_fused_sum_is_rounded_once():
    rng = np.random.default_rng(0)
    a, b, c = ((rng.standard_normal(300) * 2.0 ** rng.integers(-3, 3, 300)).astype(np.float32) for _ in range(3))
    for x, y, z, got in zip(a, b, c, _fused(a, b, c)):
        exact = Fraction(float(x)) * Fraction(float(y)) + Fraction(float(z))
        near = [np.nextafter(got, np.float32(-np.inf)), got, np.nextafter(got, np.float32(np.inf))]
        off = [abs(Fraction(float(n)) - exact) for n in near]
        assert off[1] <= min(off)


def _call(rt, x, pos, freqs, layout, dtype, normed):
    r, out = rt.rotary_bind(freqs, layout=layout), rt.to_device(np.zeros_like(x))
    p = rt.to_device(pos.astype(np.int32))
    if normed:
        rt.rotary_normed(r, p, [(rt.to_device(x), out)], [None], dtype=dtype)
    else:
        rt.rotary(r, p, [(rt.to_device(x), out)], dtype=dtype)
    return out.download()


def _split(y, layout, half):
    return (y[..., :half], y[..., half:2 * half]) if layout == "half" else (y[..., 0:2 * half:2], y[..., 1:2 * half:2])


@pytest.mark.parametrize("normed", [False, True])  # (of a head without a norm)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d,rot", [(64, 64), (80, 50)])
def test_a_pair_has_two_roundings(rt, layout, normed, d, rot):
    """Pairs (1, 0) give cos and sin as the device has them; then every result
    is known to its last bit."""
    print("rotary rounding", layout, normed, d, rot, flush=True)
    rng = np.random.default_rng(d)
    t, half = 300, rot // 2
    freqs = 10000.0 ** (-np.arange(half) / half)
    pos = rng.integers(0, 100000, t)
    one = np.zeros((t, 1, d), np.float32)
    _split(one, layout, half)[0][...] = 1.0
    c, s = _split(_call(rt, one, pos, freqs, layout, "f32", normed), layout, half)
    x = rng.standard_normal((t, 3, d)).astype(np.float32)
    x1, x2 = _split(x, layout, half)
    y1, y2 = _split(_call(rt, x, pos, freqs, layout, "f32", normed), layout, half)
    c, s = np.broadcast_to(c, x1.shape), np.broadcast_to(s, x1.shape)
    np.testing.assert_array_equal(y1, _fused(x1, c, -(x2 * s)))
    np.testing.assert_array_equal(y2, _fused(x2, c, x1 * s))


@pytest.mark.parametrize("normed", [False, True])
def test_far_positions_that_are_almost_whole_turns(rt, normed):
    """The sine of what is left of a turn, which is far below the f64 rounding
    of position * turns (2^-25 at 2^28 turns).  What is left is exact to f64's
    2^-53 of it, in f32 to 2^-24, and the sine adds a few 2^-24: 2^-20 of it."""
    print("rotary far", normed, flush=True)
    freq = 1.0
    turns = freq / (2.0 * np.pi)
    pos = np.arange(2 ** 31 - 40_000_000, 2 ** 31, dtype=np.int64)
    left = pos * turns
    near = pos[np.argsort(np.abs(left - np.rint(left)))[:64]]
    exact = [Fraction(int(p)) * Fraction(turns) for p in near]
    rest = np.array([float(e - round(e)) for e in exact])
    assert (np.abs(rest) < 1e-5).all() and (rest != 0).all()
    x = np.zeros((len(near), 1, 2), np.float32)
    x[..., 0] = 1.0
    got = _call(rt, x, near, np.array([freq]), "half", "f32", normed)[:, 0, 1]
    want = np.sin(2 * np.pi * rest)
    assert (np.abs(got - want) <= 2.0 ** -20 * np.abs(want)).all()


@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d,rot", [(64, 64), (47, 40), (80, 50), (20, 4)])
def test_narrow_results_are_those_of_f32(rt, d, rot, dtype, layout, normed):
    """16-bit elements: the f32 results of the same numbers, rounded once more,
    whichever kernel and lane works them out."""
    print("rotary narrow", d, rot, dtype, layout, normed, flush=True)
    rng = np.random.default_rng(3)
    t = 8199
    freqs, pos = 10000.0 ** (-np.arange(rot // 2) / rot), rng.integers(0, 100000, t)
    bits = to_bits(rng.standard_normal((t, 3, d)), dtype)
    wide = _call(rt, from_bits(bits, dtype), pos, freqs, layout, "f32", normed)
    np.testing.assert_array_equal(_call(rt, bits, pos, freqs, layout, dtype, normed), to_bits(wide, dtype))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d,rot", [(64, 64), (47, 40), (80, 50), (20, 4)])
def test_narrow_normed_results_are_those_of_f32(rt, d, rot, layout):
    rng = np.random.default_rng(4)
    t = 8199
    r = rt.rotary_bind(10000.0 ** (-np.arange(rot // 2) / rot), layout=layout)
    p, w = rt.to_device(rng.integers(0, 100000, t).astype(np.int32)), rt.to_device(rng.uniform(0.5, 2, d).astype(np.float32))
    bits = to_bits(rng.standard_normal((t, 3, d)), "f16")
    found = []
    for x, dtype in ((bits, "f16"), (from_bits(bits, "f16"), "f32")):
        out = rt.to_device(np.zeros_like(x))
        rt.rotary_normed(r, p, [(rt.to_device(x), out)], [w], dtype=dtype)
        found.append(out.download())
    # the sums of squares come in another order of their f64 additions: one factor
    # in 10^8 rounds to its neighbour
    assert (found[0] != to_bits(found[1], "f16")).mean() < 1e-5
