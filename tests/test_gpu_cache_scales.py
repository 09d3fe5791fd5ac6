"""Attention over pages whose v scales lie far apart.  The bound of a row knows
only what the row sees: the sum of |weight * v|, and the largest of weight *
v_max, below which the operands of the second product lose bits."""
import numpy as np
import pytest

from cache_oracle import EPS, filled, from_bits, to_bits

pytestmark = pytest.mark.gpu

MANY = 1 << 22  # (as `longest`: the evenly cut kernel)


def _dev(rt, x):
    return rt.to_device(np.asarray(x, np.int32))


def _offsets(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)


def _attend(m, q, off, scale, window, dtype):
    """(out, tolerance, lse, its tolerance) of causal rows, in 64 bits."""
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    lse, ltol = np.zeros(q.shape[:2]), np.zeros(q.shape[:2])
    group = q.shape[1] // m.heads
    for i in range(len(off) - 1):
        k, v = m.values(0, i)
        n, c = len(k), off[i + 1] - off[i]
        v_max = np.repeat(m.vm[0, m.tables[i, :m.held(i)]].astype(np.float64), m.page, 0)[:n]
        for j in range(c):
            row, pos = off[i] + j, n - c + j
            see = slice(max(0, pos - window + 1) if window else 0, pos + 1)
            for h in range(q.shape[1]):
                kk, vv = k[see, h // group], v[see, h // group]
                sc = kk @ q[row, h] * scale
                p = np.exp(sc - sc.max())
                l = p.sum()
                out[row, h], lse[row, h] = p @ vv / l, sc.max() + np.log(l)
                # a score: products and sums of f32, its scaling, exp2's argument
                delta = ((m.d + 8) * 2.0 ** -24 * (np.abs(kk) @ np.abs(q[row, h])).max() * abs(scale)
                         + 8 * 2.0 ** -24 * max(1.0, np.abs(sc).max()))
                # log2 of a scale (up to 2^7) and what is added to it: four roundings
                delta += 4 * 2.0 ** -24 * 2.0 ** 7
                # p in f16: half a step, 2^-11; below the normal range half of its smallest
                # step, 2^-25, of operands that reach 2^7 at least; f32 sums
                tol[row, h] = ((p @ np.abs(vv) / l) * (2 * delta + 2.0 ** -11 + (len(p) + 64) * 2.0 ** -24)
                               + len(p) * 2.0 ** -32 * (p * v_max[see, h // group]).max() / l)
                ltol[row, h] = delta + 2.0 ** -21 * max(1.0, abs(lse[row, h])) + len(p) * 2.0 ** -24
    # the result's own rounding (f16's smallest step is 2^-24, bf16's 2^-133)
    return out, tol + np.abs(out) * EPS[dtype] + (2.0 ** -25 if dtype == "f16" else 2.0 ** -133), lse, ltol


def _run(rt, m, bits, off, dtype, scale, window, longest):
    c = m.upload(rt)
    out, lse = rt.empty(bits.shape, np.uint16), rt.empty(bits.shape[:2], np.float32)
    c.attention(0, rt.to_device(bits), _dev(rt, off), out=out, lse=lse, scale=scale, window=window, longest=longest,
                dtype=dtype)
    res = out.download(), lse.download()
    c.close()
    return res


def _check(rt, m, rng, dtype, heads, counts, window=0, longest=None, q_scale=2.0, scale=None):
    off = _offsets(counts)
    bits = to_bits(rng.standard_normal((int(off[-1]), heads, m.d)) * q_scale, dtype)
    scale = m.d ** -0.5 if scale is None else scale
    want, tol, lse, ltol = _attend(m, from_bits(bits, dtype).astype(np.float64), off, scale, window, dtype)
    got, gl = _run(rt, m, bits, off, dtype, scale, window, longest)
    got = from_bits(got, dtype).astype(np.float64)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], tol[bad][:5])
    assert (np.abs(gl - lse) <= ltol).all()


# rows a sequence and longest: single tokens, tiles of 32 rows, cut evenly, prompts
FORMS = [([1, 1], None), ([8, 5], None), ([1, 1], MANY), ([7, 8], MANY), ([120, 70], None)]


@pytest.mark.parametrize("counts,longest", FORMS)
@pytest.mark.parametrize("low,high,dtype", [(-6, 4, "f16"), (-8, 8, "bf16"), (-18, 18, "bf16"), (-37, 37, "bf16")])
def test_random_scales(rt, counts, longest, low, high, dtype):
    """Every page its own power of ten, scores that differ by tens."""
    print("scales", counts, longest, low, high, dtype, flush=True)
    rng = np.random.default_rng(high)
    m = filled(rng, [400, 170], 16, 2, 64)
    rows = m.tables[m.tables >= 0]
    m.vm[:, rows] = 10.0 ** rng.uniform(low, high, m.vm[:, rows].shape)
    for q_scale in (0.3, 2.0, 20.0):
        _check(rt, m, rng, dtype, 4, counts, longest=longest, q_scale=q_scale)


@pytest.mark.parametrize("counts,longest", FORMS)
@pytest.mark.parametrize("ratio", [2.0 ** 14, 1e6, 1e8, 1e18, 1e36])
def test_large_values_of_no_weight(rt, counts, longest, ratio):
    """A page of values `ratio` times as large whose scores are 45 and more
    below the others: it weighs exp(-45) and no more."""
    print("no weight", counts, longest, ratio, flush=True)
    rng = np.random.default_rng(5)
    m = filled(rng, [330, 200], 16, 1, 64)
    for s in range(2):
        rows = m.tables[s, :m.held(s)]
        # the first column alone decides: 60 for all keys but those of the large page
        m.k[0, rows] = 0
        m.k[0, rows, 0, :, 0] = 127
        m.km[0, rows] = 1.0
        m.vm[0, rows] = 0.25
        large = rows[[0, 2, 5]]
        m.k[0, large, 0, :, 0] = 127 - 105
        m.vm[0, large] = 0.25 * ratio
    off = _offsets(counts)
    q = np.zeros((int(off[-1]), 4, 64))
    q[:, :, 0] = 60.0
    bits = to_bits(q, "bf16")
    want, tol, lse, ltol = _attend(m, from_bits(bits, "bf16").astype(np.float64), off, 1.0, 0, "bf16")
    got, gl = _run(rt, m, bits, off, "bf16", 1.0, 0, longest)
    got = from_bits(got, "bf16").astype(np.float64)
    assert (np.abs(got - want) <= tol).all(), np.abs((got - want) / tol).max()
    assert (np.abs(gl - lse) <= ltol).all()


@pytest.mark.parametrize("dtype,low,high", [("f16", 1e-6, 1e4), ("bf16", 1e-30, 1e30)])
@pytest.mark.parametrize("counts,lengths,window,longest", [
    ([160], [160], 0, None), ([90, 70], [200, 90], 0, None), ([64, 64], [100, 200], 1, None), ([1, 1], [81, 150], 1, None),
    ([6, 3], [81, 150], 1, None), ([1, 1], [81, 150], 1, MANY), ([5, 3], [150, 70], 16, MANY), ([128], [128], 16, None),
])
def test_pages_that_a_row_does_not_see(rt, dtype, low, high, counts, lengths, window, longest):
    """Small pages first and large ones after them, and the other way round:
    causality and the window hide the large ones from rows of the same tile and
    step."""
    print("hidden", dtype, counts, window, longest, flush=True)
    rng = np.random.default_rng(len(counts) + window)
    m = filled(rng, lengths, 16, 2, 64)
    for order in (1, -1):
        for s in range(len(lengths)):
            rows = m.tables[s, :m.held(s)][::order]
            m.vm[0, rows] = np.where(np.arange(len(rows)) < (len(rows) + 1) // 2, low, high)[:, None]
        _check(rt, m, rng, dtype, 4, counts, window=window, longest=longest)


@pytest.mark.parametrize("counts,window,longest", [([130, 90], 0, None), ([8, 4], 24, None), ([1, 1], 17, MANY),
                                                   ([100, 64], 20, None)])
def test_rows_do_not_depend_on_hidden_pages(rt, counts, window, longest):
    """Bit for bit: the rows before a page, and those whose window has passed
    it, with its values as they were and 10^30 times as large."""
    print("independent", counts, window, longest, flush=True)
    rng = np.random.default_rng(3)
    m = filled(rng, [250, 170], 16, 2, 64)
    off = _offsets(counts)
    bits = to_bits(rng.standard_normal((int(off[-1]), 4, 64)) * 2, "bf16")
    first = _run(rt, m, bits, off, "bf16", 0.125, window, longest)

    def hidden(s, length):  # a page amid the rows, or the last that the window has passed
        return (length - counts[s] // 2) // 16 if counts[s] > 16 else (length - counts[s] - window + 1) // 16 - 1

    for s, length in enumerate((250, 170)):
        at = hidden(s, length)
        m.vm[0, m.tables[s, at]] *= 1e30
        m.k[0, m.tables[s, at]] = 127
    second = _run(rt, m, bits, off, "bf16", 0.125, window, longest)
    compared = 0
    for s, length in enumerate((250, 170)):
        at = hidden(s, length)
        for j in range(counts[s]):
            pos = length - counts[s] + j
            if pos < 16 * at or (window and pos - window + 1 >= 16 * (at + 1)):
                compared += 1
                for a, b in zip(first, second):
                    np.testing.assert_array_equal(a[off[s] + j], b[off[s] + j])
    assert compared


@pytest.mark.parametrize("counts,longest", FORMS)
def test_values_near_the_largest_number(rt, counts, longest):
    """Sums of values of 3e38 in several parts stay finite."""
    print("largest", counts, longest, flush=True)
    rng = np.random.default_rng(8)
    m = filled(rng, [1200, 900], 32, 2, 64)
    rows = m.tables[m.tables >= 0]
    m.vm[:, rows] = 3e38
    m.v[0, rows] = np.abs(m.v[0, rows])
    m.v[0, rows, :, :3] = 127
    _check(rt, m, rng, "bf16", 4, counts, longest=longest)


@pytest.mark.parametrize("counts,longest", FORMS)
def test_pages_of_zeros(rt, counts, longest):
    """A largest value of 0 makes zeros of any codes, exactly."""
    print("zeros", counts, longest, flush=True)
    rng = np.random.default_rng(9)
    m = filled(rng, [180, 180], 16, 2, 64)
    rows = m.tables[m.tables >= 0]
    m.vm[:, rows] = 0.0
    off = _offsets(counts)
    bits = to_bits(rng.standard_normal((int(off[-1]), 4, 64)), "bf16")
    got, lse = _run(rt, m, bits, off, "bf16", 0.125, 0, longest)
    assert (from_bits(got, "bf16") == 0).all() and np.isfinite(lse).all()


@pytest.mark.parametrize("counts,longest", FORMS)
@pytest.mark.parametrize("q_scale", [1e4, 1e6, 1e8])
def test_one_key_far_above_the_others(rt, counts, longest, q_scale):
    """Scores whose f32 steps are large: the row is the one key's v."""
    print("one key", counts, longest, q_scale, flush=True)
    rng = np.random.default_rng(10)
    m = filled(rng, [300, 260], 16, 1, 64)
    top = {0: 100, 1: 40}
    for s in range(2):
        rows = m.tables[s, :m.held(s)]
        m.k[0, rows] = 0
        m.k[0, rows, 0, :, 0] = rng.integers(-127, 101, (len(rows), 16))
        m.km[0, rows] = 1.0
        m.vm[0, rows] = 10.0 ** rng.uniform(-3, 3, (len(rows), 1))
        m.k[0, rows[top[s] // 16], 0, top[s] % 16, 0] = 127
    off = _offsets(counts)
    q = np.zeros((int(off[-1]), 2, 64))
    q[:, :, 0] = q_scale
    got, _ = _run(rt, m, to_bits(q, "bf16"), off, "bf16", 1.0, 0, longest)
    got = from_bits(got, "bf16")
    for s in range(2):
        _, v = m.values(0, s)
        # p's rounding, the scale's and the result's
        want = v[top[s], 0]
        np.testing.assert_allclose(got[off[s]:off[s + 1]], np.broadcast_to(want, (counts[s], 2, 64)),
                                   rtol=2.0 ** -8 + 2.0 ** -11 + 2.0 ** -14)
