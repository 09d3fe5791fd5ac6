"""Attention over the 8-bit cache against softmax in 64 bits on the values the
codes stand for.  The bounds (Model.attend) count the roundings: f32 scores,
p and v as f16 operands of f32 sums, and the result's type."""
import numpy as np
import pytest

from cache_oracle import EPS, filled, from_bits, to_bits
from manta_amd import _lib, rocm

pytestmark = pytest.mark.gpu


def _dev(rt, x):
    return rt.to_device(np.asarray(x, np.int32))


def _offsets(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)


def _check(rt, m, rng, dtype, heads, counts, seqs=None, scale=None, causal=True, window=0, longest=None, layer=0,
           q_scale=2.0, extra_rows=0):
    off = _offsets(counts)
    t = int(off[-1]) + extra_rows
    bits = to_bits(rng.standard_normal((t, heads, m.d)) * q_scale, dtype)
    q = from_bits(bits, dtype).astype(np.float64)
    scale = m.d ** -0.5 if scale is None else scale
    want, lse, err, lerr = m.attend(layer, q, off, seqs, scale, causal, window)
    c = m.upload(rt)
    out = rt.to_device(np.full((t, heads, m.d), 0x5555, np.uint16))
    ld = rt.to_device(np.full((t, heads), 77.0, np.float32))
    c.attention(layer, rt.to_device(bits), _dev(rt, off), None if seqs is None else _dev(rt, seqs), out=out, lse=ld,
                scale=scale, causal=causal, window=window, longest=longest, dtype=dtype)
    got, gl = from_bits(out.download(), dtype).astype(np.float64), ld.download()
    n = int(off[-1])
    tol = err + np.abs(want) * EPS[dtype] + (2.0 ** -25 if dtype == "f16" else 0)
    bad = ~(np.abs(got - want)[:n] <= tol[:n])
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:5], got[:n][bad][:5], want[:n][bad][:5], tol[:n][bad][:5])
    none = np.isneginf(lse[:n])
    np.testing.assert_array_equal(np.isneginf(gl[:n]), none)
    assert (np.abs(gl[:n] - lse[:n])[~none] <= lerr[:n][~none]).all()
    if extra_rows:  # rows no sequence owns are not written
        assert (out.download()[n:] == 0x5555).all() and (gl[n:] == 77.0).all()
    # the same call again, and without lse: the same bits
    first = out.download()
    c.attention(layer, rt.to_device(bits), _dev(rt, off), None if seqs is None else _dev(rt, seqs), out=out,
                scale=scale, causal=causal, window=window, longest=longest, dtype=dtype)
    np.testing.assert_array_equal(out.download(), first)
    c.close()


STEPS = [
    # page, kv heads, group, d, lengths
    (16, 1, 1, 32, [1]), (16, 6, 1, 64, [1, 2, 15, 16, 17, 33, 63, 64, 65]), (32, 2, 4, 128, [300, 1, 77, 129]),
    (64, 8, 4, 128, [1000, 64, 128, 129]), (128, 1, 8, 256, [500, 127, 128]), (16, 2, 5, 80, [40, 200]),
    (64, 1, 16, 96, [333]), (32, 1, 17, 64, [95, 1]), (16, 3, 2, 33, [50, 49]), (64, 2, 40, 192, [200]),
    (128, 4, 3, 1, [130]), (64, 2, 4, 128, [5000]), (16, 1, 2, 160, [2500, 7]), (32, 1, 1, 224, [100]),
]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("page,kv,group,d,lengths", STEPS)
def test_single_tokens(rt, dtype, page, kv, group, d, lengths):
    print("attend step", dtype, page, kv, group, d, lengths, flush=True)
    rng = np.random.default_rng(page + d + group)
    m = filled(rng, lengths, page, kv, d)
    _check(rt, m, rng, dtype, kv * group, [1] * len(lengths), longest=max(lengths))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("page,kv,group,d,lengths,counts,window", [
    (16, 2, 2, 64, [40, 20, 5], [5, 20, 3], 0), (64, 1, 8, 128, [500, 70], [7, 70], 0),
    (32, 2, 6, 96, [400, 33], [5, 6], 100), (16, 1, 1, 32, [130], [130], 0), (64, 2, 4, 128, [300, 200], [260, 129], 0),
    (128, 1, 2, 256, [150], [90], 0), (32, 1, 3, 80, [222, 10], [200, 10], 17), (16, 2, 1, 40, [90], [64], 1),
    (64, 1, 4, 128, [700], [300], 64), (16, 1, 4, 192, [100, 5], [40, 5], 0), (64, 1, 12, 64, [420], [333], 0),
    (32, 1, 1, 160, [200], [150], 33), (128, 2, 5, 224, [140], [70], 0), (64, 1, 16, 16, [250], [180], 0),
])
def test_many_tokens(rt, dtype, page, kv, group, d, lengths, counts, window):
    print("attend tokens", dtype, page, kv, group, d, lengths, counts, window, flush=True)
    rng = np.random.default_rng(page + d + group)
    m = filled(rng, lengths, page, kv, d)
    _check(rt, m, rng, dtype, kv * group, counts, window=window)


@pytest.mark.parametrize("counts", [[1, 1, 1, 1], [4, 1, 30, 2], [70, 130, 64, 80]])
@pytest.mark.parametrize("causal", [True, False])
def test_rows_that_see_nothing(rt, counts, causal):
    """Sequences of length 0, more rows than tokens (the first of them before
    position 0), rows that no sequence owns."""
    print("attend nothing", counts, causal, flush=True)
    rng = np.random.default_rng(1)
    m = filled(rng, [0, 1, 20, 66], 16, 2, 64)
    _check(rt, m, rng, "f16", 4, counts, causal=causal, extra_rows=3)


@pytest.mark.parametrize("counts", [[1, 2], [40, 70]])
def test_all_tokens_seen(rt, counts):
    print("attend all", counts, flush=True)
    rng = np.random.default_rng(2)
    m = filled(rng, [300, 90], 32, 2, 64)
    _check(rt, m, rng, "bf16", 8, counts, causal=False)


@pytest.mark.parametrize("count", [1, 100])
def test_listed_sequences_second_layer(rt, count):
    print("attend listed", count, flush=True)
    rng = np.random.default_rng(3)
    m = filled(rng, [100, 40, 7, 300, 120], 16, 2, 64, layers=3)
    _check(rt, m, rng, "f16", 4, [count, count, count], seqs=[3, 0, 4], layer=2)


@pytest.mark.parametrize("count,window", [(1, 0), (3, 9), (120, 0), (120, 50)])
def test_shared_pages(rt, count, window):
    """Branches of one prefix read the same pages."""
    print("attend shared", count, window, flush=True)
    rng = np.random.default_rng(4)
    m = filled(rng, [150, 0, 0], 64, 1, 128)
    m.fork([0, 0], [1, 2], [150, 137])
    _check(rt, m, rng, "bf16", 4, [count] * 3, window=window)


@pytest.mark.parametrize("count", [1, 80])
@pytest.mark.parametrize("longest", [1, 100, 1 << 20])
def test_any_longest(rt, count, longest):
    """longest sets how the work is split, not what is computed."""
    print("attend longest", count, longest, flush=True)
    rng = np.random.default_rng(5)
    m = filled(rng, [3000, 90], 64, 1, 64)
    _check(rt, m, rng, "f16", 2, [count, count], longest=longest)


@pytest.mark.parametrize("count", [1, 20, 90])
@pytest.mark.parametrize("q_scale,scale", [(0.0, None), (1e-3, None), (300.0, 1.0), (30.0, -0.5), (1e-6, 1.0)])
def test_flat_peaked_and_tiny_scores(rt, count, q_scale, scale):
    print("attend scores", count, q_scale, scale, flush=True)
    rng = np.random.default_rng(6)
    m = filled(rng, [260, 120], 32, 1, 64)
    for dtype in ("f16", "bf16"):
        _check(rt, m, rng, dtype, 2, [count, count], q_scale=q_scale, scale=scale)


@pytest.mark.parametrize("count", [1, 5, 100])
def test_page_scales_far_apart(rt, count):
    """Pages whose largest values differ by powers of ten, and pages of zeros:
    each keeps its weight in the sums."""
    print("attend scales", count, flush=True)
    rng = np.random.default_rng(7)
    m = filled(rng, [400, 170], 16, 2, 64)
    m.vm[:] = np.where(np.isfinite(m.vm), 10.0 ** rng.uniform(-6, 4, m.vm.shape), m.vm)
    m.km[:] = np.where(np.isfinite(m.km), rng.choice([0.0, 0.5, 3.0], m.km.shape), m.km)
    m.vm[0, m.tables[0, 3:9]] = 0.0
    m.vm[0, m.tables[1, 0]] = 0.0
    _check(rt, m, rng, "f16", 4, [count, count])


@pytest.mark.parametrize("count", [1, 60])
def test_far_magnitudes(rt, count):
    """bf16 queries, keys and values far outside f16's range."""
    print("attend far", count, flush=True)
    rng = np.random.default_rng(8)
    m = filled(rng, [200, 64], 64, 1, 64)
    live = np.isfinite(m.km) & (m.km < 1e29)
    m.km[live] *= 1e-12
    m.vm[live] *= 1e20
    _check(rt, m, rng, "bf16", 4, [count, count], q_scale=1e12)
    m.km[live] *= 1e30
    m.vm[live] *= 1e-35
    _check(rt, m, rng, "bf16", 4, [count, count], q_scale=1e-18)


@pytest.mark.parametrize("count,window", [(1, 0), (70, 0), (70, 20), (3, 16)])
def test_values_that_are_not_finite(rt, count, window):
    """A page's head whose largest value is NaN makes NaN of the rows that see
    it, and of no others."""
    print("attend nan", count, window, flush=True)
    rng = np.random.default_rng(9)
    lengths = [200, 130]
    m = filled(rng, lengths, 32, 2, 64)
    m.km[0, m.tables[0, 4], 1] = np.nan  # tokens 128..159, kv head 1
    m.vm[0, m.tables[1, 2], 0] = np.nan  # tokens 64..95, kv head 0
    c = m.upload(rt)
    off = _offsets([count, count])
    bits = to_bits(rng.standard_normal((2 * count, 4, 64)), "f16")
    out, lse = rt.empty(bits.shape, np.uint16), rt.empty(bits.shape[:2], np.float32)
    c.attention(0, rt.to_device(bits), _dev(rt, off), out=out, lse=lse, window=window)
    got = from_bits(out.download(), "f16")
    nan = np.isnan(got)
    assert (nan.all(-1) == nan.any(-1)).all()
    nan = nan.any(-1)
    for i, (n, a, b, head) in enumerate(((200, 128, 160, 1), (130, 64, 96, 0))):
        for j in range(count):
            pos = n - count + j
            sees = pos >= a and (not window or pos - window + 1 < b)
            for h in range(4):
                assert nan[off[i] + j, h] == (sees and h // 2 == head), (i, j, h)
    c.close()


def test_strided_queries_in_place(rt):
    print("attend strided", flush=True)
    rng = np.random.default_rng(10)
    m = filled(rng, [90, 40], 16, 2, 48)
    c = m.upload(rt)
    for counts, width, offset in (([1, 1], 4 * 48 + 3, 1), ([1, 1], 4 * 48 + 8, 8), ([60, 33], 4 * 48 + 3, 1),
                                  ([60, 33], 4 * 48 + 8, 8)):
        off = _offsets(counts)
        t = int(off[-1])
        bits = to_bits(rng.standard_normal((t, width)), "f16")
        a = rt.to_device(bits)
        v = rocm.View(a, (t, 4, 48), (width, 48, 1), offset)
        c.attention(0, v, _dev(rt, off), out=v)
        q = from_bits(bits, "f16").astype(np.float64)[:, offset:offset + 192].reshape(t, 4, 48)
        want, _, err, _ = m.attend(0, q, off, None, 48 ** -0.5, True, 0)
        got = a.download()
        keep = np.ones(width, bool)
        keep[offset:offset + 192] = False
        np.testing.assert_array_equal(got[:, keep], bits[:, keep])
        got = from_bits(got, "f16").astype(np.float64)[:, offset:offset + 192].reshape(t, 4, 48)
        assert (np.abs(got - want) <= err + np.abs(want) * 2.0 ** -11 + 2.0 ** -25).all()
        # heads before tokens
        h = rt.to_device(np.ascontiguousarray(bits[:, offset:offset + 192].reshape(t, 4, 48).transpose(1, 0, 2)))
        o = rt.empty((t, 4, 48), np.uint16)
        c.attention(0, rocm.View(h, (t, 4, 48), (48, t * 48, 1)), _dev(rt, off), out=o)
        np.testing.assert_array_equal(from_bits(o.download(), "f16"), got)
    c.close()


def test_refusals(rt):
    print("attend refusals", flush=True)
    rng = np.random.default_rng(11)
    m = filled(rng, [90, 40], 16, 2, 64)
    c = m.upload(rt)
    q = rt.to_device(to_bits(rng.standard_normal((2, 4, 64)), "f16"))
    off = _dev(rt, [0, 1, 2])
    for f, error, text in (
            (lambda: c.attention(1, q, off), _lib.MantaRocmError, "layer 1"),
            (lambda: c.attention(0, rt.empty((2, 3, 64), np.uint16), off), _lib.MantaRocmError, "3 query heads"),
            (lambda: c.attention(0, rt.empty((2, 4, 64), np.float32), off), _lib.Unsupported, "f16 or bf16"),
            (lambda: c.attention(0, q, off, causal=False, window=5), _lib.MantaRocmError, "window"),
            (lambda: c.attention(0, q, off, window=-1), _lib.MantaRocmError, "window"),
            (lambda: c.attention(0, q, off, scale=float("nan")), _lib.MantaRocmError, "scale"),
            (lambda: c.attention(0, q, off, longest=-2), _lib.MantaRocmError, "length"),
            (lambda: c.attention(0, rt.empty((2, 4, 32), np.uint16), off), ValueError, "q must be"),
            (lambda: c.attention(0, q, off, out=rt.empty((2, 4, 32), np.uint16)), ValueError, "out must be"),
            (lambda: c.attention(0, q, off, lse=rt.empty((2, 2), np.float32)), ValueError, "lse must be"),
            (lambda: c.attention(0, q, off, dtype="f32"), TypeError, "does not hold")):
        with pytest.raises(error, match=text):
            f()
    # the device's findings: the call ends, the row of the bad sequence is zeros
    out = c.attention(0, q, off, _dev(rt, [0, 5]))
    with pytest.raises(_lib.MantaRocmError, match="sequence 5 out of range"):
        rt.synchronize()
    assert (out.download()[1] == 0).all()
    m.tables[1, 1] = m.pages
    c.book.upload(m.book())
    c.attention(0, q, off)
    with pytest.raises(_lib.MantaRocmError, match="page %d out of range" % m.pages):
        rt.synchronize()
    rt.synchronize()
    c.close()
