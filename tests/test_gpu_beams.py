"""The choice of the next beams: parents and tokens equal to those of 64 bits,
totals within their one rounding, 2^-24, and the sums' error.  Each term of a
sum is within 1e-10 of it but the largest, exp(0), which is exact: with p the
largest's share the sum is off by 1e-10 (1 - p) of itself at most, its logarithm
by as much, and 1 - p <= -log p, which is no more than |total| where scores are
not positive.  So 1e-10 |total|; that of f64 additions is some 1e-15."""
import numpy as np
import pytest

from cache_oracle import from_bits, to_bits
from decode_oracle import beams
from manta_amd import _lib, rocm

pytestmark = pytest.mark.gpu


def _run(rt, logits, scores, best, dtype, ended=None, end_token=0, stride=None, offset=0, handle=None):
    """logits f32 [groups, beams, vocab] -> the device's answer, checked."""
    g, b, v = logits.shape
    stride = stride or v
    bits = to_bits(logits, dtype).reshape(g * b, v)
    host = to_bits(np.full((offset + g * b * stride,), 1e4), dtype)  # (would win if it were read)
    for r in range(g * b):
        host[offset + r * stride:offset + r * stride + v] = bits[r]
    view = rocm.View(rt.to_device(host), (g, b, v), (b * stride, stride, 1), offset)
    out = [rt.to_device(np.full((g, best), -7, np.int32)) for _ in range(2)] + [rt.empty((g, best), np.float32)]
    h = handle or rt.beams(g, b, best)
    h.select(view, rt.to_device(np.asarray(scores, np.float32)), *out,
             ended=None if ended is None else rt.to_device(np.asarray(ended, np.int32)), end_token=end_token, dtype=dtype)
    parents, tokens, totals = (x.download() for x in out)
    wp, wt, ws = beams(from_bits(bits, dtype).reshape(g, b, v), np.asarray(scores, np.float32), best, ended, end_token)
    np.testing.assert_array_equal(parents, wp)
    np.testing.assert_array_equal(tokens, wt)
    live = wp >= 0
    assert np.isneginf(totals[~live]).all()
    assert (np.abs(totals[live] - ws[live]) <= np.abs(ws[live]) * (2.0 ** -24 + 1e-10) * 1.0001 + 1e-30).all()
    return parents, tokens, totals


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("groups,nb,vocab,best", [
    (1, 1, 1, 1), (1, 1, 1, 4), (3, 2, 5, 7), (2, 4, 100, 8), (1, 4, 8191, 8), (1, 4, 8192, 8), (2, 3, 8193, 6),
    (5, 8, 20000, 16), (1, 64, 300, 64), (2, 5, 70001, 10), (70, 1, 501, 2), (1, 2, 600001, 64), (4, 16, 3001, 32),
    (1000, 2, 17, 4)])
def test_sizes_and_types(rt, dtype, groups, nb, vocab, best):
    print("beams", dtype, groups, nb, vocab, best, flush=True)
    rng = np.random.default_rng(groups + nb * 10 + vocab)
    logits = (rng.standard_normal((groups, nb, vocab)) * 3).astype(np.float32)
    _run(rt, logits, -10 - 4 * rng.random((groups, nb)), best, dtype)


@pytest.mark.parametrize("dtype,stride,offset", [("f32", 1003, 1), ("f16", 1001, 3), ("bf16", 1008, 8)])
def test_rows_start_anywhere(rt, dtype, stride, offset):
    print("beams strided", dtype, stride, offset, flush=True)
    rng = np.random.default_rng(5)
    _run(rt, (rng.standard_normal((3, 4, 1000)) * 3).astype(np.float32), -rng.random((3, 4)) * 9, 8, dtype,
         stride=stride, offset=offset)


@pytest.mark.parametrize("vocab", [40, 9001])
def test_ties_go_to_the_lowest(rt, vocab):
    """Rows of equal logits, beams that are equal throughout, few distinct
    values: the lowest beam and token."""
    print("beams ties", vocab, flush=True)
    rng = np.random.default_rng(2)
    logits = np.zeros((4, 3, vocab), np.float32)
    logits[1] = 5.0
    logits[2] = rng.integers(0, 2, (1, vocab)) * 2.0  # the three beams alike
    logits[3] = rng.integers(0, 3, (3, vocab))
    scores = np.full((4, 3), -2.5, np.float32)
    for dtype in ("f32", "bf16"):
        p, t, _ = _run(rt, logits, scores, 12, dtype)
        assert (p[0] == 0).all() and (t[0] == np.arange(12)).all()
    # more equal totals than are ranked at once: 64 beams, 64 results, 20 parts a row
    many = np.zeros((1, 64, 20 * 8192), np.float32)
    p, t, _ = _run(rt, many, np.zeros((1, 64), np.float32), 64, "f16")
    assert (p == 0).all() and (t[0] == np.arange(64)).all()


def test_masks_and_what_is_not_finite(rt):
    print("beams masks", flush=True)
    rng = np.random.default_rng(3)
    logits = rng.standard_normal((8, 3, 9000)).astype(np.float32)
    scores = np.full((8, 3), -1.0, np.float32)
    logits[0, :, 5:] = -np.inf          # few tokens left: fewer than asked for
    logits[1, 1] = -np.inf              # a row that its mask leaves empty
    logits[2] = -np.inf                 # ... all of a group's
    logits[3, 0, 17] = np.nan           # no statistics: the beam is out
    logits[3, 1, 8999] = np.inf
    logits[4] = np.finfo(np.float32).min  # a mask of the type's lowest value everywhere
    logits[4, 2, 7] = 0.0
    scores[5] = [0.0, -np.inf, -np.inf]   # the first step: one live beam
    scores[6] = -np.inf
    scores[7, 0] = np.nan
    logits[7, 1].view(np.uint32)[4] = 0xFFFFFFFF  # a NaN of all ones
    want = _run(rt, logits[[0, 1, 2, 3, 4, 5, 6]], scores[:7], 18, "f32")
    assert (want[0][2] == -1).all() and (want[0][6] == -1).all() and (want[0][3] == 2).all()
    out = [rt.empty((1, 4), np.int32) for _ in range(2)] + [rt.empty((1, 4), np.float32)]
    rt.beams(1, 3, 4).select(rt.to_device(logits[7:]), rt.to_device(scores[7:]), *out)
    assert (out[0].download() == 2).all()


@pytest.mark.parametrize("vocab", [30, 20001])
def test_ended_beams(rt, vocab):
    """One continuation, their total as it was; their logits are not read."""
    print("beams ended", vocab, flush=True)
    rng = np.random.default_rng(4)
    logits = rng.standard_normal((6, 4, vocab)).astype(np.float32)
    ended = (rng.random((6, 4)) < 0.5).astype(np.int32)
    ended[0], ended[1] = 0, 1
    logits[ended != 0] = np.nan
    scores = (-3 * rng.random((6, 4))).astype(np.float32)
    scores[1, 2] = -np.inf
    p, t, s = _run(rt, logits, scores, 8, "f32", ended, 2)
    assert (p[1] >= 0).sum() == 3 and (t[1][:3] == 2).all()
    _run(rt, logits, scores, 8, "f16", ended, vocab - 1)


def test_a_handle_serves_smaller_calls_and_repeats(rt):
    """One handle, calls of other sizes after each other, scores in place."""
    print("beams handle", flush=True)
    rng = np.random.default_rng(6)
    h = rt.beams(5, 8, 16)
    for g, b, v, best in ((5, 8, 30000, 16), (1, 1, 7, 1), (2, 4, 9000, 4), (5, 8, 100, 16)):
        for _ in range(2):
            _run(rt, rng.standard_normal((g, b, v)).astype(np.float32), -rng.random((g, b)), best, "f16", handle=h)
    logits = rng.standard_normal((3, 4, 5000)).astype(np.float32)
    scores = (-rng.random((3, 4))).astype(np.float32)
    d, s = rt.to_device(logits), rt.to_device(scores)
    out = [rt.empty((3, 4), np.int32) for _ in range(2)]
    h.select(d, s, *out, s)
    wp, wt, ws = beams(logits, scores, 4)
    np.testing.assert_array_equal(out[0].download(), wp)
    np.testing.assert_array_equal(out[1].download(), wt)
    np.testing.assert_allclose(s.download(), ws, rtol=2.0 ** -23)


def test_one_beam_a_group_at_any_stride(rt):
    """The middle axis of a view has one entry: its stride says nothing."""
    rng = np.random.default_rng(12)
    logits = rng.standard_normal((5, 900)).astype(np.float32)
    whole = rt.to_device(logits)
    scores = rt.to_device(np.zeros((5, 1), np.float32))
    h = rt.beams(5, 1, 3)
    for stride in (900, 1, 7):
        out = [rt.empty((5, 3), np.int32), rt.empty((5, 3), np.int32), rt.empty((5, 3), np.float32)]
        h.select(rocm.View(whole, (5, 1, 700), (900, stride, 1), 20), scores, *out)
        parents, tokens, _ = (x.download() for x in out)
        wp, wt, _ = beams(logits[:, None, 20:720], np.zeros((5, 1), np.float32), 3)
        np.testing.assert_array_equal(parents, wp)
        np.testing.assert_array_equal(tokens, wt)


def test_in_place(rt):
    """scores and ended are the results' own memory: as many results as beams,
    or the call is refused."""
    rng = np.random.default_rng(13)
    logits, scores = rng.standard_normal((6, 4, 5000)).astype(np.float32), -rng.random((6, 4)).astype(np.float32)
    ended = (rng.random((6, 4)) < 0.3).astype(np.int32)
    want = beams(logits, scores, 4, ended, 9)
    s, e, d = rt.to_device(scores), rt.to_device(ended), rt.to_device(logits)
    p, t = rt.empty((6, 4), np.int32), rt.empty((6, 4), np.int32)
    h = rt.beams(6, 4, 8)
    h.select(d, s, p, t, s, ended=e, end_token=9, out_ended=e)
    np.testing.assert_array_equal(p.download(), want[0])
    np.testing.assert_array_equal(t.download(), want[1])
    np.testing.assert_array_equal(e.download(), want[1] == 9)
    assert (np.abs(s.download() - want[2]) <= np.abs(want[2]) * (2.0 ** -24 + 1e-10) * 1.0001).all()
    other = rt.empty((24,), np.float32)
    for totals, now in ((s.addr, None), (other.addr, e.addr)):
        with pytest.raises(_lib.MantaRocmError, match="in place"):
            _lib.call("manta_rocm_beam_select", rt.handle, h.handle, 32, d.addr, 5000, 6, 4, 5000, s.addr, e.addr, 9, 3,
                      p.addr, t.addr, totals, now)
    np.testing.assert_array_equal(t.download(), want[1])
