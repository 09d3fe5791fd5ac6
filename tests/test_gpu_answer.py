"""The decoding calls used together: an answerer whose every call is checked
against the operator's own oracle on the data that the device had, its steps in
a HIP graph, and the answers that come back."""
import ctypes as C

import numpy as np
import pytest

from cache_oracle import EPS, from_bits
from decode_oracle import beams, product, quantise, rotary_normed, rounding
from manta_amd import _lib, rocm
from manta_amd.answer import Answerer, random_model

pytestmark = pytest.mark.gpu


def _host(a):
    """A device array's or view's values."""
    if isinstance(a, rocm.View):
        flat = a.array.download().reshape(-1)
        at = (a.addr - a.array.addr) // a.dtype.itemsize
        for n, s in zip(a.shape, a.strides):
            at = np.asarray(at)[..., None] + np.arange(n) * s
        flat = flat[at]
    else:
        flat = a.download()
    return from_bits(flat, "f16") if flat.dtype == np.uint16 else flat


class Checked:
    """A runtime that checks the calls that pass through it."""

    def __init__(self, rt):
        self.rt, self.weights, self.checked = rt, {}, []

    def __getattr__(self, name):
        return getattr(self.rt, name)

    def weight(self, codes, scales, gate=None):
        w = self.rt.weight(codes, scales, gate=gate)
        self.weights[id(w)] = (codes, scales)
        return w

    def quantize_rows(self, x, out=None, norm=None, eps=1e-6, dtype=None):
        host = _host(x)
        out = self.rt.quantize_rows(x, out, norm=norm, eps=eps, dtype=dtype)
        codes, scales = out.values()
        want, want_scales = quantise(host, None if norm is None else norm.download(), eps)
        np.testing.assert_array_equal(codes, want)
        np.testing.assert_allclose(scales, want_scales, rtol=2.0 ** -23)
        self.checked.append("quantize")
        return out

    def matmul_q8(self, w, x, out=None, add=None, dtype=None):
        base = None if add is None else _host(add)
        out = self.rt.matmul_q8(w, x, out=out, add=add, dtype=dtype)
        codes, scales = x.values()
        kind = "f32" if out.dtype == np.float32 else "f16"
        want, tol = product(codes, scales.astype(np.float64), *self.weights[id(w)], kind, base, w.gate)
        assert (np.abs(_host(out) - want) <= tol).all()
        self.checked.append("matmul")
        return out

    def rotary_normed(self, rot, positions, parts, norms, eps=1e-6, dtype=None):
        before = [_host(x) for x, _ in parts]
        self.rt.rotary_normed(rot, positions, parts, norms, eps=eps, dtype=dtype)
        freqs = rocm.rotary_freqs(rot.rot)
        for x, w, (_, out) in zip(before, norms, parts):
            want, off = rotary_normed(x, w.download(), eps, positions.download(), freqs, "half", 1.0)
            assert (np.abs(_host(out) - want) <= off + rounding(np.abs(want) + off, "f16")).all()
        self.checked.append("rotary")

    def beams(self, *args):
        choice, checked = self.rt.beams(*args), self.checked

        class Choice:
            def close(self):
                choice.close()

            def select(self, logits, scores, parents, tokens, totals, ended=None, end_token=0, out_ended=None):
                l, s, e = logits.download(), scores.download(), None if ended is None else ended.download()
                choice.select(logits, scores, parents, tokens, totals, ended=ended, end_token=end_token,
                              out_ended=out_ended)
                p, t, v = beams(l, s, parents.shape[1], e, end_token)
                np.testing.assert_array_equal(parents.download(), p)
                np.testing.assert_array_equal(tokens.download(), t)
                np.testing.assert_allclose(totals.download(), v, rtol=2.0 ** -23)
                np.testing.assert_array_equal(out_ended.download(), (t == end_token).astype(np.int32))
                checked.append("beams")

        return Choice()


def _check_attention(a, lengths):
    """The last layer's outputs of a step against softmax in 64 bits over what
    the cache holds."""
    m, layer = a.model, len(a.model.blocks) - 1
    n = a.questions * a.beams
    q, got = _host(a.rows.q).astype(np.float64), _host(a.rows.attended)
    for s in range(n):
        k, v = (a.rt.empty((lengths[s], m.kv_heads, m.head_dim), np.float32) for _ in range(2))
        a.cache.read(layer, a._ints([0, lengths[s]]), k, v, a._ints([s]))
        k, v = k.download().astype(np.float64), v.download().astype(np.float64)
        for h in range(m.q_heads):
            kk, vv = k[:, h * m.kv_heads // m.q_heads], v[:, h * m.kv_heads // m.q_heads]
            z = kk @ q[s, h] / np.sqrt(m.head_dim)
            w = np.exp(z - z.max())
            w /= w.sum()
            # scores and weights in f32, the second product's operands once in f16, the result once
            tol = (w @ np.abs(vv)) * (4 * 2.0 ** -11) + 2.0 ** -25 * lengths[s] * np.abs(vv).max()
            assert (np.abs(got[s, h] - w @ vv) <= tol + EPS["f16"] * np.abs(w @ vv)).all()


@pytest.mark.parametrize("q_heads,kv_heads,d,nb,page", [(4, 2, 64, 4, 16), (3, 3, 32, 3, 32), (2, 1, 80, 1, 16)])
def test_every_call_of_an_answer(rt, q_heads, kv_heads, d, nb, page):
    print("answer", q_heads, kv_heads, d, nb, page, flush=True)
    rng = np.random.default_rng(d)
    checked = Checked(rt)
    m = random_model(checked, rng, 2, 300, 144, q_heads, kv_heads, d, 200)
    a = Answerer(checked, m, 2, nb, 70, end_token=2, page_tokens=page)
    questions = [rng.integers(3, 300, n).tolist() for n in (37, 5)]
    a.ask(questions)
    lengths = np.repeat([37, 5], nb)
    for _ in range(6):
        refs, held, tables = a.cache.tables()
        np.testing.assert_array_equal(held, lengths)
        before = tables.copy()
        a.step()
        lengths = lengths + 1
        refs, held, tables = a.cache.tables()
        np.testing.assert_array_equal(held, lengths)
        # references are those of the tables
        np.testing.assert_array_equal(refs, np.bincount(tables[tables >= 0], minlength=len(refs)))
        # a beam holds what its parent held; whole pages of it are shared, not copied
        parents = a.parents.download()
        for g in range(2):
            for b in range(nb):
                source = g * nb + parents[g, b]
                whole = (lengths[g * nb + b] - 1) // page
                np.testing.assert_array_equal(tables[g * nb + b, :whole], before[source, :whole])
    if nb == 1:
        _check_attention(a, lengths)
    assert {"quantize", "matmul", "rotary", "beams"} <= set(checked.checked)
    a.close()
    m.close()


def test_attention_of_the_beams(rt):
    """Before the reorder, sequences are the rows: the choice that keeps every
    beam where it is."""
    print("answer attention", flush=True)
    rng = np.random.default_rng(5)
    m = random_model(rt, rng, 1, 300, 128, 4, 2, 64, 128)
    a = Answerer(rt, m, 2, 3, 64, end_token=2)
    a.ask([rng.integers(3, 300, n).tolist() for n in (20, 9)])
    a.cache.reorder = lambda *args: None
    for _ in range(3):
        a.step()
    _check_attention(a, [23] * 3 + [12] * 3)
    a.close()
    m.close()


def test_beams_and_their_scores(rt):
    """Beams come best first, no two alike; what does not fit is refused."""
    print("answer beams", flush=True)
    rng = np.random.default_rng(9)
    m = random_model(rt, rng, 1, 200, 128, 2, 2, 64, 128)
    question = [rng.integers(3, 200, 12).tolist()]
    found = {}
    for nb in (1, 6):
        a = Answerer(rt, m, 1, nb, 64, end_token=2)
        found[nb] = a.answer(question, 8)[0]
        a.close()
    assert len(found[1]) == 1 and len(found[6]) == 6
    scores = [s for _, s in found[6]]
    assert scores == sorted(scores, reverse=True)
    assert len({tuple(t) for t, _ in found[6]}) == 6  # no two alike
    with pytest.raises(ValueError, match="more than 64"):
        b = Answerer(rt, m, 1, 2, 64, end_token=2)
        b.answer(question, 60)
    with pytest.raises(ValueError, match="1 questions"):
        b.ask(question * 2)
    b.close()
    m.close()


def test_steps_in_a_graph():
    """A step captured once and replayed, with other work between the replays:
    the same choices, scores and book, bit for bit, as the calls one by one."""
    print("answer graph", flush=True)
    hip = _lib.load()

    def ok(name, *args):
        assert getattr(hip, name)(*args) == 0, name

    with rocm.Runtime(0) as rt:
        stream = C.c_void_p()
        ok("hipStreamCreate", C.byref(stream))
        rt.set_stream(stream.value)
        results = []
        for captured in (False, True):
            rng = np.random.default_rng(21)
            m = random_model(rt, rng, 2, 500, 128, 4, 2, 32, 256)
            a = Answerer(rt, m, 3, 4, 64, end_token=2)
            a.ask([rng.integers(3, 500, n).tolist() for n in (30, 7, 15)])
            graph, run = C.c_void_p(), C.c_void_p()
            if captured:
                rt.synchronize()
                ok("hipStreamBeginCapture", stream, 2)  # relaxed
                a.step()
                ok("hipStreamEndCapture", stream, C.byref(graph))
                ok("hipGraphInstantiate", C.byref(run), graph, None, None, C.c_size_t(0))
            other = rt.empty((64, 128), np.float32)
            steps = []
            for _ in range(7):
                if captured:
                    ok("hipGraphLaunch", run, stream)
                else:
                    a.step()
                rt.normalize_rows(other.upload(rng.standard_normal((64, 128)).astype(np.float32)))
                steps.append([a.parents.download(), a.next.download(), a.scores.download(), a.logits.download(),
                              a.cache.book.download()])
            results.append(steps)
            if captured:
                ok("hipGraphExecDestroy", run)
                ok("hipGraphDestroy", graph)
            a.close()
            m.close()
        for one, two in zip(*results):
            for x, y in zip(one, two):
                np.testing.assert_array_equal(x, y)
        rt.set_stream(0)
        ok("hipStreamDestroy", stream)
