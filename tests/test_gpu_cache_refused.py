"""What a refused extend, or an append to a shared page, leaves of the cache:
all of it, bit for bit, until the refusal has been reported."""
import ctypes as C

import numpy as np
import pytest

from cache_oracle import filled, from_bits, to_bits
from manta_amd import _lib, rocm

pytestmark = pytest.mark.gpu


def _dev(rt, x):
    return rt.to_device(np.asarray(x, np.int32))


def _contents(c):
    return [p.download() for p in (c.k_codes, c.v_codes, c.k_max, c.v_max, c.book)]


def _same(a, b):
    for x, y in zip(a, b):
        np.testing.assert_array_equal(x, y)


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("why", ["pages", "entry"])
def test_appends_after_a_refused_extend(rt, new, why):
    """A step of two sequences that is refused, its appends to both layers, and
    another step of them: nothing changes.  A third sequence, extended by a
    call of its own, is written.  After the report and a release the step goes
    through."""
    print("refused", new, why, flush=True)
    rng = np.random.default_rng(new)
    heads, d, page = 2, 64, 16
    m = filled(rng, [30, 45, 33, 60], page, heads, d, layers=2, extra_pages=3, dirty=False)
    m.table_pages += 6
    m.tables = np.concatenate([m.tables, np.full((4, 6), -1, np.int32)], 1)
    c = m.upload(rt)
    seqs, off = _dev(rt, [1, 0]), _dev(rt, [0, new, 2 * new])
    x = [to_bits(rng.standard_normal((2 * new, heads, d)) * 3, "f16") for _ in range(2)]
    k, v = (rt.to_device(y) for y in x)
    # too few pages (the third sequence gets them first), or a count that does not fit
    first = [3 * page] if why == "pages" else [2]
    counts = [new, new] if why == "pages" else [new, 10 ** 6]
    if why == "pages" and new == 1:
        counts = [3 + page, 2 + page]  # (a page each; the appends are the single token's)
    assert m.extend([2], first)
    c.extend(_dev(rt, [2]), _dev(rt, first))
    before = _contents(c)
    c.extend(seqs, _dev(rt, counts))
    for layer in (0, 1):
        c.append(layer, k, v, off, seqs)
    c.extend(seqs, _dev(rt, [0, 0]))  # refused with the first
    c.append(1, k, v, off, seqs)
    y = to_bits(rng.standard_normal((2, heads, d)), "f16")
    yd = rt.to_device(y)
    with pytest.raises(_lib.MantaRocmError, match="out of pages" if why == "pages" else "count 1000000"):
        rt.synchronize()
    _same(_contents(c), before)
    rt.synchronize()
    # the same, with a sequence that was extended among those appended
    c.extend(seqs, _dev(rt, counts))
    c.append(0, yd, yd, _dev(rt, [0, 1, 2]), _dev(rt, [2, 0]))
    with pytest.raises(_lib.MantaRocmError):
        rt.synchronize()
    m.append(0, from_bits(y[:1], "f16"), from_bits(y[:1], "f16"), [0, 1], [2])
    m.check_book(c)
    m.check_pages(c)
    # and now there is room
    c.release(_dev(rt, [3, 2]))
    m.release([3, 2])
    assert m.extend([1, 0], [new, new])
    c.extend(seqs, _dev(rt, [new, new]))
    for layer in (0, 1):
        c.append(layer, k, v, off, seqs)
        m.append(layer, from_bits(x[0], "f16"), from_bits(x[1], "f16"), [0, new, 2 * new], [1, 0])
    rt.synchronize()
    m.check_book(c)
    m.check_pages(c)
    c.close()


@pytest.mark.parametrize("tokens", [1, 30])
def test_append_leaves_shared_pages(rt, tokens):
    """Last tokens that a branch shares are not written over; the same rows of a
    sequence whose pages are its own are."""
    print("shared", tokens, flush=True)
    rng = np.random.default_rng(tokens)
    m = filled(rng, [40, 40, 0], 16, 2, 64, dirty=False)
    m.fork([0], [2])
    c = m.upload(rt)
    before = _contents(c)
    x = to_bits(rng.standard_normal((2 * tokens, 2, 64)) * 9, "bf16")
    xd = rt.to_device(x)
    for s in (0, 2):
        c.append(0, xd, xd, _dev(rt, [0, tokens]), _dev(rt, [s]), dtype="bf16")
        with pytest.raises(_lib.MantaRocmError, match="is shared"):
            rt.synchronize()
        _same(_contents(c), before)
    c.append(0, xd, xd, _dev(rt, [0, tokens, 2 * tokens]), _dev(rt, [0, 1]), dtype="bf16")
    with pytest.raises(_lib.MantaRocmError, match="is shared"):
        rt.synchronize()
    y = from_bits(x, "bf16")[tokens:]
    m.append(0, y, y, [0, tokens], [1])
    m.check_pages(c)
    m.check_book(c)
    c.close()


def test_another_cache_goes_on(rt):
    """A refusal in one cache does not touch another of the same runtime."""
    print("refused, two caches", flush=True)
    rng = np.random.default_rng(9)
    a, b = (filled(rng, [16], 16, 1, 32, extra_pages=e, dirty=False) for e in (0, 2))
    ca, cb = a.upload(rt), b.upload(rt)
    one, off = _dev(rt, [1]), _dev(rt, [0, 1])
    x = rng.standard_normal((1, 1, 32)).astype(np.float32)
    xd = rt.to_device(x)
    for c in (ca, cb):
        c.extend(_dev(rt, [0]), one)
        c.append(0, xd, xd, off)
    with pytest.raises(_lib.MantaRocmError, match="1 needed, 0 free"):
        rt.synchronize()
    assert b.extend([0], [1])
    b.append(0, x, x, [0, 1])
    for m, c in ((a, ca), (b, cb)):
        m.check_book(c)
        m.check_pages(c)
        c.close()


def test_replays_of_a_step_that_runs_out_of_pages():
    """extend and append captured; the pages last for three of six replays.
    What the cache held after the third is there after the sixth."""
    print("refused, graph", flush=True)
    hip = _lib.load()

    def ok(name, *args):
        assert getattr(hip, name)(*args) == 0, name

    rng = np.random.default_rng(31)
    n, kv, d = 2, 2, 64
    with rocm.Runtime(0) as rt:
        stream = C.c_void_p()
        ok("hipStreamCreate", C.byref(stream))
        rt.set_stream(stream.value)
        m = filled(rng, [13, 29], 16, kv, d, layers=2, extra_pages=0, dirty=False)
        m.table_pages += 2
        m.tables = np.concatenate([m.tables, np.full((n, 2), -1, np.int32)], 1)
        c = m.upload(rt)
        seqs, ones, off = _dev(rt, [0, 1]), _dev(rt, [1, 1]), _dev(rt, [0, 1, 2])
        k, v = (rt.empty((n, kv, d), np.uint16) for _ in range(2))
        graph, run = C.c_void_p(), C.c_void_p()
        rt.synchronize()
        ok("hipStreamBeginCapture", stream, 2)  # relaxed
        c.extend(seqs, ones)
        for layer in (0, 1):
            c.append(layer, k, v, off)
        ok("hipStreamEndCapture", stream, C.byref(graph))
        ok("hipGraphInstantiate", C.byref(run), graph, None, None, C.c_size_t(0))

        def replay():
            x = [to_bits(rng.standard_normal((n, kv, d)), "f16") for _ in range(2)]
            k.upload(x[0])
            v.upload(x[1])
            ok("hipGraphLaunch", run, stream)
            return [from_bits(y, "f16") for y in x]

        for step in range(3):
            x = replay()
            rt.synchronize()
            assert m.extend([0, 1], [1, 1])
            for layer in (0, 1):
                m.append(layer, x[0], x[1], [0, 1, 2])
        m.check_book(c)
        m.check_pages(c)
        for step in range(3):
            replay()
            ok("hipStreamSynchronize", stream)
        with pytest.raises(_lib.MantaRocmError, match="2 needed, 0 free"):
            rt.synchronize()
        m.check_book(c)
        m.check_pages(c)
        # room for both after all: the same graph goes on
        m.release([0], [5])
        c.release(_dev(rt, [0]), _dev(rt, [5]))
        m.release([1], [20])
        c.release(_dev(rt, [1]), _dev(rt, [20]))
        x = replay()
        rt.synchronize()
        assert m.extend([0, 1], [1, 1])
        for layer in (0, 1):
            m.append(layer, x[0], x[1], [0, 1, 2])
        m.check_book(c)
        m.check_pages(c)
        ok("hipGraphExecDestroy", run)
        ok("hipGraphDestroy", graph)
        c.close()
        rt.synchronize()
        rt.set_stream(0)
        ok("hipStreamDestroy", stream)
