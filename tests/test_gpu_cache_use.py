"""The rotary and cache calls used together: a reader of branches against a
recomputation from what its cache holds, decoding captured into a HIP graph,
batches of more sequences than a wave has lanes, and caches past 2^31 bytes."""

import ctypes as C

import numpy as np
import pytest

from cache_oracle import filled, from_bits, rotate, to_bits
from manta_amd import _lib, rocm
from manta_amd.reader import PassageReader, random_layers

pytestmark = pytest.mark.gpu


def _dev(rt, x):
    return rt.to_device(np.asarray(x, np.int32))


def _offsets(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)


@pytest.mark.parametrize("q_heads,kv_heads,d,page", [(4, 2, 64, 16), (6, 6, 32, 64)])
def test_reader_reads_its_cache(rt, q_heads, kv_heads, d, page):
    """One layer: the states that the reader returns against softmax in 64 bits
    over the keys and values that its branches hold."""
    print("reader", q_heads, kv_heads, d, page, flush=True)
    rng = np.random.default_rng(d)
    width = 48
    layers = random_layers(rng, 1, width, q_heads, kv_heads, d)
    question = rng.standard_normal((21, width)).astype(np.float32)
    passages = [rng.standard_normal((n, width)).astype(np.float32) for n in (1, 17, 70, 5)]
    label = rng.standard_normal(width).astype(np.float32)
    reader = PassageReader(rt, layers, q_heads, kv_heads, d, 4, 128, page)
    got = reader.read(question, passages, [label, label])
    freqs = rocm.rotary_freqs(d)
    for i, p in enumerate(passages):
        n = len(question) + len(p) + 2
        assert reader.lengths[1 + i] == n
        k, v = (rt.empty((n, kv_heads, d), np.float32) for _ in range(2))
        reader.cache.read(0, _dev(rt, [0, n]), k, v, _dev(rt, [1 + i]))
        k, v = k.download().astype(np.float64), v.download().astype(np.float64)
        # the codes are those of the tokens' own keys and values: half a step
        # when written, and half a step more for each later token of the page
        # that raised its largest value; 128 tokens' worth is not reached
        plain = np.concatenate([question, p, [label, label]])
        step = np.abs(plain @ layers[0].v).max() / 127
        assert np.abs(v - (plain @ layers[0].v).reshape(n, kv_heads, d)).max() <= 8 * step
        q = (label @ layers[0].q).reshape(1, q_heads, d)
        q = rotate(q.astype(np.float16), [n - 1], freqs, "half")[0]
        want, tol = np.zeros(q_heads * d), np.zeros(q_heads * d)
        for h in range(q_heads):
            kk, vv = k[:, h * kv_heads // q_heads], v[:, h * kv_heads // q_heads]
            s = kk @ q[h] / np.sqrt(d)
            w = np.exp(s - s.max())
            w /= w.sum()
            # q is f16 twice (the product's sum in f32 may round to its neighbour) and the
            # operands of the second product once each
            delta = (np.abs(kk) @ np.abs(q[h])).max() / np.sqrt(d) * 4 * 2.0 ** -11
            want[h * d:(h + 1) * d] = w @ vv
            tol[h * d:(h + 1) * d] = (w @ np.abs(vv)) * (2 * delta + 6 * 2.0 ** -11) + 1e-6
        err = tol @ np.abs(layers[0].o) + 1e-5
        assert (np.abs(got[i] - (label + want @ layers[0].o)) <= err).all()
    assert reader.keep([1, 2]) == sum((reader.lengths[s] + page - 1) // page for s in (2, 3)) - len(question) // page
    refs, lengths, tables = reader.cache.tables()
    assert (refs > 0).sum() == reader.cache.pages - (refs == 0).sum() and lengths[0] == lengths[1] == lengths[4] == 0
    assert (np.flatnonzero(refs) == np.arange((refs > 0).sum())).all()
    with pytest.raises(ValueError, match="cannot take"):
        reader.append([2], [np.zeros((200, width))])
    with pytest.raises(ValueError, match="4 passages"):
        reader.read(question, passages[:3])
    reader.close()


def test_a_decoding_step_in_a_graph():
    """extend, rotary, append and attention captured once and replayed, with
    other work between the replays: the same cache and outputs, bit for bit, as
    the calls made one by one."""
    print("graph", flush=True)
    hip = _lib.load()  # (and what it is linked to)

    def ok(name, *args):
        assert getattr(hip, name)(*args) == 0, name

    rng = np.random.default_rng(12)
    lengths = [15, 0, 63, 200, 31]
    n, heads, kv, d = len(lengths), 8, 2, 64
    with rocm.Runtime(0) as rt:
        stream = C.c_void_p()
        ok("hipStreamCreate", C.byref(stream))
        rt.set_stream(stream.value)
        m = filled(rng, lengths, 16, kv, d, layers=2, extra_pages=40)
        m.table_pages += 4
        m.tables = np.concatenate([m.tables, np.full((n, 4), -1, np.int32)], 1)
        rot = rt.rotary_bind(rocm.rotary_freqs(d))
        seqs, ones, off = _dev(rt, range(n)), _dev(rt, [1] * n), _dev(rt, range(n + 1))
        steps = [[to_bits(rng.standard_normal((n, h, d)), "f16") for h in (heads, kv, kv)] for _ in range(6)]
        results = []
        for captured in (False, True):
            c = m.upload(rt)
            pos = rt.empty((n,), np.int32)
            q, k, v = (rt.empty((n, h, d), np.uint16) for h in (heads, kv, kv))
            q2, k2 = (rt.empty((n, h, d), np.uint16) for h in (heads, kv))
            outs = [rt.empty((n, heads, d), np.uint16) for _ in range(2)]
            other = rt.empty((n, heads, d), np.uint16)

            def step():
                rt.copy(pos, c.lengths)
                c.extend(seqs, ones)
                rt.rotary(rot, pos, [(q, q2), (k, k2)])
                for layer in (0, 1):
                    c.append(layer, k2, v, off)
                    c.attention(layer, q2, off, out=outs[layer], longest=256)

            graph, run = C.c_void_p(), C.c_void_p()
            if captured:
                rt.synchronize()
                ok("hipStreamBeginCapture", stream, 2)  # relaxed
                step()
                ok("hipStreamEndCapture", stream, C.byref(graph))
                ok("hipGraphInstantiate", C.byref(run), graph, None, None, C.c_size_t(0))
            seen = []
            for x in steps:
                for a, b in zip((q, k, v), x):
                    a.upload(b)
                if captured:
                    ok("hipGraphLaunch", run, stream)
                    rt.synchronize()
                    # a call of one's own between the replays
                    c.attention(0, q2, off, out=other, longest=256)
                else:
                    step()
                rt.synchronize()
                seen.append([o.download() for o in outs])
            results.append((seen, [p.download() for p in (c.k_codes, c.v_codes, c.k_max, c.v_max, c.book)]))
            if captured:
                ok("hipGraphExecDestroy", run)
                ok("hipGraphDestroy", graph)
            c.close()
        for a, b in zip(results[0][0], results[1][0]):
            for x, y in zip(a, b):
                np.testing.assert_array_equal(x, y)
        for x, y in zip(results[0][1], results[1][1]):
            np.testing.assert_array_equal(x, y)
        assert (results[0][1][4][m.pages:m.pages + n] == np.array(lengths) + 6).all()
        rt.synchronize()
        rt.set_stream(0)
        ok("hipStreamDestroy", stream)


@pytest.mark.parametrize("counts", ["ones", "few", "many"])
def test_more_sequences_than_lanes(rt, counts):
    """150 sequences, some of them empty or without rows, listed out of order:
    append, read and attention."""
    print("many sequences", counts, flush=True)
    rng = np.random.default_rng(13)
    n, heads, kv, d, page = 150, 4, 2, 32, 16
    c_of = {"ones": [1] * n, "few": list(rng.integers(0, 9, n)), "many": list(rng.integers(0, 60, n))}[counts]
    c_of = [int(x) for x in c_of]
    lens = [x + int(rng.integers(0, 40)) for x in c_of]
    lens[3], lens[77] = 0, 0
    order = rng.permutation(n)
    by_seq = [0] * n
    for i, s in enumerate(order):
        by_seq[s] = lens[i]
    m = filled(rng, by_seq, page, kv, d)
    c = m.upload(rt)
    off = _offsets(c_of)
    t = int(off[-1])
    k, v = (to_bits(rng.standard_normal((t, kv, d)), "f16") for _ in range(2))
    seqs = [int(s) for s in order]
    c.append(0, rt.to_device(k), rt.to_device(v), _dev(rt, off), _dev(rt, seqs))
    m.append(0, from_bits(k, "f16"), from_bits(v, "f16"), off, seqs)
    m.check_pages(c)
    ko, vo = (rt.to_device(np.zeros((t, kv, d), np.float32)) for _ in range(2))
    c.read(0, _dev(rt, off), ko, vo, _dev(rt, seqs))
    ko = ko.download()
    bits = to_bits(rng.standard_normal((t, heads, d)), "f16")
    out, lse = rt.empty(bits.shape, np.uint16), rt.empty(bits.shape[:2], np.float32)
    c.attention(0, rt.to_device(bits), _dev(rt, off), _dev(rt, seqs), out=out, lse=lse, longest=max(lens))
    want, wl, err, lerr = m.attend(0, from_bits(bits, "f16").astype(np.float64), off, seqs, d ** -0.5, True, 0)
    got = from_bits(out.download(), "f16")
    assert (np.abs(got - want) <= err + np.abs(want) * 2.0 ** -11 + 2.0 ** -25).all()
    for i, s in enumerate(seqs):
        seen = min(c_of[i], lens[i])
        wk, _ = m.values(0, s)
        np.testing.assert_allclose(ko[int(off[i + 1]) - seen:int(off[i + 1])], wk[len(wk) - seen:], rtol=2.0 ** -23)
    c.close()


def test_pages_past_2_31_bytes(rt):
    """The last pages of a pool of 2.6 GB: append, read, attention, copy."""
    print("large pool", flush=True)
    rng = np.random.default_rng(14)
    kv, d, page, pages = 8, 128, 64, 40000
    c = rt.cache(pages=pages, kv_heads=kv, head_dim=d, seqs=2, table_pages=8, page_tokens=page)
    assert c.k_codes.nbytes > 1 << 31
    small = rt.cache(pages=10, kv_heads=kv, head_dim=d, seqs=2, table_pages=8, page_tokens=page)
    book = c.book.download()
    book[:pages - 6] = 1  # all but the last pages are taken
    c.book.upload(book)
    counts = [150, 70]
    off, seqs = _dev(rt, _offsets(counts)), _dev(rt, [0, 1])
    k, v, q = (rt.to_device(to_bits(rng.standard_normal((220, h, d)), "bf16")) for h in (kv, kv, 16))
    outs = []
    for x in (c, small):
        x.extend(seqs, _dev(rt, counts))
        x.append(0, k, v, off, dtype="bf16")
        ko, vo = (rt.empty((220, kv, d), np.float32) for _ in range(2))
        x.read(0, off, ko, vo)
        many = x.attention(0, q, off, longest=150, dtype="bf16").download()
        few = rt.empty((2, 16, d), np.uint16)
        x.attention(0, rocm.View(q, (2, 16, d), (16 * d, d, 1)), _dev(rt, [0, 1, 2]), out=few, longest=150, dtype="bf16")
        outs.append((ko.download(), vo.download(), many, few.download()))
    for a, b in zip(*outs):
        np.testing.assert_array_equal(a, b)
    _, _, tables = c.tables()
    last = int(tables[1, 1])
    assert last == pages - 2
    c.copy_pages(_dev(rt, [last]), _dev(rt, [pages - 1]))
    tables[1, 1] = pages - 1
    book = c.book.download()
    book[-16:] = tables.ravel()
    c.book.upload(book)
    ko, vo = (rt.empty((220, kv, d), np.float32) for _ in range(2))
    c.read(0, off, ko, vo)
    np.testing.assert_array_equal(ko.download(), outs[0][0])
    np.testing.assert_array_equal(vo.download(), outs[0][1])
    c.close()
    small.close()


def test_more_rows_than_a_launch_holds(rt):
    c = rt.cache(pages=4, kv_heads=1, head_dim=32, seqs=2, table_pages=2, page_tokens=16)
    x = _dev(rt, [0, 1])
    h = _lib.Heads(x.addr, x.addr, 16, 512, 32, 512, 32)
    with pytest.raises(_lib.MantaRocmError, match="too many rows"):
        _lib.call("manta_rocm_cache_attention", rt.handle, c.handle, 0, _lib.F16, C.byref(h), None, x.addr, None, 1,
                  1 << 25, 1.0, 1, 0, 1)
    with pytest.raises(_lib.MantaRocmError, match="too many sequences or tokens"):
        _lib.call("manta_rocm_cache_attention", rt.handle, c.handle, 0, _lib.F16, C.byref(h), None, x.addr, None, 1,
                  1 << 26, 1.0, 1, 0, 1)
    c.close()
