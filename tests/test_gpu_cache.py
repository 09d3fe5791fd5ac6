"""The 8-bit cache's contents and pages against a host restatement: codes,
largest values, tables and reference counts bit for bit."""
import numpy as np
import pytest

from cache_oracle import Model, filled, from_bits, to_bits
from manta_amd import _lib, rocm

pytestmark = pytest.mark.gpu


def _dev(rt, x):
    return rt.to_device(np.asarray(x, np.int32))


def _offsets(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)


# ----------------------------------------------------------- append and read

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page,heads,d,lengths,counts", [
    (16, 1, 32, [1], [1]), (16, 2, 64, [16, 17, 40], [16, 1, 30]), (32, 3, 96, [33, 5, 0, 70], [3, 5, 0, 64]),
    (64, 2, 128, [64, 65, 200], [64, 2, 131]), (128, 1, 256, [129, 300], [1, 299]), (16, 2, 33, [50, 18], [1, 7]),
    (64, 8, 128, [700], [700]), (32, 1, 1, [40], [9]), (16, 5, 80, [3, 3, 31], [5, 3, 31]),
])
def test_append_and_read(rt, dtype, page, heads, d, lengths, counts):
    """Pages that begin, continue and end anywhere; a count beyond the length
    (its first rows lie before position 0); an empty sequence."""
    print("append", dtype, page, heads, d, lengths, counts, flush=True)
    rng = np.random.default_rng(page + d)
    m = filled(rng, lengths, page, heads, d)
    c = m.upload(rt)
    off = _offsets(counts)
    t = int(off[-1])
    spread = rng.choice([0.1, 1.0, 5.0], (t, heads, 1))
    k, v = (to_bits(rng.standard_normal((t, heads, d)) * spread, dtype) for _ in range(2))
    c.append(0, rt.to_device(k), rt.to_device(v), _dev(rt, off), dtype=dtype)
    m.append(0, from_bits(k, dtype), from_bits(v, dtype), off)
    m.check_pages(c)
    ko, vo = rt.to_device(np.zeros((t, heads, d), np.float32)), rt.to_device(np.zeros((t, heads, d), np.float32))
    c.read(0, _dev(rt, off), ko, vo)
    ko, vo = ko.download(), vo.download()
    for i, n in enumerate(counts):
        wk, wv = m.values(0, i)
        seen = min(n, lengths[i])
        rows = slice(int(off[i + 1]) - seen, int(off[i + 1]))
        for got, want in ((ko, wk), (vo, wv)):
            # (code * max) / 127 in f32: two roundings
            np.testing.assert_allclose(got[rows], want[len(want) - seen:], rtol=2.0 ** -23, atol=1e-37)
            np.testing.assert_array_equal(got[int(off[i]):rows.start], 0)  # rows before position 0: not written
    c.close()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_single_tokens_fill_a_page(rt, dtype):
    """A sequence written token by token, its magnitudes rising: every step
    re-rounds the page's codes as the definition does."""
    print("append steps", dtype, flush=True)
    rng = np.random.default_rng(4)
    m = Model(2, 6, 16, 2, 64, 2, 3, rng)
    c = m.upload(rt)
    ones, off = [1, 1], np.array([0, 1, 2])
    seqs = _dev(rt, [1, 0])
    for step in range(37):
        assert m.extend([1, 0], ones)
        c.extend(seqs, _dev(rt, ones))
        for layer in (0, 1):
            x = to_bits(rng.standard_normal((2, 2, 2, 64)) * (1 + 0.2 * step * (layer + 1)), dtype)
            c.append(layer, rt.to_device(x[0]), rt.to_device(x[1]), _dev(rt, off), seqs, dtype=dtype)
            m.append(layer, from_bits(x[0], dtype), from_bits(x[1], dtype), off, [1, 0])
    m.check_book(c)
    m.check_pages(c)
    c.close()


def test_values_at_the_edges(rt):
    """Halves (k + 1/2 steps), zeros, numbers below the smallest normal, the
    largest finite ones, and values that are not finite."""
    print("append edges", flush=True)
    rng = np.random.default_rng(6)
    m = Model(1, 8, 16, 1, 32, 8, 1, rng)
    x = np.zeros((8, 16, 1, 32), np.float32)
    x[0] = rng.integers(-254, 255, (16, 1, 32)) / 2.0
    x[0, 0, 0, 0] = 127.0
    x[2] = rng.standard_normal((16, 1, 32)) * 1e-39
    x[3] = rng.standard_normal((16, 1, 32)) * 3e-38
    x[4] = rng.uniform(-3.4e38, 3.4e38, (16, 1, 32))
    x[5] = rng.standard_normal((16, 1, 32))
    x[5, 3, 0, 7] = np.nan
    x[6] = rng.standard_normal((16, 1, 32))
    x[6, 15, 0, 31] = -np.inf
    x[7] = -0.0
    x = x.reshape(128, 1, 32)
    assert m.extend(range(8), [16] * 8)
    c = m.upload(rt)
    off = np.arange(9) * 16
    c.append(0, rt.to_device(x), rt.to_device(x[::-1].copy()), _dev(rt, off))
    with np.errstate(all="ignore"):
        m.append(0, x, x[::-1], off)
    m.check_pages(c)
    assert np.isnan(m.km[0, m.tables[5, 0], 0]) and np.isnan(m.km[0, m.tables[6, 0], 0])
    c.close()


def test_append_strided_listed_and_second_layer(rt):
    print("append strided", flush=True)
    rng = np.random.default_rng(8)
    m = filled(rng, [20, 50, 9], 16, 2, 48, layers=3)
    before = m.k[[0, 2]].copy()
    c = m.upload(rt)
    counts, seqs = [50, 4], [1, 0]
    off = _offsets(counts)
    for width, offset in ((2 * 2 * 48 + 5, 3), (2 * 2 * 48 + 8, 8)):
        buf = to_bits(rng.standard_normal((54, width)), "f16")
        a = rt.to_device(buf)
        k = rocm.View(a, (54, 2, 48), (width, 48, 1), offset)
        v = rocm.View(a, (54, 2, 48), (width, 48, 1), offset + 96)
        c.append(1, k, v, _dev(rt, off), _dev(rt, seqs))
        x = from_bits(buf, "f16")
        m.append(1, x[:, offset:offset + 96].reshape(54, 2, 48), x[:, offset + 96:offset + 192].reshape(54, 2, 48),
                 off, seqs)
    m.check_pages(c)
    np.testing.assert_array_equal(c.k_codes.download()[[0, 2]], before)
    # read into heads-before-tokens, rounded to bf16
    o = rt.to_device(np.zeros((2, 2, 54, 48), np.uint16))
    views = [rocm.View(o, (54, 2, 48), (48, 54 * 48, 1), i * 54 * 96) for i in (0, 1)]
    c.read(1, _dev(rt, off), views[0], views[1], _dev(rt, seqs), dtype="bf16")
    got = from_bits(o.download(), "bf16").transpose(0, 2, 1, 3)
    for i, s in enumerate(seqs):
        for j, want in enumerate(m.values(1, s)):
            np.testing.assert_allclose(got[j, off[i]:off[i + 1]], want[len(want) - counts[i]:], rtol=2.0 ** -8 * 1.01)
    c.close()


# ------------------------------------------------------------------- pages

@pytest.mark.parametrize("seed,page,pages,seqs", [(1, 16, 40, 9), (2, 64, 130, 20), (3, 128, 1100, 40),
                                                  (4, 32, 2500, 1200)])
def test_a_random_history_of_page_calls(rt, seed, page, pages, seqs):
    """extend (too many tokens at times: nothing may change), fork, release,
    compact and copy in random order; the book after every call, the pages'
    contents at the end."""
    print("pages", seed, flush=True)
    rng = np.random.default_rng(seed)
    m = Model(2, pages, page, 1, 32, seqs, 6)
    m.k[:] = rng.integers(-127, 128, m.k.shape)
    m.v[:] = rng.integers(-127, 128, m.v.shape)
    m.km[:], m.vm[:] = rng.uniform(1, 2, m.km.shape), rng.uniform(1, 2, m.vm.shape)
    c = m.upload(rt)
    live = rt.empty((1,), np.int32)
    refused = 0
    for step in range(60):
        call = rng.choice(["extend", "extend", "fork", "release", "compact", "copy"])
        who = rng.permutation(seqs)[:int(rng.integers(1, seqs + 1))]
        if call == "extend":
            counts = [int(min(rng.integers(0, 3 * page), 6 * page - m.lengths[s])) for s in who]
            done = m.extend(who, counts)
            c.extend(_dev(rt, who), _dev(rt, counts))
            if not done:
                refused += 1
                with pytest.raises(_lib.MantaRocmError, match="out of pages: "):
                    rt.synchronize()
        elif call == "fork":
            empty, full = [s for s in who if m.lengths[s] == 0], [s for s in who if m.lengths[s]]
            if not empty or not full:
                continue
            parents = [int(rng.choice(full)) for _ in empty]
            tokens = [int(rng.integers(0, m.lengths[p] + 1)) for p in parents] if step % 2 else None
            m.fork(parents, empty, tokens)
            c.fork(_dev(rt, parents), _dev(rt, empty), None if tokens is None else _dev(rt, tokens))
        elif call == "release":
            who = who[:max(1, len(who) // 2)]
            keep = [int(rng.integers(0, m.lengths[s] + 1)) for s in who] if step % 2 else None
            m.release(who, keep)
            c.release(_dev(rt, who), None if keep is None else _dev(rt, keep))
        elif call == "compact":
            n = m.compact()
            c.compact(live)
            assert int(live.download()[0]) == n
        else:
            # free pages only: what sequences hold stays
            free = np.flatnonzero(m.refs == 0)
            src = rng.permutation(np.flatnonzero(m.refs > 0))[:len(free)]
            dst = rng.permutation(free)[:len(src)]
            if not len(src):
                continue
            m.copy(src, dst)
            c.copy_pages(_dev(rt, src), _dev(rt, dst))
        m.check_book(c)
    m.check_pages(c)
    np.testing.assert_array_equal(c.k_codes.download(), m.k)
    np.testing.assert_array_equal(c.v_max.download(), m.vm)
    assert refused or seed != 1
    c.close()


def test_what_the_device_finds_wrong(rt):
    """Sequences and pages out of range, counts that do not fit, a child that
    is in use: reported by the next synchronizing call, in-bounds memory
    untouched, the calls after it as ever."""
    print("cache refusals", flush=True)
    rng = np.random.default_rng(3)
    m = filled(rng, [20, 5, 0], 16, 1, 32, extra_seqs=1)
    c = m.upload(rt)
    x = rt.to_device(rng.standard_normal((4, 1, 32)).astype(np.float32))
    zero = rt.to_device(np.zeros((4, 1, 32), np.float32))
    cases = [
        (lambda: c.extend(_dev(rt, [4]), _dev(rt, [1])), "sequence 4 out of range"),
        (lambda: c.extend(_dev(rt, [-1]), _dev(rt, [1])), "sequence -1 out of range"),
        (lambda: c.extend(_dev(rt, [0]), _dev(rt, [-1])), "sequence 0: count -1"),
        (lambda: c.extend(_dev(rt, [1, 0]), _dev(rt, [1, 10 ** 6])), "sequence 0: count 1000000"),
        (lambda: c.fork(_dev(rt, [0]), _dev(rt, [1])), "sequence 1 is not empty"),
        (lambda: c.fork(_dev(rt, [2]), _dev(rt, [2])), "sequence 2 is not empty"),
        (lambda: c.fork(_dev(rt, [0]), _dev(rt, [2]), _dev(rt, [21])), "sequence 0: count 21"),
        (lambda: c.fork(_dev(rt, [9]), _dev(rt, [2])), "sequence 9 out of range"),
        (lambda: c.release(_dev(rt, [7])), "sequence 7 out of range"),
        (lambda: c.release(_dev(rt, [1]), _dev(rt, [6])), "sequence 1: count 6"),
        (lambda: c.copy_pages(_dev(rt, [0]), _dev(rt, [m.pages])), "page %d out of range" % m.pages),
        (lambda: c.copy_pages(_dev(rt, [-5]), _dev(rt, [0])), "page -5 out of range"),
        (lambda: c.append(0, x, x, _dev(rt, [0, 4]), _dev(rt, [4])), "sequence 4 out of range"),
        (lambda: c.read(0, _dev(rt, [0, 4]), zero, zero, _dev(rt, [-3])), "sequence -3 out of range"),
    ]
    for f, text in cases:
        f()
        with pytest.raises(_lib.MantaRocmError, match=text):
            rt.synchronize()
        rt.synchronize()  # reported once
        m.check_book(c)
    np.testing.assert_array_equal(zero.download(), 0)
    # a table that names a page that is not there
    m.tables[0, 1], good = m.pages + 3, m.tables[0, 1]
    c.book.upload(m.book())
    c.append(0, x, x, _dev(rt, [0, 4]))
    with pytest.raises(_lib.MantaRocmError, match="page %d out of range" % (m.pages + 3)):
        rt.synchronize()
    c.extend(_dev(rt, [0]), _dev(rt, [1]))
    with pytest.raises(_lib.MantaRocmError, match="page %d out of range" % (m.pages + 3)):
        rt.synchronize()
    m.tables[0, 1] = good
    c.book.upload(m.book())
    m.check_pages(c)
    # what the host sees
    off = _dev(rt, [0, 4])
    for f, text in ((lambda: c.append(1, x, x, off), "layer 1 out of range"),
                    (lambda: c.append(-1, x, x, off), "layer -1 out of range"),
                    (lambda: c.append(0, x, x, _dev(rt, [0, 1, 2, 3, 4, 4])), "more sequences"),
                    (lambda: c.extend(_dev(rt, [0] * 5), _dev(rt, [0] * 5)), "sequence count 5"),
                    (lambda: rt.cache(4, 1, 64, 2, 2, page_tokens=20), "page_tokens"),
                    (lambda: rt.copy(x, x), "overlap")):
        with pytest.raises(_lib.MantaRocmError, match=text):
            f()
    for f in (lambda: c.append(0, x, rt.empty((3, 1, 32), np.float32), off),
              lambda: c.append(0, rt.empty((4, 2, 32), np.float32), x, off),
              lambda: c.append(0, x, x, rt.empty((2,), np.int64)),
              lambda: c.fork(_dev(rt, [0]), _dev(rt, [1, 2]))):
        with pytest.raises(ValueError):
            f()
    m.check_pages(c)
    c.close()


def test_lifetimes(rt):
    print("cache lifetimes", flush=True)
    with rocm.Runtime(0) as other:
        c = other.cache(4, 1, 64, 2, 2)
        ones = rt.to_device(np.ones(1, np.int32))
        with pytest.raises(_lib.MantaRocmError, match="another runtime"):
            _lib.call("manta_rocm_cache_extend", rt.handle, c.handle, ones.addr, ones.addr, 1)
    with pytest.raises(_lib.MantaRocmError, match="runtime is destroyed"):
        _lib.call("manta_rocm_cache_extend", rt.handle, c.handle, ones.addr, ones.addr, 1)
    assert _lib.load().manta_rocm_cache_buffers(c.handle, _lib.CacheBuffers()) == _lib.ERROR
    c.close()
    c.close()
