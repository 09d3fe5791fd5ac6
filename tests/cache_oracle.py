"""Plain restatements of the rotary and cache operators in numpy (64 bits
where the operator rounds, f32 step by step where its result is defined bit by
bit), and the glue that puts a cache's state on the device."""
import numpy as np

EPS = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # a rounding, relative to the value


def to_bits(x, dtype):
    """f32 values -> the element type's array (bf16 and f16 as uint16 bits)."""
    x = np.asarray(x, np.float32)
    if dtype == "f32":
        return x
    if dtype == "f16":
        return x.astype(np.float16).view(np.uint16)
    u = x.view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bits(a, dtype):
    if dtype == "f32":
        return a.astype(np.float32)
    if dtype == "f16":
        return a.view(np.float16).astype(np.float32)
    return (a.astype(np.uint32) << 16).view(np.float32)


def rotate(x, pos, freqs, layout, magnitude=1.0, inverse=False):
    """x [tokens, heads, d] -> f64."""
    x = np.asarray(x, np.float64)
    rot = 2 * len(freqs)
    a = np.asarray(pos, np.float64)[:, None, None] * np.asarray(freqs, np.float64)
    c, s = magnitude * np.cos(a), magnitude * np.sin(a) * (-1.0 if inverse else 1.0)
    y = x.copy()
    if layout == "half":
        x1, x2 = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = x1 * c - x2 * s, x2 * c + x1 * s
    else:
        x1, x2 = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = x1 * c - x2 * s, x2 * c + x1 * s
    return y


class Model:
    """The cache in host memory, one token at a time where that is simplest."""

    def __init__(self, layers, pages, page, heads, d, seqs, table_pages, rng=None):
        self.page, self.heads, self.d = page, heads, d
        self.pitch = (d + 31) // 32 * 32
        self.layers, self.pages, self.seqs, self.table_pages = layers, pages, seqs, table_pages
        self.k = np.zeros((layers, pages, heads, page, self.pitch), np.int8)
        self.v = np.zeros((layers, pages, heads, self.pitch, page), np.int8)
        self.km = np.zeros((layers, pages, heads), np.float32)
        self.vm = np.zeros((layers, pages, heads), np.float32)
        if rng is not None:  # pages hold what an earlier sequence left, some of it not finite
            self.k[..., :d] = rng.integers(-127, 128, self.k[..., :d].shape)
            self.v[..., :d, :] = rng.integers(-127, 128, self.v[..., :d, :].shape)
            self.km[:] = rng.choice([np.nan, np.inf, 1e30, 0.5], self.km.shape)
            self.vm[:] = rng.choice([np.nan, np.inf, 1e30, 0.5], self.vm.shape)
        self.refs = np.zeros((pages,), np.int32)
        self.lengths = np.zeros((seqs,), np.int32)
        self.tables = np.full((seqs, table_pages), -1, np.int32)

    def held(self, seq):
        return (int(self.lengths[seq]) + self.page - 1) // self.page

    # -- pages
    def extend(self, seqs, counts):
        free = [p for p in range(self.pages) if self.refs[p] == 0]
        need, copies = [], []
        for s, c in zip(seqs, counts):
            n = (int(self.lengths[s]) + c + self.page - 1) // self.page - self.held(s)
            last = int(self.tables[s, self.held(s) - 1]) if self.lengths[s] % self.page and c else -1
            need.append((s, c, n, last if last >= 0 and self.refs[last] > 1 else -1))
        if sum(n + (l >= 0) for _, _, n, l in need) > len(free):
            return False
        for s, c, n, last in need:
            h = self.held(s)
            if last >= 0:
                p = free.pop(0)
                copies.append((last, p))
                self.tables[s, h - 1], self.refs[p] = p, 1
            for k in range(n):
                p = free.pop(0)
                self.tables[s, h + k], self.refs[p] = p, 1
            self.lengths[s] += c
        for a, b in copies:
            self.refs[a] -= 1
            self.copy([a], [b])
        return True

    def fork(self, parents, children, tokens=None):
        for i, (p, c) in enumerate(zip(parents, children)):
            n = int(self.lengths[p]) if tokens is None else tokens[i]
            h = (n + self.page - 1) // self.page
            self.tables[c, :h] = self.tables[p, :h]
            for page in self.tables[p, :h]:
                self.refs[page] += 1
            self.lengths[c] = n

    def release(self, seqs, keep=None):
        for i, s in enumerate(seqs):
            n = 0 if keep is None else keep[i]
            h = (n + self.page - 1) // self.page
            for k in range(h, self.held(s)):
                self.refs[self.tables[s, k]] -= 1
                self.tables[s, k] = -1
            self.lengths[s] = n

    def copy(self, src, dst):
        for a, b in zip(src, dst):
            for x in (self.k, self.v, self.km, self.vm):
                x[:, b] = x[:, a]

    def compact(self):
        live = int((self.refs > 0).sum())
        src = [p for p in range(live, self.pages) if self.refs[p]]
        dst = [p for p in range(live) if not self.refs[p]]
        self.copy(src, dst)
        for a, b in zip(src, dst):
            self.tables[self.tables == a] = b
            self.refs[b], self.refs[a] = self.refs[a], 0
        return live

    # -- contents
    def _quantise(self, codes, old, new):
        """codes [filled, d] of largest `old`, new f32 [n, d]: the definition,
        each f32 step rounded."""
        f32 = np.float32
        with np.errstate(all="ignore"):
            if not np.isfinite(new).all() or (len(codes) and np.isnan(old)):
                return np.zeros((len(codes) + len(new), self.d)), f32(np.nan)
            big = f32(max(np.abs(new).max(), old if len(codes) else 0))
            if big < f32(2.0 ** -126):
                return np.zeros((len(codes) + len(new), self.d)), f32(0)
            keep = codes.astype(f32)
            if big > old:
                keep = np.rint((keep * f32(old)) / big)
            fresh = np.clip(np.rint((new.astype(f32) * f32(127)) / big), -127, 127)
            return np.concatenate([keep, fresh]), big

    def append(self, layer, k, v, offsets, seqs=None):
        """k, v f32 [tokens, heads, d]."""
        for i in range(len(offsets) - 1):
            s = i if seqs is None else seqs[i]
            a, b, length = offsets[i], offsets[i + 1], int(self.lengths[s])
            start = length - (b - a)
            t = max(start, 0)
            while t < length:
                p, f = self.tables[s, t // self.page], t % self.page
                e = min(length, t - f + self.page)
                rows = slice(a + t - start, a + e - start)
                n = f + e - t
                for h in range(self.heads):
                    c, m = self._quantise(self.k[layer, p, h, :f, :self.d], self.km[layer, p, h], k[rows, h])
                    self.k[layer, p, h, :n, :self.d], self.km[layer, p, h] = c, m
                    self.k[layer, p, h, :n, self.d:] = 0
                    c, m = self._quantise(self.v[layer, p, h, :self.d, :f].T, self.vm[layer, p, h], v[rows, h])
                    self.v[layer, p, h, :self.d, :n], self.vm[layer, p, h] = c.T, m
                    self.v[layer, p, h, self.d:, :n] = 0
                t = e

    def values(self, layer, seq):
        """f64 k, v [length, heads, d] of a sequence."""
        n = int(self.lengths[seq])
        rows = self.tables[seq, :self.held(seq)]
        with np.errstate(all="ignore"):
            k = self.k[layer, rows].astype(np.float64) * self.km[layer, rows].astype(np.float64)[..., None, None] / 127
            v = self.v[layer, rows].astype(np.float64) * self.vm[layer, rows].astype(np.float64)[..., None, None] / 127
        k = k.transpose(0, 2, 1, 3).reshape(-1, self.heads, self.pitch)[:n, :, :self.d]
        v = v.transpose(0, 3, 1, 2).reshape(-1, self.heads, self.pitch)[:n, :, :self.d]
        return k, v

    def attend(self, layer, q, offsets, seqs, scale, causal, window):
        """q f64 [tokens, heads, d]: (out, lse, bound of |out|'s error without
        the last rounding, bound of lse's error)."""
        out, lse = np.zeros(q.shape), np.full(q.shape[:2], -np.inf)
        err, lerr = np.zeros(q.shape), np.zeros(q.shape[:2])
        group = q.shape[1] // self.heads
        for i in range(len(offsets) - 1):
            s = i if seqs is None else seqs[i]
            k, v = self.values(layer, s)
            n, c = len(k), offsets[i + 1] - offsets[i]
            for j in range(c):
                row, pos = offsets[i] + j, n - c + j
                hi = min(n, pos + 1) if causal else n
                lo = max(0, pos - window + 1) if window else 0
                if hi <= lo:
                    continue
                for h in range(q.shape[1]):
                    kk, vv = k[lo:hi, h // group], v[lo:hi, h // group]
                    sc = kk @ q[row, h] * scale
                    m = sc.max()
                    p = np.exp(sc - m)
                    l = p.sum()
                    out[row, h], lse[row, h] = p @ vv / l, m + np.log(l)
                    # scores: products and sums of f32, their scaling and exp2's argument
                    delta = ((self.d + 8) * 2.0 ** -24 * (np.abs(kk) @ np.abs(q[row, h])).max() * abs(scale)
                             + 8 * 2.0 ** -24 * max(1.0, np.abs(sc).max()))
                    weights = p @ np.abs(vv) / l
                    # p and v * (scale of its page) as f16 operands: half a step each; p below
                    # the normal range: a quarter of its smallest step, 2^-25, absolutely, for
                    # values up to the row's largest; f32 sums
                    err[row, h] = (weights * (2 * delta + 3 * 2.0 ** -11 + (hi - lo) * 2.0 ** -24)
                                   + 2.0 ** -25 * 2 * (hi - lo) / l * np.abs(vv).max())
                    lerr[row, h] = delta + 2.0 ** -21 * max(1.0, abs(lse[row, h])) + (hi - lo) * 2.0 ** -24
        return out, lse, err, lerr

    # -- the device
    def book(self):
        return np.concatenate([self.refs, self.lengths, self.tables.ravel()])

    def upload(self, rt):
        c = rt.cache(pages=self.pages, kv_heads=self.heads, head_dim=self.d, seqs=self.seqs,
                     table_pages=self.table_pages, page_tokens=self.page, layers=self.layers)
        for part, host in ((c.k_codes, self.k), (c.v_codes, self.v), (c.k_max, self.km), (c.v_max, self.vm),
                           (c.book, self.book())):
            part.upload(host)
        return c

    def check_book(self, c):
        refs, lengths, tables = c.tables()
        np.testing.assert_array_equal(refs, self.refs)
        np.testing.assert_array_equal(lengths, self.lengths)
        np.testing.assert_array_equal(tables, self.tables)

    def check_pages(self, c):
        """Every token that a sequence holds, bit for bit."""
        k, v, km, vm = (x.download() for x in (c.k_codes, c.v_codes, c.k_max, c.v_max))
        for s in range(self.seqs):
            for j in range(self.held(s)):
                p, n = self.tables[s, j], min(self.page, int(self.lengths[s]) - j * self.page)
                np.testing.assert_array_equal(km[:, p], self.km[:, p])
                np.testing.assert_array_equal(vm[:, p], self.vm[:, p])
                np.testing.assert_array_equal(k[:, p, :, :n], self.k[:, p, :, :n])
                np.testing.assert_array_equal(v[:, p, :, :, :n], self.v[:, p, :, :, :n])


def filled(rng, lengths, page, heads, d, layers=1, extra_pages=3, extra_seqs=0, dirty=True, order=True, big=4.0):
    """A model whose sequences hold random codes, on pages in random order."""
    counts = [(n + page - 1) // page for n in lengths]
    m = Model(layers, sum(counts) + extra_pages, page, heads, d, len(lengths) + extra_seqs,
              max(counts + [1]) + 1, rng if dirty else None)
    pages = rng.permutation(m.pages) if order else np.arange(m.pages)
    at = 0
    for s, c in enumerate(counts):
        rows = pages[at:at + c]
        at += c
        m.tables[s, :c], m.lengths[s] = rows, lengths[s]
        m.refs[rows] = 1
        m.k[:, rows, :, :, :d] = rng.integers(-127, 128, m.k[:, rows, :, :, :d].shape)
        m.v[:, rows, :, :d] = rng.integers(-127, 128, m.v[:, rows, :, :d].shape)
        m.km[:, rows] = rng.uniform(0.3, 1.0, m.km[:, rows].shape) * big
        m.vm[:, rows] = rng.uniform(0.3, 1.0, m.vm[:, rows].shape) * 3.0
    return m
