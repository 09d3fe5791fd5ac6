"""Plain restatements of the decoding operators in numpy: whole numbers as they
are defined, step by step in f32, everything else in 64 bits."""
import math

import numpy as np

from cache_oracle import EPS, rotate

U = 2.0 ** -24  # a rounding of f32, relative to the value
SMALLEST = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}


def rounding(want, dtype):
    """How far a rounding to the element type may be off."""
    return np.abs(want) * EPS[dtype] + SMALLEST[dtype] / 2


def quantise(x, norm=None, eps=1e-6):
    """x f32 [rows, width] -> (codes [rows, width], scales f64 [rows])."""
    f32 = np.float32
    with np.errstate(all="ignore"):
        z = x if norm is None else x * norm.astype(f32)
        big = np.abs(z).max(1)
        bad = ~np.isfinite(z).all(1)
        tiny = big < f32(2.0 ** -126)
        codes = np.clip(np.rint((z * f32(127)) / big[:, None]), -127, 127)
        scales = big.astype(np.float64) / 127
        if norm is not None:
            scales = scales / np.sqrt((x.astype(np.float64) ** 2).mean(1) + eps)
    codes[bad | tiny] = 0
    return codes.astype(np.int8), np.where(bad, np.nan, np.where(tiny, 0.0, scales))


def activate(v, gate):
    with np.errstate(over="ignore"):
        if gate == "silu":
            return v / (1.0 + np.exp(-v))
        return v / (1.0 + np.exp(-2.0 * 0.7978845608 * (v + 0.044715 * v ** 3)))


def product(codes, scales, w, w_scales, dtype, add=None, gate=None):
    """(result f64, how far the device's may be off).

    The sum is exact; it, the two scales' product and theirs are rounded to f32
    (3 U), and so is add's sum.  An activation: its argument is off by 3 U, its
    slope is at most 1.13; gelu's polynomial and its factors are 6 roundings and
    |u| times the logistic function's slope at u at most 0.28; exp, the sum and
    the quotient are 4 U of the result; then the product with the other half
    and that half's own 3 U."""
    y = (codes.astype(np.int64) @ w.astype(np.int64)) * np.outer(scales, np.asarray(w_scales, np.float64))
    if gate is None:
        off = 3 * U * np.abs(y)
        if add is not None:
            y = y + add
            off = off + U * np.abs(y)
    else:
        n = w.shape[1] // 2
        v, u = y[:, :n], y[:, n:]
        act = activate(v, gate)
        y = act * u
        off = np.abs(u) * np.abs(v) * (1.13 * 3 + 2 * 0.28 * 6) * U + 8 * U * np.abs(y)
    return y, off * 1.001 + rounding(np.abs(y) + off, dtype)


def rotary_normed(x, norm, eps, pos, freqs, layout, magnitude):
    """x [tokens, heads, d] -> (f64, how far f32 arithmetic may be off)."""
    x = np.asarray(x, np.float64)
    if norm is not None:
        x = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * np.asarray(norm, np.float64)
    y = rotate(x, pos, freqs, layout, magnitude)
    # the factor and two products: 3 U; the angle, cos and sin, products and sum: 12 U of both columns
    return y, 2 * np.abs(x).max(-1, keepdims=True) * abs(magnitude) * 15 * U


def beams(logits, scores, best, ended=None, end_token=0):
    """logits [groups, beams, vocab]: (parents, tokens, totals) [groups, best]."""
    groups, nb, vocab = logits.shape
    parents, tokens = np.full((groups, best), -1), np.full((groups, best), -1)
    totals = np.full((groups, best), -np.inf)
    for g in range(groups):
        found = []
        for b in range(nb):
            score = float(scores[g, b])
            if ended is not None and ended[g, b]:
                if score > -np.inf:
                    found.append((-score, b, end_token))
                continue
            row = logits[g, b].astype(np.float64)
            top = row.max()
            if not np.isfinite(row[~np.isneginf(row)]).all() or np.isneginf(top):
                continue
            log_sum = math.log(math.fsum(np.exp(row - top)))
            order = np.argsort(-row, kind="stable")[:best]
            for t in order:
                total = score + ((row[t] - top) - log_sum)
                if total > -np.inf:
                    found.append((-total, b, int(t)))
        for k, (t, b, token) in enumerate(sorted(found)[:best]):
            parents[g, k], tokens[g, k], totals[g, k] = b, token, -t
    return parents, tokens, totals


def reorder(model, seqs, parents, group):
    """cache_oracle.Model's sequences, as Cache.reorder leaves them."""
    tables, lengths = model.tables.copy(), model.lengths.copy()
    for i, (s, p) in enumerate(zip(seqs, parents)):
        source = None if p < 0 else seqs[i // group * group + p]
        new = np.full_like(tables[s], -1) if source is None else tables[source]
        for page in model.tables[s][model.tables[s] >= 0]:
            model.refs[page] -= 1
        for page in new[new >= 0]:
            model.refs[page] += 1
        model.tables[s] = new
        model.lengths[s] = 0 if source is None else lengths[source]
