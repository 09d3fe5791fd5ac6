"""Totals that are equal in 64 bits where their logits are not: within a beam
the larger logit comes first, then the lower token; the lower beam before."""
import numpy as np
import pytest

from cache_oracle import from_bits, to_bits

pytestmark = pytest.mark.gpu


def _order(logits, scores, best):
    """By (total, beam, logit, token): every total here is the score's, or the
    differences are far above 64 bits."""
    parents, tokens = [], []
    for g in range(len(logits)):
        found = []
        for b, row in enumerate(logits[g].astype(np.float64)):
            top = row.max()
            total = float(scores[g, b]) + ((row - top) - np.log(np.exp(row - top).sum()))
            found += [(-t, b, -x, i) for i, (t, x) in enumerate(zip(total, row)) if t > -np.inf]
        found = sorted(found)[:best]
        parents.append([f[1] for f in found])
        tokens.append([f[3] for f in found])
    return np.array(parents), np.array(tokens)


def _select(rt, logits, scores, best, dtype):
    out = [rt.empty((len(logits), best), np.int32) for _ in range(2)] + [rt.empty((len(logits), best), np.float32)]
    rt.beams(len(logits), logits.shape[1], best).select(
        rt.to_device(to_bits(logits, dtype)), rt.to_device(np.asarray(scores, np.float32)), *out, dtype=dtype)
    return out[0].download(), out[1].download()


def test_small_logits_beside_a_large_one(rt):
    logits = np.full((1, 2, 300), -5.0, np.float32)
    logits[0, :, 7] = 20.0
    logits[0, :, [10, 20, 30, 40]] = np.array([1e-20, 2e-20, -1e-20, 2e-20], np.float32)[:, None]
    parents, tokens = _select(rt, logits, [[-1.0, -1.0]], 10, "f32")
    assert parents.tolist() == [[0, 1] + [0] * 4 + [1] * 4]
    assert tokens.tolist() == [[7, 7] + [20, 40, 10, 30] * 2]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nb,vocab,best", [(1, 40, 8), (3, 5000, 16), (4, 20001, 64), (64, 3000, 64)])
def test_scores_that_swallow_the_logits(rt, dtype, nb, vocab, best):
    """Scores of -1e20: every total of a beam is its score.  Of 64 beams with 64
    results more totals are equal than are ranked at once."""
    print("beams order", dtype, nb, vocab, best, flush=True)
    rng = np.random.default_rng(vocab)
    logits = from_bits(to_bits(rng.standard_normal((2, nb, vocab)), dtype), dtype)
    scores = np.full((2, nb), -1e20, np.float32)
    scores[1, 0] = -2e20
    parents, tokens = _select(rt, logits, scores, best, dtype)
    want = _order(logits, scores, best)
    np.testing.assert_array_equal(parents, want[0])
    np.testing.assert_array_equal(tokens, want[1])
