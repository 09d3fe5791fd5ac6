"""Cache.reorder of groups of more than 128 sequences (fewer columns of their
tables a workgroup), and beams of more rows than a launch takes."""
import numpy as np
import pytest

from cache_oracle import Model
from decode_oracle import beams, reorder

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("groups,group,tables", [(1, 129, 70), (2, 200, 40), (1, 256, 33), (3, 300, 17), (1, 1000, 20),
                                                 (4, 1024, 9)])
def test_large_groups(rt, groups, group, tables):
    """Sequences that share the pages of the one before here and there."""
    print("reorder large", groups, group, tables, flush=True)
    rng = np.random.default_rng(group)
    n = groups * group
    seqs = rng.permutation(n + 3)[:n]
    m = Model(1, 40000, 16, 1, 32, n + 3, tables)
    free = iter(rng.permutation(m.pages))
    for i, s in enumerate(seqs):
        held = int(rng.integers(0, tables + 1)) if rng.random() < 0.2 else int(rng.integers(0, 9))
        m.lengths[s] = max(0, held * 16 - int(rng.integers(0, 16)))
        for j in range(held):
            before = m.tables[seqs[i - 1], j] if i else -1
            m.tables[s, j] = before if before >= 0 and rng.random() < 0.5 else next(free)
            m.refs[m.tables[s, j]] += 1
    c = m.upload(rt)
    for step in range(3):
        parents = rng.integers(0, group, n)
        if step == 1:
            parents = np.concatenate([rng.permutation(group) for _ in range(groups)])
        if step == 2:
            parents[rng.random(n) < 0.3] = -1
        c.reorder(rt.to_device(seqs.astype(np.int32)), rt.to_device(parents.astype(np.int32)), group)
        reorder(m, seqs, parents, group)
        m.check_book(c)


@pytest.mark.parametrize("groups,nb,vocab,best,ended", [(70000, 1, 5, 2, False), (22000, 3, 7, 4, True), (1100, 64, 9, 3, True)])
def test_more_beams_than_a_launch_takes(rt, groups, nb, vocab, best, ended):
    print("beams many", groups, nb, vocab, best, flush=True)
    rng = np.random.default_rng(groups)
    logits = rng.standard_normal((groups, nb, vocab)).astype(np.float32)
    scores = -rng.random((groups, nb)).astype(np.float32)
    over = (rng.random((groups, nb)) < 0.2).astype(np.int32) if ended else None
    out = [rt.empty((groups, best), np.int32) for _ in range(2)] + [rt.empty((groups, best), np.float32)]
    now = rt.empty((groups, best), np.int32)
    h = rt.beams(groups, nb, best)
    for _ in range(2):  # (the tickets are zero again)
        h.select(rt.to_device(logits), rt.to_device(scores), *out, ended=None if over is None else rt.to_device(over),
                 end_token=2, out_ended=now)
        want = beams(logits, scores, best, over, 2)
        np.testing.assert_array_equal(out[0].download(), want[0])
        np.testing.assert_array_equal(out[1].download(), want[1])
        np.testing.assert_allclose(out[2].download(), want[2], rtol=2.0 ** -23)
        np.testing.assert_array_equal(now.download(), (want[1] == 2).astype(np.int32))
