"""Cache.reorder: tables, lengths and references equal to the definition's."""
import numpy as np
import pytest

from cache_oracle import filled
from decode_oracle import reorder
from manta_amd import _lib

pytestmark = pytest.mark.gpu


def _dev(rt, x):
    return rt.to_device(np.asarray(x, np.int32))


def _grow(m, rng, groups, nb):
    """groups prefixes forked into nb beams each, which go on on their own."""
    for g in range(groups):
        seqs = [groups + g * nb + b for b in range(nb)]
        m.fork([g] * nb, seqs)
        assert m.extend(seqs, [int(x) for x in rng.integers(1, 40, nb)])
    m.release(range(groups))


@pytest.mark.parametrize("groups,nb,page", [(1, 1, 16), (3, 4, 16), (2, 16, 32), (5, 3, 64), (1, 70, 16)])
def test_sequences_follow_their_parents(rt, groups, nb, page):
    print("reorder", groups, nb, page, flush=True)
    rng = np.random.default_rng(groups * 100 + nb)
    m = filled(rng, [int(x) for x in rng.integers(1, 300, groups)], page, 1, 32, extra_pages=groups * nb * 12 + 40,
               extra_seqs=groups * nb + 2)
    m.tables = np.concatenate([m.tables, np.full((m.seqs, 10), -1, np.int32)], 1)
    m.table_pages += 10
    _grow(m, rng, groups, nb)
    c = m.upload(rt)
    seqs = groups + np.arange(groups * nb)
    for step in range(5):
        parents = rng.integers(0, nb, groups * nb)
        if step == 1:
            parents = np.tile(np.arange(nb)[::-1], groups)  # a permutation
        if step == 3:
            parents[rng.random(len(parents)) < 0.3] = -1
        c.reorder(_dev(rt, seqs), _dev(rt, parents), nb)
        reorder(m, seqs, parents, nb)
        m.check_book(c)
        rng.shuffle(seqs.reshape(groups, nb).T)  # other orders of the slots
        # they go on: shared last pages are copied
        counts = rng.integers(0, 3, len(seqs))
        c.extend(_dev(rt, seqs), _dev(rt, counts))
        assert m.extend(seqs, [int(x) for x in counts])
        m.check_book(c)
        m.check_pages(c)


def test_one_group_of_everything_and_slots_far_apart(rt):
    """group left out, more slots than are remembered at a time, wide tables."""
    print("reorder slots", flush=True)
    rng = np.random.default_rng(8)
    lengths = [70, 0, 33, 16 * 30]
    m = filled(rng, lengths, 16, 1, 32, extra_seqs=300000, extra_pages=5)
    far = [0, 299999, 131072, 3]
    for a, b in ((1, 299999), (2, 131072)):
        m.tables[[a, b]], m.lengths[[a, b]] = m.tables[[b, a]], m.lengths[[b, a]]
    c = m.upload(rt)
    for parents in ([3, 2, 1, 0], [0, 0, 3, -1], [1, 1, 2, 2]):
        c.reorder(_dev(rt, far), _dev(rt, parents))
        reorder(m, far, parents, 4)
        m.check_book(c)


def test_wide_tables(rt):
    """More columns than a workgroup takes."""
    print("reorder wide", flush=True)
    rng = np.random.default_rng(9)
    m = filled(rng, [16 * 900, 5, 16 * 300 + 1, 0, 16 * 600, 77], 16, 1, 32)
    c = m.upload(rt)
    for parents in ([1, 2, 0, 1, 1, 0], [2, 2, 2, 0, 0, -1]):
        c.reorder(_dev(rt, [0, 2, 4, 5, 3, 1]), _dev(rt, parents), 3)
        reorder(m, [0, 2, 4, 5, 3, 1], parents, 3)
        m.check_book(c)


def test_nothing_to_do(rt):
    print("reorder empty", flush=True)
    m = filled(np.random.default_rng(0), [5], 16, 1, 32)
    c = m.upload(rt)
    c.reorder(_dev(rt, []), _dev(rt, []))
    m.check_book(c)


@pytest.mark.parametrize("seqs,parents,group,message", [
    ([0, 1, 2, 9], [0, 1, 0, 1], 2, "sequence 9 out of range"),
    ([0, 1, 2, -1], [0, 1, 0, 1], 2, "sequence -1 out of range"),
    ([0, 1, 2, 0], [0, 1, 0, 1], 2, "names sequence 0 twice"),
    ([0, 1, 2, 3], [0, 1, 2, 1], 2, "entry 2: parent 2 out of range"),
    ([0, 1, 2, 3], [0, -2, 1, 1], 4, "entry 1: parent -2 out of range"),
])
def test_a_wrong_entry_leaves_everything(rt, seqs, parents, group, message):
    """... and its sequences alone until it is reported, as a refused extend."""
    print("reorder refused", message, flush=True)
    m = filled(np.random.default_rng(1), [20, 40, 3, 100], 16, 1, 32, extra_seqs=1)
    c = m.upload(rt)
    rt.synchronize()
    c.reorder(_dev(rt, seqs), _dev(rt, parents), group)
    c.reorder(_dev(rt, [1, 2]), _dev(rt, [1, 0]))  # names a sequence of the refused call
    c.extend(_dev(rt, [2]), _dev(rt, [1]))
    with pytest.raises(_lib.MantaRocmError, match=message):
        rt.synchronize()
    m.check_book(c)
    c.reorder(_dev(rt, [1, 2]), _dev(rt, [1, 0]))
    reorder(m, [1, 2], [1, 0], 2)
    m.check_book(c)
