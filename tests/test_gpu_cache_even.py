"""Attention of few rows where the sequences' steps are cut evenly over the
card's workgroups (`longest` says that there are many): against softmax in 64
bits with the bounds of Model.attend, as test_gpu_cache_attention.py has them."""
import numpy as np
import pytest

from cache_oracle import filled
from manta_amd import _lib
from test_gpu_cache_attention import _check, _dev, _offsets

pytestmark = pytest.mark.gpu

MANY = 1 << 22


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("page,kv,group,d,n", [
    (64, 2, 4, 128, 5), (16, 3, 1, 64, 64), (32, 1, 8, 96, 17), (128, 2, 2, 256, 3), (16, 4, 16, 32, 9), (64, 1, 3, 80, 2),
    (32, 2, 5, 160, 6), (64, 1, 1, 192, 4), (16, 1, 2, 224, 7),
])
def test_ragged_single_tokens(rt, dtype, page, kv, group, d, n):
    print("even", dtype, page, kv, group, d, n, flush=True)
    rng = np.random.default_rng(n + d)
    lengths = [int(x) for x in rng.choice([1, 2, 15, 16, 17, 64, 65, 200, 700, 1500], n)]
    lengths[0], lengths[-1] = 1, 2300
    m = filled(rng, lengths, page, kv, d)
    _check(rt, m, rng, dtype, kv * group, [1] * n, longest=MANY)


@pytest.mark.parametrize("window,causal", [(0, True), (100, True), (1, True), (0, False)])
@pytest.mark.parametrize("counts", [[1, 0, 3, 1, 0], [0, 0, 9, 1, 2], [4, 4, 4, 4, 4]])
def test_counts_windows_and_rows_that_see_nothing(rt, counts, window, causal):
    """Several tiles a sequence, sequences without rows or without tokens, more
    rows than tokens, rows that no sequence owns."""
    print("even counts", counts, window, causal, flush=True)
    rng = np.random.default_rng(21)
    m = filled(rng, [900, 0, 333, 2, 64], 32, 2, 64)
    _check(rt, m, rng, "f16", 14, counts, window=window, causal=causal, longest=MANY, extra_rows=2)


@pytest.mark.parametrize("page,kv,group,d,counts", [
    (16, 2, 4, 64, [5, 8, 1, 7, 6, 5]), (32, 1, 6, 96, [5] * 9), (64, 2, 4, 128, [8, 0, 16, 1]), (16, 1, 1, 32, [32, 20, 31]),
    (128, 1, 8, 256, [3, 4]), (64, 1, 25, 160, [1, 1, 1]),
])
def test_tiles_of_32_rows(rt, page, kv, group, d, counts):
    print("even 32 rows", page, kv, group, d, counts, flush=True)
    rng = np.random.default_rng(24)
    m = filled(rng, [c + int(x) for c, x in zip(counts, rng.integers(0, 900, len(counts)))], page, kv, d)
    for window in (0, 150):
        _check(rt, m, rng, "bf16", kv * group, counts, window=window, longest=MANY)


def test_one_long_sequence_among_short_ones(rt):
    """A tile in many parts, and workgroups that end several tiles."""
    print("even long", flush=True)
    rng = np.random.default_rng(22)
    m = filled(rng, [40000] + [70] * 20 + [5000], 64, 1, 32)
    _check(rt, m, rng, "bf16", 4, [1] * 22, longest=MANY)


def test_listed_sequences_in_place_and_again(rt):
    print("even listed", flush=True)
    rng = np.random.default_rng(23)
    m = filled(rng, [800, 90, 0, 1300, 500], 16, 2, 64, layers=2)
    for _ in range(3):  # the tickets are zero between calls
        _check(rt, m, rng, "f16", 8, [1, 1, 1], seqs=[3, 0, 4], layer=1, longest=MANY)
    c = m.upload(rt)
    q = rt.to_device(np.zeros((2, 8, 64), np.uint16))
    out = c.attention(0, q, _dev(rt, _offsets([1, 1])), _dev(rt, [0, 9]), longest=MANY)
    with pytest.raises(_lib.MantaRocmError, match="sequence 9 out of range"):
        rt.synchronize()
    assert (out.download()[1] == 0).all()
    m.tables[1, 2] = m.pages + 1
    c.book.upload(m.book())
    c.attention(0, q, _dev(rt, _offsets([1, 1])), longest=MANY)
    with pytest.raises(_lib.MantaRocmError, match="page %d out of range" % (m.pages + 1)):
        rt.synchronize()
    c.close()


@pytest.mark.parametrize("page,kv,group,d,n,count", [
    (64, 40, 16, 64, 3, 130), (16, 130, 2, 32, 4, 40), (64, 130, 1, 128, 4, 60), (32, 130, 1, 96, 4, 70),
    (16, 130, 1, 128, 4, 60),
])
def test_prompts_in_tiles_of_256_rows(rt, page, kv, group, d, n, count):
    """More tiles than the card has places."""
    print("prompts", page, kv, group, d, n, count, flush=True)
    rng = np.random.default_rng(25)
    counts = [count] + [int(x) for x in rng.integers(3 * count // 4, count, n - 1)]
    m = filled(rng, [c + int(x) for c, x in zip(counts, rng.integers(0, 80, n))], page, kv, d)
    _check(rt, m, rng, "f16", kv * group, counts, window=40 if page == 32 else 0)
