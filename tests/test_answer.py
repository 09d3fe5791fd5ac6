"""The answerer's own account of its pages, on the cache's model, and what the
next step's inputs refuse."""
import numpy as np
import pytest

from cache_oracle import Model
from decode_oracle import reorder
from manta_amd import _lib, decode
from manta_amd.answer import Answerer, pool_pages


@pytest.mark.parametrize("questions,beams,tokens,page", [
    (1, 1, 16, 16), (1, 2, 16, 16), (1, 4, 16, 16), (2, 4, 16, 16), (2, 5, 9, 16), (1, 2, 64, 64), (3, 7, 30, 32),
    (1, 2, 17, 16), (2, 4, 32, 16), (1, 8, 33, 16), (2, 6, 70, 16), (2, 3, 128, 64)])
def test_no_course_of_the_beams_is_out_of_pages(questions, beams, tokens, page):
    n = questions * beams
    seqs = list(range(n))
    rng = np.random.default_rng(n * tokens)
    for course in range(40):
        m = Model(1, pool_pages(questions, beams, tokens, page), page, 1, 32, n, (tokens + page - 1) // page)
        # from one token, from a full context but one, from anywhere
        asked = {0: 1, 1: tokens - 1}.get(course, 0)
        counts = [asked or int(rng.integers(1, tokens)) for _ in range(questions)]
        assert m.extend([g * beams for g in range(questions)], counts)
        others = [s for s in seqs if s % beams]
        m.fork([s // beams * beams for s in others], others)
        lowest = rng.random() < 0.5  # most beams go on from a few
        for _ in range(tokens - max(counts)):
            assert m.extend(seqs, [1] * n)
            parents = rng.integers(0, beams, n)
            if lowest:
                parents = np.minimum(parents, rng.integers(0, beams, n))
            if course % 4 == 2:
                parents = np.arange(n) % beams // 2 * 2  # by twos
            if course % 4 == 3:
                parents[rng.random(n) < 0.2] = -1  # some have no continuation
            reorder(m, seqs, parents, beams)


def test_inputs_that_are_refused():
    class Array:
        strides = None

        def __init__(self, n, dtype=np.int32):
            self.dtype, self.shape, self.nbytes, self.addr = np.dtype(dtype), (n,), n * np.dtype(dtype).itemsize, 4096

    for tokens, out in ((Array(3, np.float32), Array(3)), (Array(3), Array(4)), (Array(3), Array(3, np.uint32))):
        with pytest.raises(ValueError, match="whole int32 array"):
            decode.beam_inputs(None, tokens, out, 0)
    for n, instead, p, message in ((-1, 0, 4096, "token count"), ((1 << 25) + 1, 0, 4096, "token count"),
                                   (1, -1, 4096, "token -1"), (1, 1 << 31, 4096, "token 2147483648"), (1, 0, None, "nil")):
        with pytest.raises(_lib.MantaRocmError, match=message):
            _lib.call("manta_rocm_beam_inputs", None, p, n, instead, p)


@pytest.mark.parametrize("most", [0, -3])
def test_answers_of_no_tokens(most):
    a = Answerer.__new__(Answerer)
    a.tokens = 64
    with pytest.raises(ValueError, match="answers of %d tokens" % most):
        a.answer([[5, 6]], most)
