"""Answers in caches as small as they may be, and of questions that come to
nothing."""
import numpy as np
import pytest

from manta_amd.answer import Answerer, random_model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("questions,beams,tokens,page", [(1, 4, 16, 16), (2, 2, 64, 64), (2, 5, 9, 16)])
def test_a_question_and_its_answer_in_one_page(rt, questions, beams, tokens, page):
    """... and as in pages of which there are several."""
    print("answer one page", questions, beams, tokens, page, flush=True)
    rng = np.random.default_rng(tokens)
    m = random_model(rt, rng, 2, 200, 128, 2, 2, 64, 128)
    asked = [rng.integers(3, 200, 3 + g).tolist() for g in range(questions)]
    found = []
    for t in (tokens, 10 * page):
        a = Answerer(rt, m, questions, beams, t, end_token=2, page_tokens=page)
        found.append(a.answer(asked, tokens - 4))
        a.close()
    assert all(len(beams_of) == beams for beams_of in found[0])
    assert [[b for b, _ in q] for q in found[0]] == [[b for b, _ in q] for q in found[1]]
    m.close()
