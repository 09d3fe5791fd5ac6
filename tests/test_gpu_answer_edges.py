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


def _inputs(rt, tokens, instead):
    t = rt.to_device(np.asarray(tokens, np.int32))
    out = rt.to_device(np.full(t.shape, -9, np.int32))
    rt.beam_inputs(t, out, instead)
    return out.download()


def test_inputs_of_the_next_step(rt):
    rng = np.random.default_rng(0)
    for shape in ((1,), (3, 4), (1000, 7), (0,)):
        tokens = rng.integers(-2, 5, shape).astype(np.int32)
        np.testing.assert_array_equal(_inputs(rt, tokens, 9), np.where(tokens < 0, 9, tokens))
    t = rt.to_device(np.array([-1, 2 ** 31 - 1, 0], np.int32))
    rt.beam_inputs(t, t, 2 ** 31 - 1)
    assert t.download().tolist() == [2 ** 31 - 1, 2 ** 31 - 1, 0]


@pytest.mark.parametrize("beams", [1, 3])
def test_a_question_without_continuations_leaves_the_others_alone(rt, beams):
    """Logits that are not numbers: from the start (the question has a token
    whose row is not finite), and after some steps (it comes to one)."""
    print("answer dead", beams, flush=True)

    def ask(bad, questions):
        m = random_model(rt, np.random.default_rng(beams), 2, 400, 128, 2, 2, 64, 128)
        table = m.table.download()
        table[bad] = np.float16(np.inf).view(np.uint16)
        m.table.upload(table)
        a = Answerer(rt, m, 2, beams, 64, end_token=2)
        found = a.answer(questions, 8)
        chosen = a.parents.download(), a.next.download()
        # the cache is as whole as it was: another answer
        again = a.answer(questions, 8)
        a.close()
        m.close()
        assert again == found
        return found, chosen

    rng = np.random.default_rng(77)
    one, other = rng.integers(3, 200, 11).tolist(), rng.integers(3, 200, 6).tolist()
    whole, _ = ask([], [one, other])
    bad = min(set(range(200, 400)) - {x for q in whole for t, _ in q for x in t})
    found, (parents, tokens) = ask([bad], [one, other[:3] + [bad] + other[4:]])
    assert found[0] == whole[0]
    assert found[1] == [] and (parents[1] == -1).all() and (tokens[1] == -1).all()
    # every token that the other question's beams begin with, and the first one's have nowhere
    first = {t[k] for t, _ in whole[1] for k in (1, 2) if len(t) > k} - {x for t, _ in whole[0] for x in t}
    assert first
    found, _ = ask(sorted(first), [one, other])
    assert found[0] == whole[0] and len(found[1]) <= beams


def test_all_questions_without_continuations(rt):
    m = random_model(rt, np.random.default_rng(1), 1, 300, 128, 2, 2, 64, 128)
    m.table.upload(np.full(m.table.shape, np.float16(np.nan).view(np.uint16)))
    a = Answerer(rt, m, 2, 2, 64, end_token=2)
    assert a.answer([[5, 6], [7]], 5) == [[], []]
    a.close()
    m.close()
