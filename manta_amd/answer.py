"""Answers to questions, by beams: how the calls of decode.py and cache.py make
a decoder, every step of it on the device.  A question enters the cache once;
its best first tokens become beams that share its pages (fork); and a step
reads one token of every beam, chooses the next ones (Beams.select) and makes
the cache's sequences follow them (Cache.reorder).

A layer is x + o(attention(rotate(norm(q)), rotate(norm(k)), v)) of x normed
and projected, then x + down(silu(x G) * (x U)) of x normed; weights are 8-bit
codes with a scale a column, activations f16 between the products and 8-bit
codes with a scale a token within them.

`python -m manta_amd.answer` answers random questions with random weights.
"""
from __future__ import annotations

from typing import List, Sequence, Tuple

import numpy as np

from .rocm import Runtime, View, pack_q8_rows, rotary_freqs


def columns_q8(w: np.ndarray) -> Tuple[np.ndarray, np.ndarray]:
    """A weight [width, n] as int8 codes with an f32 scale a column."""
    codes, scales = pack_q8_rows(np.asarray(w, np.float32).T)
    return np.ascontiguousarray(codes.T), scales


class Block:
    """A layer's weights on the device: q, k and v side by side, o, gate and up
    side by side, down (all f32 [width, columns] on the way in), and the norms
    of the layer's two inputs [width] and of queries and keys [head_dim]."""

    def __init__(self, rt: Runtime, q, k, v, o, gate, up, down, attend_norm, feed_norm, q_norm, k_norm):
        self.qkv = rt.weight(*columns_q8(np.concatenate([q, k, v], 1)))
        self.o = rt.weight(*columns_q8(o))
        self.feed = rt.weight(*columns_q8(np.concatenate([gate, up], 1)), gate="silu")
        self.down = rt.weight(*columns_q8(down))
        self.attend_norm, self.feed_norm, self.q_norm, self.k_norm = (
            rt.to_device(np.asarray(x, np.float32)) for x in (attend_norm, feed_norm, q_norm, k_norm))

    def close(self) -> None:
        for w in (self.qkv, self.o, self.feed, self.down):
            w.close()


class Model:
    """table f16 [vocab, width] (rows the tokens' inputs), the blocks, the last
    norm [width] and the head f32 [width, vocab]."""

    def __init__(self, rt: Runtime, table, blocks: Sequence[Block], norm, head, q_heads: int, kv_heads: int,
                 head_dim: int):
        self.table = rt.to_device(np.asarray(table, np.float16).view(np.uint16))
        self.blocks, self.norm = list(blocks), rt.to_device(np.asarray(norm, np.float32))
        self.head = rt.weight(*columns_q8(head))
        self.vocab, self.width = self.table.shape
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim

    def close(self) -> None:
        for b in self.blocks:
            b.close()
        self.head.close()


class _Rows:
    """The activations of `rows` tokens."""

    def __init__(self, rt: Runtime, m: Model, rows: int):
        d, q, kv = m.head_dim, m.q_heads, m.kv_heads
        self.x = rt.empty((rows, m.width), np.uint16)
        self.qkv = rt.empty((rows, (q + 2 * kv) * d), np.uint16)
        strides = ((q + 2 * kv) * d, d, 1)
        self.q = View(self.qkv, (rows, q, d), strides)
        self.k = View(self.qkv, (rows, kv, d), strides, q * d)
        self.v = View(self.qkv, (rows, kv, d), strides, (q + kv) * d)
        self.attended = rt.empty((rows, q, d), np.uint16)
        self.flat = View(self.attended, (rows, q * d), (q * d, 1))
        self.fed = rt.empty((rows, m.blocks[0].feed.n), np.uint16)
        self.x8, self.a8, self.f8 = (rt.quantized(rows, w) for w in (m.width, q * d, m.blocks[0].feed.n))


def pool_pages(questions: int, beams: int, tokens: int, page_tokens: int) -> int:
    """Pages that any course of the beams finds enough: each beam's own, and of
    beams of one page one more for every two.  (Several beams that go on from
    one take a copy each of its last page before that page is free; of more
    than one page they share the others, and have as many to spare.)"""
    each = (tokens + page_tokens - 1) // page_tokens
    return questions * (beams * each + (beams // 2 if each == 1 else 0))


class Answerer:
    """Answers up to `questions` questions at once with `beams` beams each;
    a question and its answer have at most `tokens` tokens.  Sequence
    g * beams + b of the cache is beam b of question g."""

    def __init__(self, rt: Runtime, model: Model, questions: int, beams: int, tokens: int, end_token: int,
                 page_tokens: int = 16):
        if beams > model.vocab:
            raise ValueError("%d beams of a vocabulary of %d" % (beams, model.vocab))
        self.rt, self.model, self.beams, self.tokens, self.end_token = rt, model, beams, tokens, end_token
        self.questions = questions
        n = questions * beams
        each = (tokens + page_tokens - 1) // page_tokens
        self.cache = rt.cache(pages=pool_pages(questions, beams, tokens, page_tokens), kv_heads=model.kv_heads,
                              head_dim=model.head_dim, seqs=n, table_pages=each, page_tokens=page_tokens,
                              layers=len(model.blocks))
        self.rot = rt.rotary_bind(rotary_freqs(model.head_dim))
        self.choice = rt.beams(questions, beams, beams)
        self.seqs, self.ones = self._ints(range(n)), self._ints([1] * n)
        self.offsets = self._ints(range(n + 1))
        self.positions, self.tokens_now = self._ints([0] * n), self._ints([0] * n)
        self.rows = _Rows(rt, model, n)
        self.last8 = rt.quantized(n, model.width)
        self.logits = rt.empty((questions, beams, model.vocab), np.float32)
        self.flat_logits = View(self.logits, (n, model.vocab), (model.vocab, 1))
        self.scores = rt.empty((questions, beams), np.float32)
        self.ended = rt.empty((questions, beams), np.int32)
        self.parents = rt.empty((questions, beams), np.int32)
        self.flat_parents = View(self.parents, (n,), (1,))
        self.next = rt.empty((questions, beams), np.int32)

    def _ints(self, x):
        return self.rt.to_device(np.asarray(x, np.int32))

    def _layers(self, r: _Rows, positions, offsets, seqs) -> None:
        rt, c = self.rt, self.cache
        for i, b in enumerate(self.model.blocks):
            rt.quantize_rows(r.x, r.x8, norm=b.attend_norm)
            rt.matmul_q8(b.qkv, r.x8, out=r.qkv)
            rt.rotary_normed(self.rot, positions, [(r.q, r.q), (r.k, r.k)], [b.q_norm, b.k_norm])
            c.append(i, r.k, r.v, offsets, seqs)
            c.attention(i, r.q, offsets, seqs, out=r.attended, longest=self.tokens)
            rt.quantize_rows(r.flat, r.a8)
            rt.matmul_q8(b.o, r.a8, out=r.x, add=r.x)
            rt.quantize_rows(r.x, r.x8, norm=b.feed_norm)
            rt.matmul_q8(b.feed, r.x8, out=r.fed)
            rt.quantize_rows(r.fed, r.f8)
            rt.matmul_q8(b.down, r.f8, out=r.x, add=r.x)

    def ask(self, questions: Sequence[Sequence[int]]) -> None:
        """Read the questions (token lists) and choose their first beams."""
        if len(questions) != self.questions:
            raise ValueError("%d questions expected (got %d)" % (self.questions, len(questions)))
        counts = [len(q) for q in questions]
        if min(counts) < 1 or max(counts) >= self.tokens:
            raise ValueError("questions of 1 to %d tokens" % (self.tokens - 1))
        rt, nb = self.rt, self.beams
        self.cache.release(self.seqs)
        firsts = self._ints([g * nb for g in range(self.questions)])
        offsets = np.concatenate([[0], np.cumsum(counts)])
        off = self._ints(offsets)
        self.cache.extend(firsts, self._ints(counts))
        r = _Rows(rt, self.model, int(offsets[-1]))
        rt.gather_rows_f16(self.model.table, self._ints(np.concatenate([np.asarray(q) for q in questions])), out=r.x)
        self._layers(r, self._ints(np.concatenate([np.arange(n) for n in counts])), off, firsts)
        last = rt.quantize_rows(rt.gather_rows_f16(r.x, self._ints(offsets[1:] - 1)), norm=self.model.norm)
        logits = rt.empty((self.questions, 1, self.model.vocab), np.float32)
        rt.matmul_q8(self.model.head, last, out=View(logits, (self.questions, self.model.vocab), (self.model.vocab, 1)))
        self.choice.select(logits, rt.to_device(np.zeros((self.questions, 1), np.float32)), self.parents, self.next,
                           self.scores, end_token=self.end_token, out_ended=self.ended)
        if nb > 1:
            others = [g * nb + b for g in range(self.questions) for b in range(1, nb)]
            self.cache.fork(self._ints([s // nb * nb for s in others]), self._ints(others))

    def step(self) -> None:
        """One token of every beam, and the next ones' choice: parents and
        next hold it.  Only calls that may be recorded into a HIP graph."""
        rt, r = self.rt, self.rows
        rt.beam_inputs(self.next, self.tokens_now, self.end_token)  # (a beam without one reads that, for nothing)
        rt.copy(self.positions, self.cache.lengths)
        self.cache.extend(self.seqs, self.ones)
        rt.gather_rows_f16(self.model.table, self.tokens_now, out=r.x)
        self._layers(r, self.positions, self.offsets, self.seqs)
        rt.quantize_rows(r.x, self.last8, norm=self.model.norm)
        rt.matmul_q8(self.model.head, self.last8, out=self.flat_logits)
        self.choice.select(self.logits, self.scores, self.parents, self.next, self.scores, ended=self.ended,
                           end_token=self.end_token, out_ended=self.ended)
        self.cache.reorder(self.seqs, self.flat_parents, self.beams)

    def answer(self, questions: Sequence[Sequence[int]], most: int) -> List[List[Tuple[List[int], float]]]:
        """For each question its beams, the best first: up to `most` tokens
        (without the one that ends them) and their log probability."""
        if most < 1:
            raise ValueError("answers of %d tokens" % most)
        if max(len(q) for q in questions) + most - 1 > self.tokens:
            raise ValueError("question and answer have more than %d tokens" % self.tokens)
        self.ask(questions)
        chosen = [(self.parents.download(), self.next.download())]
        for _ in range(most - 1):
            if (self.ended.download() | (chosen[-1][0] < 0)).all():
                break
            self.step()
            chosen.append((self.parents.download(), self.next.download()))
        scores = self.scores.download()
        out = []
        for g in range(self.questions):
            beams = []
            for b in range(self.beams):
                tokens, at = [], b
                for parents, nexts in reversed(chosen):
                    if at < 0:
                        break
                    tokens.append(int(nexts[g, at]))
                    at = int(parents[g, at])
                tokens = tokens[::-1]
                if self.end_token in tokens:
                    tokens = tokens[:tokens.index(self.end_token)]
                if np.isfinite(scores[g, b]):
                    beams.append((tokens, float(scores[g, b])))
            out.append(beams)
        return out

    def close(self) -> None:
        self.cache.close()
        self.rot.close()
        self.choice.close()


def random_model(rt: Runtime, rng, layers: int, vocab: int, width: int, q_heads: int, kv_heads: int, head_dim: int,
                 feed: int) -> Model:
    def weights(n, m, gain=1.0):
        return (gain * rng.standard_normal((n, m)) / np.sqrt(n)).astype(np.float32)

    def norm(n):
        return (1.0 + 0.1 * rng.standard_normal(n)).astype(np.float32)

    q, kv = q_heads * head_dim, kv_heads * head_dim
    blocks = [Block(rt, weights(width, q), weights(width, kv), weights(width, kv), weights(q, width),
                    weights(width, feed), weights(width, feed), weights(feed, width), norm(width), norm(width),
                    norm(head_dim), norm(head_dim)) for _ in range(layers)]
    return Model(rt, rng.standard_normal((vocab, width)), blocks, norm(width), weights(width, vocab, 3.0), q_heads,
                 kv_heads, head_dim)


def main() -> None:
    rng = np.random.default_rng(0)
    vocab = 2000
    with Runtime(0) as rt:
        model = random_model(rt, rng, 4, vocab, 384, 6, 6, 64, 1024)
        a = Answerer(rt, model, 3, 4, 128, end_token=2)
        questions = [rng.integers(3, vocab, n).tolist() for n in (40, 17, 80)]
        for g, beams in enumerate(a.answer(questions, 12)):
            print("question %d (%d tokens):" % (g, len(questions[g])))
            for tokens, score in beams:
                print("  %8.3f  %s" % (score, " ".join(map(str, tokens))))
        a.close()
        model.close()


if __name__ == "__main__":
    main()
