"""Passages read after a question: how the rotary and cache calls are used
together.  The question enters the cache once; every passage is a branch of it
(fork) that goes on in pages of its own; the branches are read as one ragged
batch, then step by step; the losers are released and the cache is compacted.

The model is a stack of attention layers with given projections, x + attention
(x), whose products run on the host: this module is about the calls between
them.  `python -m manta_amd.reader` ranks random passages.
"""
from __future__ import annotations

from typing import List, Sequence

import numpy as np

from .rocm import Runtime, rotary_freqs


class Layer:
    """q [width, q_heads * head_dim], k and v [width, kv_heads * head_dim],
    o [q_heads * head_dim, width], f32."""

    def __init__(self, q, k, v, o):
        self.q, self.k, self.v, self.o = (np.asarray(x, np.float32) for x in (q, k, v, o))


class PassageReader:
    """Reads passages after a question.  Sequence 0 is the question, 1 ..
    passages its branches."""

    def __init__(self, rt: Runtime, layers: Sequence[Layer], q_heads: int, kv_heads: int, head_dim: int, passages: int,
                 tokens: int, page_tokens: int = 16):
        """tokens: the most that a question, its passage and the steps after
        them have together."""
        self.rt, self.layers = rt, list(layers)
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        self.passages, self.tokens = passages, tokens
        each = (tokens + page_tokens - 1) // page_tokens
        self.cache = rt.cache(pages=(passages + 1) * each, kv_heads=kv_heads, head_dim=head_dim, seqs=passages + 1,
                              table_pages=each, page_tokens=page_tokens, layers=len(self.layers))
        self.rot = rt.rotary_bind(rotary_freqs(head_dim))
        self.lengths = [0] * (passages + 1)

    def _ints(self, x):
        return self.rt.to_device(np.asarray(x, np.int32))

    def _heads(self, x, w, heads):
        """Rows times a projection, in f16 on the device: [tokens, heads, head_dim]."""
        y = (x @ w).reshape(len(x), heads, self.head_dim)
        return self.rt.to_device(y.astype(np.float16).view(np.uint16))

    def append(self, seqs: Sequence[int], rows: Sequence[np.ndarray]) -> List[np.ndarray]:
        """Read new tokens of sequences: rows[i] f32 [n, width] of seqs[i].
        Returns their states after the last layer."""
        counts = [len(r) for r in rows]
        for s, n in zip(seqs, counts):
            if self.lengths[s] + n > self.tokens:
                raise ValueError("sequence %d of %d tokens cannot take %d more (at most %d)"
                                 % (s, self.lengths[s], n, self.tokens))
        offsets = np.concatenate([[0], np.cumsum(counts)])
        positions = np.concatenate([self.lengths[s] + np.arange(n) for s, n in zip(seqs, counts)])
        off, pos, sq = self._ints(offsets), self._ints(positions), self._ints(seqs)
        self.cache.extend(sq, self._ints(counts))  # once, for every layer
        lengths = list(self.lengths)
        for s, n in zip(seqs, counts):
            lengths[s] += n
        x = np.concatenate([np.asarray(r, np.float32) for r in rows])
        for i, w in enumerate(self.layers):
            q, k = self._heads(x, w.q, self.q_heads), self._heads(x, w.k, self.kv_heads)
            v = self._heads(x, w.v, self.kv_heads)
            self.rt.rotary(self.rot, pos, [(q, q), (k, k)])
            self.cache.append(i, k, v, off, sq)
            out = self.cache.attention(i, q, off, sq, longest=max(lengths))
            y = out.download().view(np.float16).astype(np.float32)
            x = x + y.reshape(len(x), -1) @ w.o
        self.lengths = lengths  # (a refused extend, reported by the downloads, has left the sequences as they were)
        return [x[a:b] for a, b in zip(offsets[:-1], offsets[1:])]

    def read(self, question: np.ndarray, passages: Sequence[np.ndarray], steps: Sequence[np.ndarray] = ()) -> np.ndarray:
        """The passages' last states, f32 [passages, width]: question [n,
        width], passages of any lengths, and then `steps` (f32 [width]), one
        token for all of them at a time."""
        if len(passages) != self.passages:
            raise ValueError("%d passages expected (got %d)" % (self.passages, len(passages)))
        self.cache.release(self._ints(range(self.passages + 1)))
        self.lengths = [0] * (self.passages + 1)
        self.append([0], [question])
        branches = list(range(1, self.passages + 1))
        self.cache.fork(self._ints([0] * self.passages), self._ints(branches))
        self.lengths = [self.lengths[0]] * (self.passages + 1)
        states = self.append(branches, passages)
        for token in steps:
            states = self.append(branches, [np.asarray(token)[None]] * self.passages)
        return np.stack([s[-1] for s in states])

    def keep(self, passages: Sequence[int]) -> int:
        """Release the question and every other passage's branch and move what
        is left together; returns its pages."""
        gone = [s for s in range(self.passages + 1) if s - 1 not in set(passages)]
        self.cache.release(self._ints(gone))
        for s in gone:
            self.lengths[s] = 0
        live = self.rt.empty((1,), np.int32)
        self.cache.compact(live)
        return int(live.download()[0])

    def close(self) -> None:
        self.cache.close()
        self.rot.close()


def random_layers(rng, count: int, width: int, q_heads: int, kv_heads: int, head_dim: int) -> List[Layer]:
    def weights(n, m):
        return rng.standard_normal((n, m)).astype(np.float32) / np.sqrt(n)

    return [Layer(weights(width, q_heads * head_dim), weights(width, kv_heads * head_dim),
                  weights(width, kv_heads * head_dim), weights(q_heads * head_dim, width)) for _ in range(count)]


def main() -> None:
    rng = np.random.default_rng(0)
    width, q_heads, kv_heads, d = 384, 6, 6, 64
    question = rng.standard_normal((40, width))
    passages = [rng.standard_normal((int(n), width)) for n in rng.integers(20, 200, 12)]
    label = rng.standard_normal(width)
    with Runtime(0) as rt:
        reader = PassageReader(rt, random_layers(rng, 4, width, q_heads, kv_heads, d), q_heads, kv_heads, d,
                               len(passages), 256)
        scores = reader.read(question, passages, [label] * 3) @ label
        order = np.argsort(-scores, kind="stable")
        for p in order[:5]:
            print("passage %2d (%3d tokens): %8.3f" % (p, len(passages[p]), scores[p]))
        print("the best three hold %d pages" % reader.keep([int(p) for p in order[:3]]))
        reader.close()


if __name__ == "__main__":
    main()
