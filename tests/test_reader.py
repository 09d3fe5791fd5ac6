"""The reader's own account of its sequences, without a device: a step that the
cache refuses leaves it as it was, as the cache's."""
import numpy as np
import pytest

from manta_amd import _lib
from manta_amd.reader import PassageReader, random_layers


class _Array:
    def __init__(self, host, refuse=False):
        self.host, self.refuse = np.asarray(host), refuse
        self.shape, self.dtype = self.host.shape, self.host.dtype

    def download(self):
        if self.refuse:
            raise _lib.MantaRocmError(_lib.ERROR, "cache is out of pages: 2 needed, 0 free")
        return self.host


class _Device:
    """The calls that append makes, of a runtime and of its cache."""

    refuse = False
    longest = None

    def to_device(self, x):
        return _Array(x)

    def rotary(self, rot, positions, parts):
        self.positions = positions.host

    def extend(self, seqs, counts):
        pass

    def append(self, layer, k, v, offsets, seqs):
        return None

    def attention(self, layer, q, offsets, seqs, longest):
        self.longest = longest
        return _Array(q.host, self.refuse)


def test_a_refused_step_can_be_sent_again():
    rng = np.random.default_rng(0)
    r = PassageReader.__new__(PassageReader)
    r.rt = r.cache = _Device()
    r.layers, r.rot = random_layers(rng, 2, 16, 2, 1, 8), None
    r.q_heads, r.kv_heads, r.head_dim, r.passages, r.tokens = 2, 1, 8, 2, 50
    r.lengths = [10, 10, 10]
    rows = [rng.standard_normal((n, 16)) for n in (3, 5)]
    r.rt.refuse = True
    with pytest.raises(_lib.MantaRocmError, match="out of pages"):
        r.append([1, 2], rows)
    assert r.lengths == [10, 10, 10]
    r.rt.refuse = False
    assert [len(x) for x in r.append([1, 2], rows)] == [3, 5]
    assert r.lengths == [10, 13, 15] and r.rt.longest == 15
    assert list(r.rt.positions) == [10, 11, 12, 10, 11, 12, 13, 14]
