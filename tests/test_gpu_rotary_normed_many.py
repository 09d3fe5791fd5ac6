"""Normed rotation of prompts: several tokens a workgroup (2, 4 and 8, from
2048, 4096 and 8192 tokens on) with a ragged last run, heads that run over them,
and results past 32 MB, which are written past the caches."""
import numpy as np
import pytest

from cache_oracle import from_bits, to_bits
from decode_oracle import rotary_normed, rounding
from manta_amd import rocm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,d,rot,dtype", [
    (2049, (3, 1), 64, 64, "f32"), (5001, (2, 1, 2), 64, 32, "bf16"), (8195, (1, 2), 64, 64, "f16"),  # whole pieces
    (2048, (3,), 80, 50, "bf16"), (5003, (2, 1), 80, 50, "f32"), (8199, (1, 1, 1), 47, 40, "f16"),    # shared ones
    (2051, (2, 1), 20, 4, "f32"), (4098, (3, 1), 33, 22, "bf16"), (8193, (2, 1), 24, 16, "f16"),      # short ones
    (3000, (1, 1), 256, 2, "f32"),                                                                    # two a lane
    (8195, (12, 5), 64, 64, "f32"), (16400, (12, 4, 1), 64, 32, "bf16")])                             # past 32 MB
def test_prompts(rt, tokens, heads, d, rot, dtype, layout):
    print("rotary_normed many", tokens, heads, d, rot, dtype, layout, flush=True)
    rng = np.random.default_rng(tokens + d)
    freqs, pos = rocm.rotary_freqs(rot), rng.integers(0, 1000000, tokens)
    r, p = rt.rotary_bind(freqs, layout=layout), rt.to_device(pos.astype(np.int32))
    parts, norms, hosts = [], [], []
    for i, h in enumerate(heads):
        bits = to_bits(rng.standard_normal((tokens, h, d)), dtype)
        a = rt.to_device(bits)
        parts.append((a, a if i % 2 else rt.to_device(np.zeros_like(bits))))  # every second in place
        norms.append(rng.uniform(-2, 2, d).astype(np.float32) if i != 2 else None)
        hosts.append(from_bits(bits, dtype))
    rt.rotary_normed(r, p, parts, [None if w is None else rt.to_device(w) for w in norms], eps=1e-5, dtype=dtype)
    for x, w, (_, out) in zip(hosts, norms, parts):
        got = from_bits(out.download(), dtype)
        for t0 in range(0, tokens, 4000):
            t = slice(t0, t0 + 4000)
            want, off = rotary_normed(x[t], w, 1e-5, pos[t], freqs, layout, 1.0)
            bad = ~(np.abs(got[t] - want) <= off + rounding(np.abs(want) + off, dtype))
            assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4] + [t0, 0, 0], got[t][bad][:4], want[bad][:4])
        if w is None:  # what is not normed is rotary's, bit for bit
            b = rt.to_device(to_bits(x, dtype))
            rt.rotary(r, p, [(b, b)], dtype=dtype)
            np.testing.assert_array_equal(from_bits(b.download(), dtype), got)
