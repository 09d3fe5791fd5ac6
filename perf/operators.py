"""The operators of a model that reads what was retrieved, and how they are
timed: rotary positions, a key/value cache of pages held in 8 bits (written,
read back and attended), and the bookkeeping of its pages (fork, extend,
release, compact, copy).

A case is a dict of plain values.  `op` says which call it is:

  rotary   Runtime.rotary: q and k of a batch of tokens, forward or backward
  append   Cache.append of new tokens, then Cache.read of the pages they entered
  attend   Cache.attention: queries that are the last tokens of their sequences
  fork     Cache.release, Cache.fork and Cache.extend: branches of a shared prefix
  compact  Runtime.copy of the tables' snapshot, then Cache.compact
  copy     Cache.copy_pages

With `own` false, `run` is the operator in elementary torch operations.

The cache, as both forms hold it: k codes int8 [layers, pages, heads, page, D],
v codes int8 [layers, pages, heads, D, page], and for each of them the largest
magnitude of a page's head, f32 [layers, pages, heads]; a code stands for
code * largest / 127.  The book is int32: refs [pages], lengths [seqs], tables
[seqs, table_pages] (-1 past a sequence's pages).
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False


def listed():
    return [
        # one step of a batch of sequences: q and k of one token each; latency
        {"name": "rotary_step_64", "op": "rotary", "tokens": 64, "q_heads": 32, "kv_heads": 8, "d": 128, "rot": 128,
         "layout": "half", "dtype": "f16", "scaling": "none", "backward": False, "far": 8192},
        # a prompt of passages, positions scaled for a long context
        {"name": "rotary_prompt_8192", "op": "rotary", "tokens": 8192, "q_heads": 32, "kv_heads": 8, "d": 128,
         "rot": 128, "layout": "half", "dtype": "bf16", "scaling": "blend", "backward": False, "far": 1000000},
        # the gradient of q and k where half of the head is rotated, in 32 bits; an odd token count
        {"name": "rotary_backward_5001", "op": "rotary", "tokens": 5001, "q_heads": 12, "kv_heads": 12, "d": 64,
         "rot": 32, "layout": "interleaved", "dtype": "f32", "scaling": "linear", "backward": True, "far": 5001},
        # one step of 64 sequences: a token each, most of them into pages partly filled
        {"name": "append_step_64", "op": "append", "seqs": 64, "new": 1, "kv_heads": 8, "d": 128, "page": 16,
         "dtype": "bf16", "longest": 2000},
        # prompts of 12 ragged sequences enter the cache
        {"name": "append_prompts_12", "op": "append", "seqs": 12, "new": 2048, "kv_heads": 8, "d": 128, "page": 64,
         "dtype": "f16", "longest": 4096},
        # a step of a few short sequences, as many kv heads as query heads (384 columns); latency
        {"name": "attend_step_4x1000", "op": "attend", "seqs": 4, "new": 1, "longest": 1000, "q_heads": 6,
         "kv_heads": 6, "d": 64, "page": 16, "dtype": "f16", "window": 0},
        # a step of a served batch, ragged
        {"name": "attend_step_64x8192", "op": "attend", "seqs": 64, "new": 1, "longest": 8192, "q_heads": 32,
         "kv_heads": 8, "d": 128, "page": 64, "dtype": "bf16", "window": 0},
        # a step of one sequence with a long context
        {"name": "attend_step_1x262145", "op": "attend", "seqs": 1, "new": 1, "longest": 262145, "q_heads": 32,
         "kv_heads": 8, "d": 128, "page": 64, "dtype": "bf16", "window": 0},
        # five tokens a sequence at once (a judge's few label tokens, drafted tokens), a sliding window
        {"name": "attend_tokens_16x5", "op": "attend", "seqs": 16, "new": 5, "longest": 16000, "q_heads": 48,
         "kv_heads": 8, "d": 96, "page": 32, "dtype": "f16", "window": 4096},
        # prompts: passages read after a cached question
        {"name": "attend_prompts_4x4096", "op": "attend", "seqs": 4, "new": 4096, "longest": 6000, "q_heads": 32,
         "kv_heads": 8, "d": 128, "page": 64, "dtype": "bf16", "window": 0},
        # 64 passages branch off two questions' caches, each going on in a page of its own
        {"name": "pages_fork_64", "op": "fork", "layers": 8, "pages": 256, "page": 32, "kv_heads": 8, "d": 128,
         "parents": 2, "children": 64, "longest": 1000},
        # after many sequences came and went: live pages move down into the holes
        {"name": "pages_compact_512", "op": "compact", "layers": 8, "pages": 512, "page": 32, "kv_heads": 8, "d": 128,
         "seqs": 24, "longest": 400},
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "rotary", "append", "append", "attend", "attend", "attend", "attend", "fork",
                     "compact", "copy"])
    d = rng.choice([64, 64, 128, 128, 32, 96, 192, 256])
    kv = rng.choice([1, 2, 4, 6, 8])
    page = rng.choice([16, 32, 64, 128])
    half = rng.choice(["f16", "bf16"])
    if op == "rotary":
        group = rng.choice([1, 2, 4, 5, 8])
        tokens = _log(rng, 1, max(1, min(32768, 8192 * 40 * 128 // (kv * (group + 1) * d * 2))))
        return {"op": op, "tokens": tokens, "q_heads": kv * group, "kv_heads": kv, "d": d,
                "rot": rng.choice([d, d, d // 2, 2 * rng.randint(1, d // 2)]),
                "layout": rng.choice(["half", "interleaved"]), "dtype": rng.choice([half, half, "f32"]),
                "scaling": rng.choice(["none", "linear", "base", "blend"]), "backward": rng.random() < 0.3,
                "far": _log(rng, tokens, 2000000)}
    if op == "append":
        seqs = _log(rng, 1, 128)
        new = 1 if rng.random() < 0.4 else _log(rng, 1, max(1, min(4096, 12 * 2048 * 1024 // (seqs * kv * d * 2))))
        return {"op": op, "seqs": seqs, "new": new, "kv_heads": kv, "d": d, "page": page, "dtype": half,
                "longest": new + _log(rng, 1, 2000)}
    if op == "attend":
        group = rng.choice([1, 2, 3, 4, 6, 8, 16])
        how = rng.choice(["step", "step", "tokens", "prompt"])
        window = rng.choice([0, 0, _log(rng, 16, 8192)])
        if how == "step":
            seqs, new = _log(rng, 1, 128), 1
            longest = _log(rng, 1, max(2, min(262144, 64 * 8192 * 1024 // (seqs * kv * d))))
        elif how == "tokens":
            seqs, new = _log(rng, 1, 32), rng.randint(2, 40)
            longest = new + _log(rng, 1, max(2, min(65536, 8 * 8192 * 1024 // (seqs * kv * d))))
        else:
            seqs, new = _log(rng, 1, 8), _log(rng, 41, 4096)
            new = min(new, max(41, int(math.sqrt(4 * 4096 * 4096 * 32 * 128 / (2 * seqs * kv * group * d)))))
            longest = new + _log(rng, 1, new)
        return {"op": op, "seqs": seqs, "new": new, "longest": longest, "q_heads": kv * group, "kv_heads": kv, "d": d,
                "page": page, "dtype": half, "window": window}
    layers = rng.choice([1, 2, 4, 8])
    page_bytes = layers * 2 * kv * page * d
    pages = _log(rng, 64, max(64, min(4096, (1 << 28) // page_bytes)))
    if op == "fork":
        parents, children = rng.randint(1, 4), _log(rng, 1, max(1, min(64, pages // 8)))
        longest = _log(rng, 1, max(1, min(4000, pages // 8 * page)))
        return {"op": op, "layers": layers, "pages": pages, "page": page, "kv_heads": kv, "d": d, "parents": parents,
                "children": children, "longest": longest}
    if op == "compact":
        seqs = _log(rng, 1, 64)
        return {"op": op, "layers": layers, "pages": pages, "page": page, "kv_heads": kv, "d": d, "seqs": seqs,
                "longest": max(1, page * pages // (2 * seqs) - 1)}
    return {"op": op, "layers": layers, "pages": pages, "page": page, "kv_heads": kv, "d": d,
            "count": _log(rng, 1, pages // 2)}


# ------------------------------------------------------------------- inputs

_DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"f16": 2, "bf16": 2, "f32": 4}


def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _gen(seed):
    g = torch.Generator(device=_device())
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype=torch.float32, sigma=1.0):
    out = torch.empty(shape, dtype=dtype, device=g.device)
    flat = out.view(-1)
    step = 1 << 27
    for a in range(0, flat.numel(), step):
        b = min(flat.numel(), a + step)
        flat[a:b] = torch.randn((b - a,), generator=g, device=g.device) * sigma
    return out


def _codes(g, shape):
    """Codes of normal values whose largest stands at 127 or so."""
    out = torch.empty(shape, dtype=torch.int8, device=g.device)
    flat = out.view(-1)
    step = 1 << 27
    for a in range(0, flat.numel(), step):
        b = min(flat.numel(), a + step)
        flat[a:b] = (torch.randn((b - a,), generator=g, device=g.device) * 38).round_().clamp_(-127, 127)
    return out


def _largest(g, shape):
    return 2.5 + 2.0 * torch.rand(shape, generator=g, device=g.device)


def _lengths(case):
    """Ragged lengths from about a third of the longest up to it, the first
    one the longest, and new tokens a sequence the same way; host lists, the
    same for every seed (the outputs' shapes follow from them)."""
    rng = np.random.default_rng([case["seqs"], case["longest"]])
    n, longest, new = case["seqs"], case["longest"], case.get("new", 0)
    news = [new] + [int(x) for x in rng.integers(max(1, new // 3), new + 1, n - 1)] if new > 5 else [new] * n
    lens = [longest] + [int(x) for x in rng.integers(max(1, longest // 3), longest + 1, n - 1)]
    return [max(a, b) for a, b in zip(lens, news)], news


def _book(lengths, page, pages, rng, spare_seqs=0, table_pages=None):
    """Tables of random distinct pages: (refs, lengths, tables) as int32 arrays."""
    counts = [(x + page - 1) // page for x in lengths]
    table_pages = table_pages or max(counts)
    order = rng.permutation(pages)
    tables = np.full((len(lengths) + spare_seqs, table_pages), -1, np.int32)
    refs = np.zeros((pages,), np.int32)
    at = 0
    for i, c in enumerate(counts):
        tables[i, :c] = order[at:at + c]
        at += c
    refs[order[:at]] = 1
    return refs, np.array(list(lengths) + [0] * spare_seqs, np.int32), tables


def _inputs(case, seed):
    """The call's inputs as tensors and host arrays, from the seed alone."""
    g = _gen(seed)
    rng = np.random.default_rng([seed, 5])
    op, d = case["op"], case["d"]
    kv = case["kv_heads"]
    if op == "rotary":
        t, dt = case["tokens"], _DTYPE[case["dtype"]]
        return {"q": _normal(g, (t, case["q_heads"], d), dt), "k": _normal(g, (t, kv, d), dt),
                "pos": torch.randint(0, case["far"], (t,), generator=g, device=g.device, dtype=torch.int32)}
    page = case["page"]
    if op in ("append", "attend"):
        lengths, news = _lengths(case)
        pages = sum((x + page - 1) // page for x in lengths) + 3
        refs, lens, tables = _book(lengths, page, pages, rng)
        x = {"refs": refs, "lengths": lens, "tables": tables, "news": news, "layers": 1, "pages": pages,
             "k_codes": _codes(g, (1, pages, kv, page, d)), "v_codes": _codes(g, (1, pages, kv, d, page)),
             "k_max": _largest(g, (1, pages, kv)), "v_max": _largest(g, (1, pages, kv))}
        t, dt = sum(news), _DTYPE[case["dtype"]]
        if op == "append":
            x["k"], x["v"] = _normal(g, (t, kv, d), dt), _normal(g, (t, kv, d), dt)
        else:
            x["q"] = _normal(g, (t, case["q_heads"], d), dt, 2.0)
        return x
    layers, pages = case["layers"], case["pages"]
    x = {"layers": layers, "pages": pages, "k_codes": _codes(g, (layers, pages, kv, page, d)),
         "v_codes": _codes(g, (layers, pages, kv, d, page)), "k_max": _largest(g, (layers, pages, kv)),
         "v_max": _largest(g, (layers, pages, kv))}
    if op == "fork":
        n, m, longest = case["parents"], case["children"], case["longest"]
        lengths = [int(v) for v in rng.integers(max(1, longest // 2), longest + 1, n)]
        x["refs"], x["lengths"], x["tables"] = _book(lengths, page, pages, rng, m, (longest + page - 1) // page + 1)
        x["from"] = np.array([i % n for i in range(m)], np.int32)
        x["to"] = np.arange(n, n + m, dtype=np.int32)
        x["counts"] = np.ones((m,), np.int32)
    elif op == "compact":
        n, longest = case["seqs"], case["longest"]
        lengths = [int(v) for v in rng.integers(max(1, longest // 2), longest + 1, n)]
        x["refs"], x["lengths"], x["tables"] = _book(lengths, page, pages, rng, 0, (longest + page - 1) // page)
    else:
        order = rng.permutation(pages).astype(np.int32)
        x["src"], x["dst"] = order[:case["count"]].copy(), order[case["count"]:2 * case["count"]].copy()
        x["refs"], x["lengths"], x["tables"] = (np.ones((pages,), np.int32), np.zeros((1,), np.int32),
                                                np.full((1, 1), -1, np.int32))
    return x


# ------------------------------------------------------- the call and its state

_RT = None
_FULL = {"none": {}, "linear": {"factor": 4.0}, "base": {"factor": 8.0},
         "blend": {"factor": 8.0, "low": 1.0, "high": 4.0, "original": 8192.0}}
_BASE = 10000.0


def _frequencies(case):
    """Radians a token for each pair, in 64 bits."""
    rot, how = case["rot"], _FULL[case["scaling"]]
    p = np.arange(rot // 2, dtype=np.float64)
    base = _BASE
    if case["scaling"] == "base" and rot > 2:
        base *= how["factor"] ** (rot / (rot - 2))
    f = base ** (-2.0 * p / rot)
    if case["scaling"] == "linear":
        f = f / how["factor"]
    elif case["scaling"] == "blend":
        turns = how["original"] * f / (2.0 * math.pi)
        mix = np.clip((turns - how["low"]) / (how["high"] - how["low"]), 0.0, 1.0)
        f = f * ((1.0 - mix) / how["factor"] + mix)
    return f


def _magnitude(case):
    return 0.1 * math.log(_FULL["blend"]["factor"]) + 1.0 if case["scaling"] == "blend" else 1.0


def _offsets(news):
    return np.concatenate([[0], np.cumsum(news)]).astype(np.int32)


def _touched(lengths, news, page):
    """Tokens from the start of the first page that a sequence's new tokens
    enter: all of the cache that an append may change."""
    return [n + (int(v) - n) % page for v, n in zip(lengths, news)]


class _Memory:
    """A device array of the framework as torch sees it."""

    def __init__(self, array, typestr):
        self.array = array
        self.__cuda_array_interface__ = {"shape": array.shape, "typestr": typestr, "data": (array.addr, False),
                                         "version": 3}


_NUMPY = {torch.float32: ("<f4", np.float32), torch.float16: ("<i2", np.uint16), torch.bfloat16: ("<i2", np.uint16),
          torch.int8: ("|i1", np.int8), torch.int32: ("<i4", np.int32)}


def _view(array, dtype):
    t = torch.as_tensor(_Memory(array, _NUMPY[dtype][0]), device="cuda")
    return t.view(dtype) if dtype in (torch.float16, torch.bfloat16) else t


def _empty(rt, shape, dtype):
    """A device array of the framework and torch's view of it."""
    a = rt.empty(shape, _NUMPY[dtype][1])
    return a, _view(a, dtype)


def _put(rt, tensor):
    if isinstance(tensor, np.ndarray):
        return rt.to_device(tensor)
    a, v = _empty(rt, tuple(tensor.shape), tensor.dtype)
    v.copy_(tensor)
    return a


def _prepare_own(case, x):
    global _RT
    from manta_amd import rocm

    if _RT is None:
        _RT = rocm.Runtime(0)
    rt = _RT
    op = case["op"]
    s = {"case": case, "rt": rt}
    if op == "rotary":
        how = _FULL[case["scaling"]]
        f = rocm.rotary_freqs(case["rot"], base=_BASE, scaling=case["scaling"], **how)
        s["rot"] = rt.rotary_bind(f, layout=case["layout"], magnitude=_magnitude(case))
        dt = _DTYPE[case["dtype"]]
        s["pos"] = _put(rt, x["pos"])
        s["q"], s["k"] = _put(rt, x["q"]), _put(rt, x["k"])
        s["q_out"], qv = _empty(rt, x["q"].shape, dt)
        s["k_out"], kv = _empty(rt, x["k"].shape, dt)
        s["parts"] = [(s["q"], s["q_out"]), (s["k"], s["k_out"])]
        s["out"] = {"q": qv, "k": kv}
        torch.cuda.synchronize()
        return s
    seqs, table_pages = x["tables"].shape
    c = rt.cache(layers=x["layers"], pages=x["pages"], page_tokens=case["page"], kv_heads=case["kv_heads"],
                 head_dim=case["d"], seqs=seqs, table_pages=table_pages)
    s["cache"] = c
    views = {}
    for name, dt in (("k_codes", torch.int8), ("v_codes", torch.int8), ("k_max", torch.float32),
                     ("v_max", torch.float32)):
        views[name] = _view(getattr(c, name), dt)
        views[name].copy_(x[name])
    book = np.concatenate([x["refs"], x["lengths"], x["tables"].ravel()])
    views["book"] = _view(c.book, torch.int32)
    views["book"].copy_(torch.from_numpy(book))
    if op in ("append", "attend"):
        s["offsets"] = rt.to_device(_offsets(x["news"]))
        dt = _DTYPE[case["dtype"]]
        if op == "append":
            s["k"], s["v"] = _put(rt, x["k"]), _put(rt, x["v"])
            tail = _touched(x["lengths"], x["news"], case["page"])
            s["tail"] = rt.to_device(_offsets(tail))
            shape = (sum(tail), case["kv_heads"], case["d"])
            s["k_out"], kv = _empty(rt, shape, torch.float32)
            s["v_out"], vv = _empty(rt, shape, torch.float32)
            s["out"] = {"k": kv, "v": vv}
        else:
            s["q"] = _put(rt, x["q"])
            s["o"], ov = _empty(rt, tuple(x["q"].shape), dt)
            s["lse"], lv = _empty(rt, tuple(x["q"].shape[:2]), torch.float32)
            s["out"] = {"out": ov, "lse": lv}
    elif op == "fork":
        for name in ("from", "to", "counts"):
            s[name] = rt.to_device(x[name])
        s["out"] = views
    elif op == "compact":
        s["saved"] = rt.to_device(book)
        s["live"], lv = _empty(rt, (1,), torch.int32)
        s["out"] = dict(views, live=lv)
    else:
        s["src"], s["dst"] = rt.to_device(x["src"]), rt.to_device(x["dst"])
        s["out"] = {n: views[n] for n in ("k_codes", "v_codes", "k_max", "v_max")}
    torch.cuda.synchronize()
    return s


def prepare(case, seed):
    x = _inputs(case, seed)
    if own:
        return _prepare_own(case, x)
    dev = _device()
    s = {"case": case, "x": x}
    if case["op"] == "rotary":
        s["freqs"] = torch.from_numpy(_frequencies(case)).to(dev)
        return s
    s["tables"] = [list(map(int, r)) for r in x["tables"]]
    if case["op"] in ("append", "attend"):
        page = case["page"]
        s["rows"] = [torch.tensor(t[:(int(n) + page - 1) // page], device=dev)
                     for t, n in zip(s["tables"], x["lengths"])]
    elif case["op"] == "copy":
        s["src"], s["dst"] = torch.from_numpy(x["src"]).long().to(dev), torch.from_numpy(x["dst"]).long().to(dev)
    else:
        for name in ("refs", "lengths", "tables"):
            s[name] = torch.from_numpy(x[name]).to(dev)
        s["saved"] = [s[n].clone() for n in ("refs", "lengths", "tables")]
        if case["op"] == "fork":
            s["from"], s["to"] = torch.from_numpy(x["from"]).long().to(dev), torch.from_numpy(x["to"]).long().to(dev)
            s["counts"] = torch.from_numpy(x["counts"]).to(dev)
    return s


def run(s):
    return _run_own(s) if own else _PLAIN[s["case"]["op"]](s)


def _run_own(s):
    case, op = s["case"], s["case"]["op"]
    if op == "rotary":
        s["rt"].rotary(s["rot"], s["pos"], s["parts"], inverse=case["backward"], dtype=case["dtype"])
        return s["out"]
    c = s["cache"]
    if op == "append":
        c.append(0, s["k"], s["v"], s["offsets"], dtype=case["dtype"])
        c.read(0, s["tail"], s["k_out"], s["v_out"], dtype="f32")
    elif op == "attend":
        c.attention(0, s["q"], s["offsets"], out=s["o"], lse=s["lse"], scale=1.0 / math.sqrt(case["d"]), causal=True,
                    window=case["window"], longest=case["longest"], dtype=case["dtype"])
    elif op == "fork":
        c.release(s["to"])
        c.fork(s["from"], s["to"])
        c.extend(s["to"], s["counts"])
    elif op == "compact":
        s["rt"].copy(c.book, s["saved"])
        c.compact(s["live"])
    else:
        c.copy_pages(s["src"], s["dst"])
    return s["out"]


# ------------------------------------------------------------ the plain forms

def _rotate(x, cos, sin, case):
    rot = case["rot"]
    y = x.float()
    if case["layout"] == "half":
        a, b, rest = y[..., :rot // 2], y[..., rot // 2:rot], y[..., rot:]
    else:
        a, b, rest = y[..., 0:rot:2], y[..., 1:rot:2], y[..., rot:]
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat([a, b], -1) if case["layout"] == "half" else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([turned, rest], -1).to(x.dtype)


def _plain_rotary(s):
    case, x = s["case"], s["x"]
    angle = x["pos"].double()[:, None, None] * s["freqs"]  # far positions: 32 bits lose the angle
    m = _magnitude(case)
    cos, sin = (torch.cos(angle) * m).float(), (torch.sin(angle) * m).float()
    if case["backward"]:
        sin = -sin
    return {"q": _rotate(x["q"], cos, sin, case), "k": _rotate(x["k"], cos, sin, case)}


def _quantise(codes, old, new, filled):
    """One page's head(s): codes int8 [H, page, D] of which `filled` tokens
    stand for code * old / 127, and new tokens [H, n, D]: the page's largest
    and its codes.  A magnitude below the smallest normal number counts as 0."""
    if filled:
        largest = torch.maximum(old, new.abs().amax((1, 2)))
        keep = codes[:, :filled].float() * old[:, None, None] / largest.clamp(min=2.0 ** -126)[:, None, None]
        keep = torch.where((largest > old)[:, None, None], keep.round(), codes[:, :filled].float())
    else:
        largest, keep = new.abs().amax((1, 2)), codes[:, :0].float()
    tiny = largest < 2.0 ** -126
    fresh = new * 127.0 / largest.clamp(min=2.0 ** -126)[:, None, None]
    out = torch.cat([keep, fresh.round().clamp(-127, 127)], 1)
    return torch.where(tiny[:, None, None], torch.zeros_like(out), out), torch.where(tiny, 0.0, largest)


def _plain_append(s):
    case, x = s["case"], s["x"]
    page, at = case["page"], 0
    out_k, out_v = [], []
    for i, n in enumerate(x["news"]):
        length = int(x["lengths"][i])
        k, v = x["k"][at:at + n].float().transpose(0, 1), x["v"][at:at + n].float().transpose(0, 1)
        at += n
        t, done = length - n, 0
        while done < n:
            p, f = s["tables"][i][t // page], t % page
            c = min(page - f, n - done)
            codes, big = _quantise(x["k_codes"][0, p], x["k_max"][0, p], k[:, done:done + c], f)
            x["k_codes"][0, p, :, :f + c], x["k_max"][0, p] = codes.to(torch.int8), big
            codes, big = _quantise(x["v_codes"][0, p].transpose(1, 2), x["v_max"][0, p], v[:, done:done + c], f)
            x["v_codes"][0, p, :, :, :f + c], x["v_max"][0, p] = codes.transpose(1, 2).to(torch.int8), big
            t, done = t + c, done + c
        first = (length - n) // page
        rows, f = s["rows"][i][first:], length - first * page
        k = x["k_codes"][0][rows].float() * x["k_max"][0][rows][..., None, None] / 127.0
        v = x["v_codes"][0][rows].float() * x["v_max"][0][rows][..., None, None] / 127.0
        out_k.append(k.transpose(1, 2).flatten(0, 1)[:f])
        out_v.append(v.permute(0, 3, 1, 2).flatten(0, 1)[:f])
    return {"k": torch.cat(out_k), "v": torch.cat(out_v)}


def _plain_attend(s):
    case, x = s["case"], s["x"]
    kv, d, page = case["kv_heads"], case["d"], case["page"]
    group = case["q_heads"] // kv
    scale = 1.0 / math.sqrt(d)
    outs, lses, at = [], [], 0
    for i, n in enumerate(x["news"]):
        length, rows = int(x["lengths"][i]), s["rows"][i]
        k = x["k_codes"][0][rows].float() * (x["k_max"][0][rows] / 127.0)[..., None, None]
        v = x["v_codes"][0][rows].float() * (x["v_max"][0][rows] / 127.0)[..., None, None]
        k = k.permute(1, 3, 0, 2).reshape(kv, d, -1)[..., :length].contiguous()
        v = v.permute(1, 0, 3, 2).reshape(kv, -1, d)[:, :length].contiguous()
        q = x["q"][at:at + n].float().view(n, kv, group, d).permute(1, 2, 0, 3).reshape(kv, group * n, d).contiguous()
        at += n
        pos = torch.arange(length - n, length, device=q.device)[:, None]
        t = torch.arange(length, device=q.device)[None, :]
        hidden = t > pos
        if case["window"]:
            hidden = hidden | (t <= pos - case["window"])
        heads = max(1, min(kv, (1 << 28) // max(1, group * n * length)))
        o, l = [], []
        for a in range(0, kv, heads):
            sc = torch.matmul(q[a:a + heads], k[a:a + heads]) * scale
            sc = sc.view(-1, group, n, length).masked_fill_(hidden, float("-inf")).view(sc.shape)
            top = sc.amax(-1, keepdim=True)
            sc = (sc - top).exp_()
            total = sc.sum(-1, keepdim=True)
            o.append(torch.matmul(sc, v[a:a + heads]) / total)
            l.append((top + total.log())[..., 0])
        outs.append(torch.cat(o).view(kv, group, n, d).permute(2, 0, 1, 3).reshape(n, kv * group, d))
        lses.append(torch.cat(l).view(kv, group, n).permute(2, 0, 1).reshape(n, kv * group))
    return {"out": torch.cat(outs).to(x["q"].dtype), "lse": torch.cat(lses)}


_POOL = ("k_codes", "v_codes", "k_max", "v_max")


def _move(x, src, dst):
    for name in _POOL:
        x[name][:, dst] = x[name][:, src]


def _book_of(s):
    return torch.cat([s["refs"], s["lengths"], s["tables"].view(-1)])


def _count(refs, entries, by):
    refs.index_add_(0, entries.long(), torch.full_like(entries, by))


def _plain_fork(s):
    case, x = s["case"], s["x"]
    page, refs, lengths, tables = case["page"], s["refs"], s["lengths"], s["tables"]
    src, dst = s["from"], s["to"]
    held = tables[dst]
    _count(refs, held[held >= 0], -1)  # release
    tables[dst] = tables[src]  # fork
    lengths[dst] = lengths[src]
    held = tables[dst]
    _count(refs, held[held >= 0], 1)
    first = lengths[dst].long()  # extend
    col = (first + page - 1) // page
    more = (first + s["counts"] + page - 1) // page - col  # 0 or 1: one token each
    inside = first % page != 0
    last = tables[dst, (col - 1).clamp(min=0)].long()
    shared = inside & (refs[last] > 1)
    free = torch.nonzero(refs == 0)[:, 0]
    need = shared.long() + more
    rank = torch.cumsum(need, 0) - need
    fresh = free[rank.clamp(max=free.numel() - 1)]
    rows, cols = dst[shared], col[shared] - 1
    old, new = last[shared], fresh[shared]
    tables[rows, cols] = new.int()
    _count(refs, old.int(), -1)
    refs[new] = 1
    _move(x, old, new)
    grown = more > 0
    tables[dst[grown], col[grown]] = fresh[grown].int()
    refs[fresh[grown]] = 1
    lengths[dst] = lengths[dst] + s["counts"]
    return dict({n: x[n] for n in _POOL}, book=_book_of(s))


def _plain_compact(s):
    x = s["x"]
    for name, saved in zip(("refs", "lengths", "tables"), s["saved"]):
        s[name].copy_(saved)
    refs, tables = s["refs"], s["tables"]
    live = (refs > 0).sum()
    number = torch.arange(refs.numel(), device=refs.device)
    src, dst = number[(refs > 0) & (number >= live)], number[(refs == 0) & (number < live)]
    _move(x, src, dst)
    refs[dst] = refs[src]
    refs[src] = 0
    number[src] = dst
    s["tables"] = torch.where(tables >= 0, number[tables.clamp(min=0).long()].int(), tables)
    return dict({n: x[n] for n in _POOL}, book=_book_of(s), live=live.int().view(1))


def _plain_copy(s):
    _move(s["x"], s["src"], s["dst"])
    return {n: s["x"][n] for n in _POOL}


_PLAIN = {"rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend, "fork": _plain_fork,
          "compact": _plain_compact, "copy": _plain_copy}


# ------------------------------------------------------------ what it costs

def work(case):
    op, d, kv = case["op"], case["d"], case["kv_heads"]
    if op == "rotary":
        elements = case["tokens"] * (case["q_heads"] + kv) * d
        return {"bytes": 2 * elements * _BYTES[case["dtype"]] + 4 * case["tokens"],
                "flops": 6 * case["tokens"] * (case["q_heads"] + kv) * case["rot"] // 2}
    page = case["page"]
    if op in ("append", "attend"):
        lengths, news = _lengths(case)
    if op == "append":
        tokens = sum(news)
        back = sum(_touched(lengths, news, page))  # read back: a byte in, four out
        return {"bytes": 2 * kv * d * (tokens * (_BYTES[case["dtype"]] + 1) + 5 * back),
                "flops": 2 * 2 * kv * d * tokens}
    if op == "attend":
        rows = keys = 0
        for v, n in zip(lengths, news):
            w = case["window"] or v
            rows += sum(min(w, p + 1) for p in range(v - n, v)) if n <= 40 else _pairs(v, n, w)
            keys += min(v, w + n - 1)
        size = 2 * _BYTES[case["dtype"]] * sum(news) * case["q_heads"] * d + 4 * sum(news) * case["q_heads"]
        return {"bytes": 2 * keys * kv * d + size, "flops": 4 * rows * case["q_heads"] * d}
    page_bytes = case["layers"] * 2 * kv * (page * d + 4)
    if op == "fork":
        return {"bytes": 2 * case["children"] * page_bytes, "flops": 0}
    if op == "compact":
        # each page is live or not by chance: live * (1 - live / pages) of them lie above the rest
        live = min(case["pages"], case["seqs"] * (3 * case["longest"] / 4 + page / 2) / page)
        return {"bytes": int(2 * live * (1 - live / case["pages"]) * page_bytes), "flops": 0}
    return {"bytes": 2 * case["count"] * page_bytes, "flops": 0}


def _pairs(length, new, window):
    """Sum of min(window, p + 1) for p from length - new to length - 1."""
    p = np.arange(length - new, length, dtype=np.int64)
    return int(np.minimum(window, p + 1).sum())


# ------------------------------------------------------------ in 64 bits

def _exact_rotary(case, x):
    f = _frequencies(case)
    angle = x["pos"].double()[:, None] * torch.from_numpy(f).to(x["pos"].device)[None]
    c = torch.polar(torch.full_like(angle, _magnitude(case)), -angle if case["backward"] else angle)[:, None]
    out = {}
    for name in ("q", "k"):
        y = x[name].double().clone()
        r = y[..., :case["rot"]]
        if case["layout"] == "half":
            z = torch.complex(*(v.contiguous() for v in r.chunk(2, -1))) * c
            y[..., :case["rot"]] = torch.cat([z.real, z.imag], -1)
        else:
            z = torch.view_as_complex(r.reshape(*r.shape[:-1], -1, 2).contiguous()) * c
            y[..., :case["rot"]] = torch.view_as_real(z).flatten(-2)
        out[name] = y
    return out


def _exact_append(case, x):
    """The pages that new tokens entered, from the definition."""
    page, out = case["page"], {"k": [], "v": []}
    starts = _offsets(x["news"])
    for i, n in enumerate(x["news"]):
        length = int(x["lengths"][i])
        for first in range((length - n) // page * page, length, page):
            p = int(x["tables"][i][first // page])
            old = max(0, length - n - first)  # tokens of the page that were there before
            a, b = first + old - (length - n), min(first + page, length) - (length - n)
            for name in ("k", "v"):
                codes = x[name + "_codes"][0, p].double()
                codes = (codes if name == "k" else codes.transpose(1, 2))[:, :old]
                was = x[name + "_max"][0, p].double()[:, None, None]
                new = x[name][starts[i] + a:starts[i] + b].double().transpose(0, 1)
                largest = new.abs().amax((1, 2), keepdim=True)
                if old:
                    largest = torch.maximum(largest, was)
                kept = torch.where(largest > was, torch.round(codes * was / largest), codes)
                both = torch.cat([kept, torch.round(new * 127.0 / largest)], 1) * largest / 127.0
                out[name].append(both.transpose(0, 1))
    return {name: torch.cat(v) for name, v in out.items()}


def _exact_attend(case, x):
    if work(case)["flops"] > 4e12:
        return None
    kv, d, page = case["kv_heads"], case["d"], case["page"]
    group = case["q_heads"] // kv
    out = torch.zeros(x["q"].shape, dtype=torch.float64, device=x["q"].device)
    lse = torch.zeros(x["q"].shape[:2], dtype=torch.float64, device=x["q"].device)
    starts = _offsets(x["news"])
    for i, n in enumerate(x["news"]):
        length = int(x["lengths"][i])
        rows = torch.from_numpy(x["tables"][i][:(length + page - 1) // page]).long().to(out.device)
        pos = torch.arange(length - n, length, device=out.device)
        t = torch.arange(length, device=out.device)
        seen = t[None, :] <= pos[:, None]
        if case["window"]:
            seen &= t[None, :] > pos[:, None] - case["window"]
        for h in range(kv):
            keys = x["k_codes"][0, rows, h].double() * x["k_max"][0, rows, h].double()[:, None, None] / 127.0
            vals = x["v_codes"][0, rows, h].double() * x["v_max"][0, rows, h].double()[:, None, None] / 127.0
            keys = keys.reshape(-1, d)[:length].t().contiguous()
            vals = vals.transpose(1, 2).reshape(-1, d)[:length].contiguous()
            for j in range(h * group, (h + 1) * group):
                q = x["q"][starts[i]:starts[i + 1], j].double()
                sc = torch.where(seen, (q @ keys) / math.sqrt(d), -math.inf)
                lse[starts[i]:starts[i + 1], j] = torch.logsumexp(sc, -1)
                out[starts[i]:starts[i + 1], j] = torch.softmax(sc, -1) @ vals
    return {"out": out, "lse": lse}


def exact(case, seed):
    op = case["op"]
    if op not in ("rotary", "append", "attend"):
        return None
    x = _inputs(case, seed)
    return {"rotary": _exact_rotary, "append": _exact_append, "attend": _exact_attend}[op](case, x)
