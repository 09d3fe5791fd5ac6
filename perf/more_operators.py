"""The operators of a step that writes an answer, and how they are timed:
products in 8 bits with a scale for each token and each output column, gated or
not, norms of queries and keys with their rotation, the choice of the next
beams, and the cache's sequences following it.

A case is a dict of plain values.  `op` says which calls it is:

  product  Runtime.quantize_rows (with or without an RMS norm), then
           Runtime.matmul_q8 (with or without what is added to its result)
  gated    the same with a gated weight: act(x G) * (x U)
  rotary   Runtime.rotary_normed: q and k of a batch of tokens
  beams    Beams.select: the best continuations of every group's beams
  reorder  Runtime.copy of the tables' snapshot, then Cache.reorder

With `own` false, `run` is the operator in elementary torch operations.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False


def listed():
    return [
        # q, k and v of one step of twelve passages, the width and heads of the
        # reader's example (384 columns); latency
        {"name": "product_step_12x384", "op": "product", "rows": 12, "k": 384, "n": 1152, "norm": True, "add": False,
         "dtype": "f16"},
        # one step of a batch of sequences: the residual's norm, then q, k and v
        # of 32 query and 8 kv heads of 128
        {"name": "product_step_16x4096", "op": "product", "rows": 16, "k": 4096, "n": 6144, "norm": True, "add": False,
         "dtype": "bf16"},
        # prompts of passages: attention's output projection onto the residual
        {"name": "product_prompt_8192", "op": "product", "rows": 8192, "k": 4096, "n": 4096, "norm": False,
         "add": True, "dtype": "bf16"},
        # the feed-forward block of one step
        {"name": "gated_step_48", "op": "gated", "rows": 48, "k": 4096, "n": 12288, "norm": True, "gate": "silu",
         "dtype": "f16"},
        # ... and of a ragged batch of prompts
        {"name": "gated_prompt_3001", "op": "gated", "rows": 3001, "k": 4096, "n": 12288, "norm": True,
         "gate": "gelu", "dtype": "bf16"},
        # one step of a batch of sequences: q and k of one token each; latency
        {"name": "rotary_normed_step_64", "op": "rotary", "tokens": 64, "q_heads": 32, "kv_heads": 8, "d": 128,
         "rot": 128, "layout": "half", "dtype": "f16", "far": 8192},
        # a prompt of passages at the positions of a long context
        {"name": "rotary_normed_prompt_8192", "op": "rotary", "tokens": 8192, "q_heads": 32, "kv_heads": 8, "d": 128,
         "rot": 128, "layout": "half", "dtype": "bf16", "far": 1000000},
        # half of the head rotated, in 32 bits; an odd token count
        {"name": "rotary_normed_5001", "op": "rotary", "tokens": 5001, "q_heads": 12, "kv_heads": 12, "d": 64,
         "rot": 32, "layout": "interleaved", "dtype": "f32", "far": 5001},
        # a question's four beams; latency
        {"name": "beams_1x4", "op": "beams", "groups": 1, "beams": 4, "vocab": 32000, "k": 8, "dtype": "f16",
         "ended": False},
        # many questions at once, logits in 32 bits, an odd vocabulary, some beams ended
        {"name": "beams_64x8", "op": "beams", "groups": 64, "beams": 8, "vocab": 130001, "k": 16, "dtype": "f32",
         "ended": True},
        # the same step's caches: 16 questions of 4 beams
        {"name": "reorder_16x4", "op": "reorder", "groups": 16, "beams": 4, "shared": 1000, "longest": 1500,
         "page": 64},
        # long contexts, small pages: a question's 16 beams go on from one of 100,000 tokens
        {"name": "reorder_8x16_long", "op": "reorder", "groups": 8, "beams": 16, "shared": 100000, "longest": 104000,
         "page": 16},
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["product", "product", "product", "gated", "gated", "rotary", "rotary", "beams", "beams",
                     "reorder"])
    if op in ("product", "gated"):
        k, n = _log(rng, 40, 16384), _log(rng, 24, 16384)
        if rng.random() < 0.6:  # widths of models: whole runs of 64 columns
            k, n = max(64, k // 64 * 64), max(64, n // 64 * 64)
        most = 8192 * 4096 * 4096 // (k * n * (2 if op == "gated" else 1))
        rows = rng.choice([_log(rng, 1, 64), _log(rng, 1, 16384), _log(rng, 64, 16384)])
        case = {"op": op, "rows": max(1, min(rows, most)), "k": k, "n": n, "norm": rng.random() < 0.5,
                "dtype": rng.choice(["f16", "bf16", "bf16", "f32"])}
        if op == "gated":
            case["gate"] = rng.choice(["silu", "gelu"])
        else:
            case["add"] = rng.random() < 0.5
        return case
    if op == "rotary":
        d = rng.choice([64, 64, 128, 128, 32, 96, 192, 256, 80])
        kv, group = rng.choice([1, 2, 4, 6, 8]), rng.choice([1, 2, 4, 5, 8])
        tokens = _log(rng, 1, max(1, min(32768, 8192 * 40 * 128 // (kv * (group + 1) * d * 2))))
        return {"op": op, "tokens": tokens, "q_heads": kv * group, "kv_heads": kv, "d": d,
                "rot": rng.choice([d, d, d // 2, 2 * rng.randint(1, d // 2)]),
                "layout": rng.choice(["half", "interleaved"]), "dtype": rng.choice(["f16", "bf16", "f32"]),
                "far": _log(rng, tokens, 2000000)}
    if op == "beams":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
        vocab = _log(rng, 500, 260000)
        groups = _log(rng, 1, max(1, min(128, 64 * 8 * 130001 // (beams * vocab))))
        return {"op": op, "groups": groups, "beams": beams, "vocab": vocab, "k": rng.choice([beams, 2 * beams]),
                "dtype": rng.choice(["f16", "bf16", "f32"]), "ended": rng.random() < 0.5}
    page = rng.choice([16, 32, 64, 128])
    groups, beams = _log(rng, 1, 32), rng.choice([2, 3, 4, 5, 8, 16])
    longest = _log(rng, 10, max(20, min(page * 7000, 8 * 16 * 6500 * page // (groups * beams))))
    return {"op": op, "groups": groups, "beams": beams, "shared": rng.randint(longest // 2, longest - 1),
            "longest": longest, "page": page}


# ------------------------------------------------------------------- inputs

_DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"f16": 2, "bf16": 2, "f32": 4}
_EPS = 1e-6
_END = 2  # the token that ends an answer


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


def _book(case, rng):
    """Beams' tables: a group's beams share the pages of their common tokens and
    go on in pages of their own.  (refs, lengths, tables, pages)."""
    page, groups, beams = case["page"], case["groups"], case["beams"]
    table_pages = (case["longest"] + page - 1) // page
    common = case["shared"] // page
    pages = groups * (common + beams * (table_pages - common)) + 3
    order = rng.permutation(pages).astype(np.int32)
    tables = np.full((groups * beams, table_pages), -1, np.int32)
    lengths = np.zeros((groups * beams,), np.int32)
    refs = np.zeros((pages,), np.int32)
    at = 0
    for g in range(groups):
        # a group's beams are of one length; groups are ragged
        n = int(rng.integers(max(case["shared"], 1), case["longest"] + 1)) if g else case["longest"]
        held = (n + page - 1) // page
        first = min(common, held)
        both = order[at:at + first]
        at += first
        refs[both] = beams
        for b in range(beams):
            row = g * beams + b
            own_pages = order[at:at + held - first]
            at += held - first
            tables[row, :first], tables[row, first:held] = both, own_pages
            refs[own_pages] = 1
            lengths[row] = n
    return refs, lengths, tables, pages


def _inputs(case, seed):
    """The call's inputs as tensors and host arrays, from the seed alone."""
    g = _gen(seed)
    op = case["op"]
    if op in ("product", "gated"):
        rows, k, n = case["rows"], case["k"], case["n"]
        columns = 2 * n if op == "gated" else n
        dt = _DTYPE[case["dtype"]]
        # a few channels of the residual are much larger than the others
        big = 1.0 + 15.0 * (torch.rand((k,), generator=g, device=g.device) < 0.01).float()
        x = {"x": (_normal(g, (rows, k)) * big).to(dt),
             "codes": _normal(g, (k, columns), sigma=38.0).round_().clamp_(-127, 127).to(torch.int8),
             "scales": (0.5 + torch.rand((columns,), generator=g, device=g.device)) / (38.0 * math.sqrt(k))}
        if case["norm"]:
            x["norm"] = 1.0 + 0.2 * torch.randn((k,), generator=g, device=g.device)
        if case.get("add"):
            x["add"] = _normal(g, (rows, n), dt)
        return x
    if op == "rotary":
        t, d, dt = case["tokens"], case["d"], _DTYPE[case["dtype"]]
        return {"q": _normal(g, (t, case["q_heads"], d), dt, 2.0), "k": _normal(g, (t, case["kv_heads"], d), dt, 2.0),
                "q_norm": 1.0 + 0.2 * torch.randn((d,), generator=g, device=g.device),
                "k_norm": 1.0 + 0.2 * torch.randn((d,), generator=g, device=g.device),
                "pos": torch.randint(0, case["far"], (t,), generator=g, device=g.device, dtype=torch.int32)}
    groups, beams = case["groups"], case["beams"]
    if op == "beams":
        shape = (groups, beams)
        x = {"logits": _normal(g, shape + (case["vocab"],), _DTYPE[case["dtype"]], 3.0),
             "scores": -12.0 - 4.0 * torch.rand(shape, generator=g, device=g.device)}
        if case["ended"]:
            x["ended"] = (torch.rand(shape, generator=g, device=g.device) < 0.15).to(torch.int32)
            x["ended"][:, 0] = 0  # (a group that has ended is not asked again)
        return x
    rng = np.random.default_rng([seed, 7])
    refs, lengths, tables, pages = _book(case, np.random.default_rng([groups, beams, case["longest"]]))
    # most beams go on from themselves or from the best ones
    parents = np.minimum(rng.integers(0, beams, groups * beams), rng.integers(0, beams, groups * beams))
    return {"refs": refs, "lengths": lengths, "tables": tables, "pages": pages, "parents": parents.astype(np.int32)}


# ------------------------------------------------------- the call and its state

_RT = None


def _frequencies(case):
    """Radians a token for each pair, in 64 bits."""
    return 10000.0 ** (-2.0 * np.arange(case["rot"] // 2, dtype=np.float64) / case["rot"])


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
    a, v = _empty(rt, tuple(tensor.shape), tensor.dtype)
    v.copy_(tensor)
    return a


def _prepare_own(case, x):
    global _RT
    from manta_amd import rocm

    if _RT is None:
        _RT = rocm.Runtime(0)
    rt, op = _RT, case["op"]
    s = {"case": case, "rt": rt}
    if op in ("product", "gated"):
        w = rt.weight(x["codes"].cpu().numpy(), x["scales"].cpu().numpy(), gate=case.get("gate"))
        dt = _DTYPE[case["dtype"]]
        s["weight"] = w
        s["x"] = _put(rt, x["x"])
        s["norm"] = _put(rt, x["norm"]) if case["norm"] else None
        s["add"] = _put(rt, x["add"]) if case.get("add") else None
        s["quantized"] = rt.quantized(case["rows"], case["k"])
        s["y"], yv = _empty(rt, (case["rows"], case["n"]), dt)
        s["out"] = {"out": yv}
    elif op == "rotary":
        dt = _DTYPE[case["dtype"]]
        s["rot"] = rt.rotary_bind(_frequencies(case), layout=case["layout"])
        s["pos"] = _put(rt, x["pos"])
        s["q"], s["k"] = _put(rt, x["q"]), _put(rt, x["k"])
        s["norms"] = [_put(rt, x["q_norm"]), _put(rt, x["k_norm"])]
        s["q_out"], qv = _empty(rt, x["q"].shape, dt)
        s["k_out"], kv = _empty(rt, x["k"].shape, dt)
        s["parts"] = [(s["q"], s["q_out"]), (s["k"], s["k_out"])]
        s["out"] = {"q": qv, "k": kv}
    elif op == "beams":
        shape = (case["groups"], case["k"])
        s["beams"] = rt.beams(case["groups"], case["beams"], case["k"])
        s["logits"], s["scores"] = _put(rt, x["logits"]), _put(rt, x["scores"])
        s["ended"] = _put(rt, x["ended"]) if case["ended"] else None
        s["parents"], pv = _empty(rt, shape, torch.int32)
        s["tokens"], tv = _empty(rt, shape, torch.int32)
        s["totals"], sv = _empty(rt, shape, torch.float32)
        s["out"] = {"parents": pv, "tokens": tv, "scores": sv}
    else:
        seqs, table_pages = x["tables"].shape
        # (what lies in the pages does not matter here: one small head)
        c = rt.cache(pages=x["pages"], page_tokens=case["page"], kv_heads=1, head_dim=32, seqs=seqs,
                     table_pages=table_pages)
        book = np.concatenate([x["refs"], x["lengths"], x["tables"].ravel()])
        bv = _view(c.book, torch.int32)
        bv.copy_(torch.from_numpy(book))
        s["cache"], s["saved"] = c, rt.to_device(book)
        s["seqs"] = rt.to_device(np.arange(seqs, dtype=np.int32))
        s["parents"] = rt.to_device(x["parents"])
        s["out"] = {"book": bv}
    torch.cuda.synchronize()
    return s


def prepare(case, seed):
    x = _inputs(case, seed)
    if own:
        return _prepare_own(case, x)
    dev = _device()
    s = {"case": case, "x": x}
    if case["op"] in ("product", "gated"):
        x["codes"] = x["codes"].float()  # (weights are laid out once)
    elif case["op"] == "rotary":
        s["freqs"] = torch.from_numpy(_frequencies(case)).to(dev)
    elif case["op"] == "reorder":
        groups, beams = case["groups"], case["beams"]
        for name in ("refs", "lengths", "tables"):
            s[name] = torch.from_numpy(x[name]).to(dev)
        s["saved"] = [s[n].clone() for n in ("refs", "lengths", "tables")]
        s["parents"] = torch.from_numpy(x["parents"]).to(dev)
        s["first"] = (torch.arange(groups * beams, device=dev) // beams) * beams
    return s


def run(s):
    return _run_own(s) if own else _PLAIN[s["case"]["op"]](s)


def _run_own(s):
    case, op, rt = s["case"], s["case"]["op"], s["rt"]
    if op in ("product", "gated"):
        rt.quantize_rows(s["x"], s["quantized"], norm=s["norm"], eps=_EPS, dtype=case["dtype"])
        rt.matmul_q8(s["weight"], s["quantized"], out=s["y"], add=s["add"], dtype=case["dtype"])
    elif op == "rotary":
        rt.rotary_normed(s["rot"], s["pos"], s["parts"], s["norms"], eps=_EPS, dtype=case["dtype"])
    elif op == "beams":
        s["beams"].select(s["logits"], s["scores"], s["parents"], s["tokens"], s["totals"], ended=s["ended"],
                          end_token=_END, dtype=case["dtype"])
    else:
        rt.copy(s["cache"].book, s["saved"])
        s["cache"].reorder(s["seqs"], s["parents"], case["beams"])
    return s["out"]


# ------------------------------------------------------------ the plain forms

def _quantise(x, norm):
    """Rows in 8 bits, as f32: (codes, scales).  A norm's factor of a row
    cancels in its codes and goes into its scale."""
    z = x.float()
    factor = None
    if norm is not None:
        factor = 1.0 / torch.sqrt((z * z).mean(1, keepdim=True) + _EPS)
        z = z * norm
    largest = z.abs().amax(1, keepdim=True)
    tiny = largest < 2.0 ** -126
    codes = torch.where(tiny, 0.0, (z * 127.0 / largest).round().clamp(-127, 127))
    scales = torch.where(tiny, 0.0, largest / 127.0)
    return codes, scales if factor is None else scales * factor


def _act(x, gate):
    if gate == "silu":
        return x / (1.0 + torch.exp(-x))
    return 0.5 * x * (1.0 + torch.tanh(0.7978845608 * (x + 0.044715 * x * x * x)))


def _plain_product(s):
    case, x = s["case"], s["x"]
    codes, scales = _quantise(x["x"], x.get("norm"))
    y = torch.matmul(codes, x["codes"]) * (scales * x["scales"])
    if case["op"] == "gated":
        n = case["n"]
        y = _act(y[:, :n], case["gate"]) * y[:, n:]
    elif "add" in x:
        y = y + x["add"].float()
    return {"out": y.to(x["x"].dtype)}


def _plain_rotary(s):
    case, x, rot = s["case"], s["x"], s["case"]["rot"]
    angle = x["pos"].double()[:, None, None] * s["freqs"]  # far positions: 32 bits lose the angle
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    out = {}
    for name in ("q", "k"):
        y = x[name].float()
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + _EPS) * x[name + "_norm"]
        if case["layout"] == "half":
            a, b, rest = y[..., :rot // 2], y[..., rot // 2:rot], y[..., rot:]
        else:
            a, b, rest = y[..., 0:rot:2], y[..., 1:rot:2], y[..., rot:]
        a, b = a * cos - b * sin, b * cos + a * sin
        turned = torch.cat([a, b], -1) if case["layout"] == "half" else torch.stack([a, b], -1).flatten(-2)
        out[name] = torch.cat([turned, rest], -1).to(x[name].dtype)
    return out


def _plain_beams(s):
    case, x = s["case"], s["x"]
    vocab, k = case["vocab"], case["k"]
    y = x["logits"].double()  # totals of different beams lie closer than 32 bits tell apart
    top = y.amax(-1, keepdim=True)
    y = y - (top + torch.exp(y - top).sum(-1, keepdim=True).log())
    if case["ended"]:
        over = x["ended"].bool()[..., None]
        y = torch.where(over, float("-inf"), y)
        y[..., _END:_END + 1] = torch.where(over, 0.0, y[..., _END:_END + 1])
    y = (y + x["scores"].double()[..., None]).flatten(1)
    values, places = [], []
    for _ in range(k):  # the first of equal ones each time
        best = y.argmax(1, keepdim=True)
        values.append(y.gather(1, best))
        places.append(best)
        y.scatter_(1, best, float("-inf"))
    values, places = torch.cat(values, 1), torch.cat(places, 1)
    return {"parents": (places // vocab).int(), "tokens": (places % vocab).int(), "scores": values.float()}


def _plain_reorder(s):
    for name, saved in zip(("refs", "lengths", "tables"), s["saved"]):
        s[name].copy_(saved)
    source = s["first"] + s["parents"].long()
    before, after = s["tables"], s["tables"][source]
    for entries, by in ((before, -1), (after, 1)):
        held = entries[entries >= 0]
        s["refs"].index_add_(0, held.long(), torch.full_like(held, by))
    s["tables"] = after
    s["lengths"] = s["lengths"][source]
    return {"book": torch.cat([s["refs"], s["lengths"], s["tables"].view(-1)])}


_PLAIN = {"product": _plain_product, "gated": _plain_product, "rotary": _plain_rotary, "beams": _plain_beams,
          "reorder": _plain_reorder}


# ------------------------------------------------------------ what it costs

def work(case):
    op = case["op"]
    if op in ("product", "gated"):
        rows, k, n, size = case["rows"], case["k"], case["n"], _BYTES[case["dtype"]]
        columns = 2 * n if op == "gated" else n
        results = rows * n * (2 if case.get("add") else 1)
        return {"bytes": size * (rows * k + results) + k * columns + 4 * columns + (4 * k if case["norm"] else 0),
                "flops": 2 * rows * k * columns}
    if op == "rotary":
        heads = case["tokens"] * (case["q_heads"] + case["kv_heads"])
        return {"bytes": 2 * heads * case["d"] * _BYTES[case["dtype"]] + 4 * case["tokens"] + 8 * case["d"],
                "flops": heads * (4 * case["d"] + 3 * case["rot"])}
    rows = case["groups"] * case["beams"]
    if op == "beams":
        # (an ended beam's logits need not be read: 0.15 of them)
        read = rows * case["vocab"] * (0.85 if case["ended"] else 1.0)
        return {"bytes": int(read * _BYTES[case["dtype"]]) + 4 * rows + 12 * case["groups"] * case["k"],
                "flops": int(3 * read)}
    # every sequence's table and length is read, and written where it changes
    table_pages = (case["longest"] + case["page"] - 1) // case["page"]
    apart = table_pages - case["shared"] // case["page"]
    return {"bytes": 4 * rows * (table_pages + 3 + 3 * apart), "flops": 0}


# ------------------------------------------------------------ in 64 bits

def _exact_product(case, x):
    # codes are whole numbers that f32 arithmetic defines; what follows is in 64 bits
    v = x["x"].float() * x["norm"] if case["norm"] else x["x"].float()
    m = v.abs().max(dim=1).values
    live = m >= 2.0 ** -126
    m1 = torch.where(live, m, torch.ones_like(m))
    c = torch.clamp(torch.round((v * 127.0) / m1[:, None]), min=-127, max=127).double() * live[:, None]
    s = m.double() / 127.0
    if case["norm"]:
        s = s * (x["x"].double().pow(2).sum(1) / case["k"] + _EPS).rsqrt()
    y = (c @ x["codes"].double()).mul_(s[:, None]).mul_(x["scales"].double()[None])
    if case["op"] == "gated":
        a, b = y.chunk(2, 1)
        if case["gate"] == "silu":
            return {"out": a * torch.sigmoid(a) * b}
        return {"out": a * torch.sigmoid(2.0 * 0.7978845608 * a * (1.0 + 0.044715 * a * a)) * b}
    return {"out": y + x["add"].double() if case["add"] else y}


def _exact_rotary(case, x):
    f = _frequencies(case)
    angle = x["pos"].double()[:, None] * torch.from_numpy(f).to(x["pos"].device)[None]
    c = torch.polar(torch.ones_like(angle), angle)[:, None]
    out = {}
    for name in ("q", "k"):
        y = x[name].double()
        y = y * (y.pow(2).sum(-1, keepdim=True) / case["d"] + _EPS).rsqrt() * x[name + "_norm"].double()
        r = y[..., :case["rot"]]
        if case["layout"] == "half":
            z = torch.complex(*(v.contiguous() for v in r.chunk(2, -1))) * c
            y[..., :case["rot"]] = torch.cat([z.real, z.imag], -1)
        else:
            z = torch.view_as_complex(r.reshape(*r.shape[:-1], -1, 2).contiguous()) * c
            y[..., :case["rot"]] = torch.view_as_real(z).flatten(-2)
        out[name] = y
    return out


def _exact_beams(case, x):
    """Group by group: every beam's own best k, then the best k of those."""
    out = {"parents": [], "tokens": [], "scores": []}
    for g in range(case["groups"]):
        found = []
        for b in range(case["beams"]):
            score = float(x["scores"][g, b])
            if case["ended"] and int(x["ended"][g, b]):
                found.append((-score, b, _END))
                continue
            row = x["logits"][g, b].double()
            lse = float(torch.logsumexp(row, 0))
            least = row.sort(descending=True).values[min(case["k"], row.numel()) - 1]
            for t in torch.nonzero(row >= least)[:, 0].tolist():
                found.append((-(score + (float(row[t]) - lse)), b, t))
        found = sorted(found)[:case["k"]]
        out["scores"].append([-f[0] for f in found])
        out["parents"].append([f[1] for f in found])
        out["tokens"].append([f[2] for f in found])
    dev = x["scores"].device
    return {"parents": torch.tensor(out["parents"], device=dev, dtype=torch.int32),
            "tokens": torch.tensor(out["tokens"], device=dev, dtype=torch.int32),
            "scores": torch.tensor(out["scores"], device=dev, dtype=torch.float64)}


def exact(case, seed):
    if case["op"] == "reorder":
        return None
    x = _inputs(case, seed)
    return {"product": _exact_product, "gated": _exact_product, "rotary": _exact_rotary,
            "beams": _exact_beams}[case["op"]](case, x)
