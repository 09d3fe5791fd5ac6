"""Rotary positions and the 8-bit key/value cache (include/manta_cache.h):
what a model that reads retrieved passages needs between its products.

A decoding step of one layer:

    cache.extend(seqs, ones)                          # once for all layers
    rt.rotary(rot, positions, [(q, q), (k, k)])
    cache.append(layer, k, v, offsets, seqs)
    cache.attention(layer, q, offsets, seqs, out=o)
"""
from __future__ import annotations

import ctypes as C
import math
import struct
from typing import Optional

import numpy as np

from . import _lib
from ._lib import call, load

_KINDS = {"f32": (_lib.F32, 4), "f16": (_lib.F16, 2), "bf16": (_lib.BF16, 2)}


_HEADS = struct.Struct("=QQqqqqq").pack  # MantaRocmHeads
_SEEN: dict = {}  # (name, array type) -> element type


def _kind(a, dtype: Optional[str]) -> int:
    """The element type of a device array: given by name, else its own."""
    known = _SEEN.get((dtype, a.dtype))
    if known is None:
        known = _SEEN[(dtype, a.dtype)] = _find_kind(a, dtype)
    return known


def _find_kind(a, dtype: Optional[str]) -> int:
    if dtype is None:
        dtype = {"f": {4: "f32", 2: "f16"}, "u": {2: "f16"}}.get(a.dtype.kind, {}).get(a.dtype.itemsize)
    kind = _KINDS.get(dtype)
    if kind is None:
        raise TypeError("elements must be f32, f16 or bf16 (got %s)" % (dtype or a.dtype))
    if a.dtype.itemsize != kind[1] or a.dtype.kind not in "fu":
        raise TypeError("an array of %s does not hold %s" % (a.dtype, dtype))
    return kind[0]


def _rows(name: str, a, heads: Optional[int] = None, dim: Optional[int] = None):
    """(address, tokens, heads, dim, token stride, head stride)."""
    if len(a.shape) != 3:
        raise ValueError("%s must be [tokens, heads, head_dim] (got %s)" % (name, a.shape))
    t, h, d = a.shape
    if (heads is not None and h != heads) or (dim is not None and d != dim):
        raise ValueError("%s must be [tokens, %s, %s] (got %s)" % (name, heads, dim, a.shape))
    try:
        strides = a.strides
    except AttributeError:
        strides = None
    return (a.addr, t, h, d, h * d, d) if strides is None else (a.addr, t, h, d, strides[0], strides[1])


def _ints(name: str, a, n: Optional[int] = None) -> int:
    if a.dtype != np.int32 or len(a.shape) != 1 or (n is not None and a.shape[0] != n):
        raise ValueError("%s must be int32 [%s] (got %s %s)" % (name, "n" if n is None else n, a.dtype, a.shape))
    return a.addr


class Rotary:
    """Bound frequencies (Runtime.rotary_bind)."""

    def __init__(self, rt, freqs, layout: str, magnitude: float):
        layouts = {"half": _lib.ROTARY_HALF, "interleaved": _lib.ROTARY_INTERLEAVED}
        if layout not in layouts:
            raise ValueError("unknown rotary layout %r (half, interleaved)" % (layout,))
        freqs = np.ascontiguousarray(freqs, np.float64)
        if freqs.ndim != 1:
            raise ValueError("rotary frequencies must be one axis (got %s)" % (freqs.shape,))
        self.rt, self.rot = rt, 2 * freqs.shape[0]
        self.handle = C.c_void_p()
        call("manta_rocm_rotary_bind", rt.handle, freqs.ctypes.data_as(C.c_void_p), self.rot, layouts[layout],
             float(magnitude), C.byref(self.handle))

    def close(self) -> None:
        if self.handle is not None and self.handle.value:
            load().manta_rocm_rotary_unbind(self.handle)
        self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _parts(rot, parts, dtype):
    """(element type, tokens, head_dim, the packed tensors, their number)."""
    parts = list(parts)
    if not parts:
        raise ValueError("rotary needs at least one tensor")
    packed = b""
    kind = _kind(parts[0][0], dtype)
    tokens = dim = None
    for x, out in parts:
        if _kind(x, dtype) != kind or _kind(out, dtype) != kind:
            raise TypeError("rotary tensors must have one element type")
        xp, t, h, d, xt, xh = _rows("x", x)
        if tuple(out.shape) != tuple(x.shape):
            raise ValueError("rotary out must be %s (got %s)" % (x.shape, out.shape))
        op, _, _, _, ot, oh = _rows("out", out)
        packed += _HEADS(xp, op, h, xt, xh, ot, oh)
        if tokens is None:
            tokens, dim = t, d
        elif (t, d) != (tokens, dim):
            raise ValueError("rotary tensors must agree on tokens and head_dim")
    return kind, tokens, dim, packed, len(parts)


def rotary(rt, rot: Rotary, positions, parts, inverse: bool, dtype: Optional[str]) -> None:
    kind, tokens, dim, packed, n = _parts(rot, parts, dtype)
    call("manta_rocm_rotary", rt.handle, rot.handle, kind, _ints("positions", positions, tokens), tokens, dim, packed,
         n, 1 if inverse else 0)


def rotary_normed(rt, rot: Rotary, positions, parts, norms, eps: float, dtype: Optional[str]) -> None:
    kind, tokens, dim, packed, n = _parts(rot, parts, dtype)
    if len(norms) != n:
        raise ValueError("rotary_normed needs a norm (or None) for each tensor (%d for %d)" % (len(norms), n))
    addrs = []
    for w in norms:
        if w is not None and (w.dtype != np.float32 or tuple(w.shape) != (dim,) or w.strides not in (None, (1,))):
            raise ValueError("a norm must be f32 [%d] (got %s %s)" % (dim, w.dtype, w.shape))
        addrs.append(0 if w is None else w.addr)
    call("manta_rocm_rotary_normed", rt.handle, rot.handle, kind, _ints("positions", positions, tokens), tokens, dim,
         packed, struct.pack("=%dQ" % n, *addrs), n, eps)


class _Part:
    """Device memory that a Cache owns, as an array (download, rt.copy)."""

    strides = None

    def __init__(self, cache: "Cache", addr: int, shape, dtype):
        self.cache, self.rt, self.addr = cache, cache.rt, addr
        self.shape, self.dtype = tuple(int(s) for s in shape), np.dtype(dtype)
        self.nbytes = int(np.prod(self.shape, dtype=np.int64)) * self.dtype.itemsize

    def download(self) -> np.ndarray:
        out = np.empty(self.shape, self.dtype)
        call("manta_rocm_download", self.rt.handle, out.ctypes.data_as(C.c_void_p), self.addr, self.nbytes)
        return out

    def upload(self, host: np.ndarray) -> "_Part":
        host = np.ascontiguousarray(host, self.dtype)
        if host.nbytes != self.nbytes:
            raise ValueError("upload size mismatch: %d vs %d" % (host.nbytes, self.nbytes))
        call("manta_rocm_upload", self.rt.handle, self.addr, host.ctypes.data_as(C.c_void_p), self.nbytes)
        return self


class Cache:
    """Keys and values in 8 bits, in pages that sequences share.  k_codes,
    v_codes, k_max, v_max and book are its device memory, lengths the part of
    book that a loop on the device takes positions from."""

    def __init__(self, rt, layers, pages, page_tokens, kv_heads, head_dim, seqs, table_pages):
        self.rt = rt
        self.layers, self.pages, self.page_tokens = int(layers), int(pages), int(page_tokens)
        self.kv_heads, self.head_dim = int(kv_heads), int(head_dim)
        self.seqs, self.table_pages = int(seqs), int(table_pages)
        self.handle = C.c_void_p()
        shape = _lib.CacheShape(self.layers, self.pages, self.page_tokens, self.kv_heads, self.head_dim, self.seqs,
                                self.table_pages)
        call("manta_rocm_cache_create", rt.handle, C.byref(shape), C.byref(self.handle))
        b = _lib.CacheBuffers()
        load().manta_rocm_cache_buffers(self.handle, C.byref(b))
        self.pitch = b.pitch
        lead = (self.layers, self.pages, self.kv_heads)
        self.k_codes = _Part(self, b.k_codes, lead + (self.page_tokens, b.pitch), np.int8)
        self.v_codes = _Part(self, b.v_codes, lead + (b.pitch, self.page_tokens), np.int8)
        self.k_max = _Part(self, b.k_max, lead, np.float32)
        self.v_max = _Part(self, b.v_max, lead, np.float32)
        self.book = _Part(self, b.book, (b.book_count,), np.int32)
        self.lengths = _Part(self, b.book + 4 * self.pages, (self.seqs,), np.int32)

    def close(self) -> None:
        if self.handle is not None and self.handle.value:
            load().manta_rocm_cache_destroy(self.handle)
        self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # -------------------------------------------------------------- pages
    def tables(self):
        """(refs [pages], lengths [seqs], tables [seqs, table_pages]) on the
        host; waits for the stream."""
        b = self.book.download()
        p, s = self.pages, self.seqs
        return b[:p], b[p:p + s], b[p + s:].reshape(s, self.table_pages)

    def extend(self, seqs, counts) -> None:
        """Grow sequences by counts[i] tokens (both int32 device arrays)."""
        call("manta_rocm_cache_extend", self.rt.handle, self.handle, _ints("seqs", seqs),
             _ints("counts", counts, seqs.shape[0]), seqs.shape[0])

    def fork(self, parents, children, tokens=None) -> None:
        """children[i] shares the first tokens[i] tokens (all) of parents[i]."""
        n = parents.shape[0]
        call("manta_rocm_cache_fork", self.rt.handle, self.handle, _ints("parents", parents),
             _ints("children", children, n), None if tokens is None else _ints("tokens", tokens, n), n)

    def release(self, seqs, keep=None) -> None:
        """Cut sequences to keep[i] tokens (0)."""
        n = seqs.shape[0]
        call("manta_rocm_cache_release", self.rt.handle, self.handle, _ints("seqs", seqs),
             None if keep is None else _ints("keep", keep, n), n)

    def reorder(self, seqs, parents, group: Optional[int] = None) -> None:
        """Groups of `group` sequences (all of them): entry i takes over what
        entry parents[i] of its group held; -1 empties it."""
        n = seqs.shape[0]
        call("manta_rocm_cache_reorder", self.rt.handle, self.handle, _ints("seqs", seqs), _ints("parents", parents, n),
             n, max(n, 1) if group is None else group)

    def compact(self, live=None) -> None:
        """Move live pages down into free ones; live: int32 [1], their count."""
        call("manta_rocm_cache_compact", self.rt.handle, self.handle, None if live is None else _ints("live", live, 1))

    def copy_pages(self, src, dst) -> None:
        call("manta_rocm_cache_copy_pages", self.rt.handle, self.handle, _ints("src", src),
             _ints("dst", dst, src.shape[0]), src.shape[0])

    # ----------------------------------------------------------- contents
    def _batch(self, offsets, seqs):
        n = offsets.shape[0] - 1
        if n < 0:
            raise ValueError("offsets must be int32 [n + 1]")
        return _ints("offsets", offsets), None if seqs is None else _ints("seqs", seqs, n), n

    def _kv(self, entry, layer, k, v, offsets, seqs, dtype):
        kind = _kind(k, dtype)
        if _kind(v, dtype) != kind:
            raise TypeError("k and v must have one element type")
        kp, t, _, _, kt, kh = _rows("k", k, self.kv_heads, self.head_dim)
        vp, tv, _, _, vt, vh = _rows("v", v, self.kv_heads, self.head_dim)
        if t != tv:
            raise ValueError("k and v must have as many tokens (%d, %d)" % (t, tv))
        off, sq, n = self._batch(offsets, seqs)
        call(entry, self.rt.handle, self.handle, layer, kind, kp, kt, kh, vp, vt, vh, off, sq, n, t)

    def append(self, layer: int, k, v, offsets, seqs=None, dtype: Optional[str] = None) -> None:
        """Quantise the sequences' last tokens, rows offsets[i] ..
        offsets[i + 1] of k and v [tokens, kv_heads, head_dim], into the pages
        that extend gave them."""
        self._kv("manta_rocm_cache_append", layer, k, v, offsets, seqs, dtype)

    def read(self, layer: int, offsets, k, v, seqs=None, dtype: Optional[str] = None) -> None:
        """The sequences' last tokens as numbers, into k and v."""
        self._kv("manta_rocm_cache_read", layer, k, v, offsets, seqs, dtype)

    def attention(self, layer: int, q, offsets, seqs=None, out=None, lse=None, scale: Optional[float] = None,
                  causal: bool = True, window: int = 0, longest: Optional[int] = None, dtype: Optional[str] = None):
        """softmax(scale q k^T) v of q [tokens, heads, head_dim] (f16 or bf16)
        over the sequences' cached tokens; scale by default
        head_dim^-1/2.  Returns out."""
        kind = _kind(q, dtype)
        if out is None:
            out = self.rt.empty(q.shape, q.dtype)
        elif tuple(out.shape) != tuple(q.shape) or _kind(out, dtype) != kind:
            raise ValueError("attention out must be %s like q" % (q.shape,))
        qp, t, heads, _, qt, qh = _rows("q", q, None, self.head_dim)
        op, _, _, _, ot, oh = _rows("out", out)
        packed = _HEADS(qp, op, heads, qt, qh, ot, oh)
        if lse is not None and (lse.dtype != np.float32 or tuple(lse.shape) != tuple(q.shape[:2])
                                or lse.strides is not None):
            raise ValueError("attention lse must be a whole f32 array %s" % (q.shape[:2],))
        off, sq, n = self._batch(offsets, seqs)
        call("manta_rocm_cache_attention", self.rt.handle, self.handle, layer, kind, packed,
             None if lse is None else lse.addr, off, sq, n, t,
             1.0 / math.sqrt(self.head_dim) if scale is None else scale, 1 if causal else 0, window,
             self.table_pages * self.page_tokens if longest is None else longest)
        return out
