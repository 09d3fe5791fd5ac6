"""Products in 8 bits and beams (include/manta_decode.h): with the calls of
cache.py, what a model that writes an answer needs for a step.

    q = rt.quantize_rows(x, norm=w)                   # a layer
    rt.matmul_q8(qkv, q, out=y)
    rt.rotary_normed(rot, positions, [(yq, yq), (yk, yk)], norms)
    ...
    beams.select(logits, scores, parents, tokens, scores)
    cache.reorder(seqs, parents, group)
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import numpy as np

from . import _lib
from ._lib import call, load
from .cache import _kind

_F32 = np.dtype(np.float32)
_EMPTY = {"f32": np.float32, "f16": np.uint16, "bf16": np.uint16}


class Weight:
    """A bound weight (Runtime.weight)."""

    def __init__(self, rt, codes: np.ndarray, scales: np.ndarray, gate: Optional[str]):
        if gate not in _lib.GATES:
            raise ValueError("unknown gate %r (silu, gelu or None)" % (gate,))
        codes, scales = np.asarray(codes), np.asarray(scales)
        if codes.ndim != 2 or codes.dtype != np.int8:
            raise ValueError("weight codes must be int8 [width, columns] (got %s %s)" % (codes.dtype, codes.shape))
        width, columns = codes.shape
        if scales.shape != (columns,):
            raise ValueError("weight scales must be [%d] (got %s)" % (columns, scales.shape))
        if gate is not None and columns % 2:
            raise ValueError("a gated weight needs as many columns of the gate as of the other (got %d)" % columns)
        codes, scales = np.ascontiguousarray(codes), np.ascontiguousarray(scales, np.float32)
        self.rt, self.gate, self.width = rt, gate, width
        self.n = columns // 2 if gate is not None else columns
        self.handle = C.c_void_p()
        call("manta_rocm_weight_bind", rt.handle, codes.ctypes.data, scales.ctypes.data, width, self.n,
             _lib.GATES[gate], C.byref(self.handle))

    def close(self) -> None:
        if self.handle is not None and self.handle.value:
            load().manta_rocm_weight_unbind(self.handle)
        self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Quantized:
    """Rows in 8 bits with a scale each (Runtime.quantized): codes in blocks of
    16 rows and 64 columns, as the products read them."""

    shared = False  # part of a larger one (first)

    def __init__(self, rt, rows: int, width: int):
        size = load().manta_rocm_quantized_bytes(rows, width)
        if size < 0:
            raise ValueError("quantized rows: bad shape [%s, %s]" % (rows, width))
        self.rt, self.rows, self.width = rt, rows, width
        self.codes = rt.empty((size,), np.int8)
        self.scales = rt.empty((rows,), np.float32)

    def first(self, rows: int) -> "Quantized":
        """The memory of the first `rows` rows, for a batch of so many: it is
        this one's."""
        if not 0 <= rows <= self.rows:
            raise ValueError("quantized rows: %s of %d" % (rows, self.rows))
        part = Quantized.__new__(Quantized)
        part.rt, part.rows, part.width, part.codes, part.scales = self.rt, rows, self.width, self.codes, self.scales
        part.shared = True
        return part

    def values(self):
        """(codes int8 [rows, width], scales f32 [rows]) on the host; waits
        for the stream."""
        pitch = (self.width + 127) // 128 * 128
        c = self.codes.download().reshape(-1, pitch // 64, 4, 16, 16)
        c = c.transpose(0, 3, 1, 2, 4).reshape(-1, pitch)
        scales = self.scales.download()
        return np.ascontiguousarray(c[:self.rows, :self.width]), scales[:self.rows] if self.shared else scales


def _matrix(name: str, a, rows: Optional[int] = None, columns: Optional[int] = None):
    """(address, rows, columns, row stride)."""
    if len(a.shape) != 2 or (rows is not None and a.shape[0] != rows) or (columns is not None and a.shape[1] != columns):
        raise ValueError("%s must be [%s, %s] (got %s)" % (name, "rows" if rows is None else rows,
                                                           "columns" if columns is None else columns, a.shape))
    strides = a.strides
    r, c = a.shape
    return a.addr, r, c, c if strides is None else strides[0]


def _f32_row(a, width: int) -> bool:
    return (a.dtype is _F32 or a.dtype == _F32) and a.shape == (width,) and (a.strides is None or a.strides == (1,))


def quantize_rows(rt, x, out, norm, eps: float, dtype: Optional[str]):
    kind = _kind(x, dtype)
    addr, rows, width, stride = _matrix("x", x)
    if norm is not None and not _f32_row(norm, width):
        raise ValueError("norm must be f32 [%d] (got %s %s)" % (width, norm.dtype, norm.shape))
    if out is None:
        out = Quantized(rt, rows, width)
    elif out.rows != rows or out.width != width:
        raise ValueError("quantized rows must be [%d, %d] (got [%d, %d])" % (rows, width, out.rows, out.width))
    call("manta_rocm_quantize_rows", rt.handle, kind, addr, stride, rows, width, None if norm is None else norm.addr,
         eps, out.codes.addr, out.scales.addr)
    return out


def matmul_q8(rt, weight: Weight, x: Quantized, out, add, dtype: Optional[str]):
    if x.width != weight.width:
        raise ValueError("matmul mismatch [%d, %d] x [%d, %d]" % (x.rows, x.width, weight.width, weight.n))
    if out is None:
        if dtype is None:
            dtype = "f16"
        if dtype not in _EMPTY:
            raise TypeError("elements must be f32, f16 or bf16 (got %s)" % dtype)
        out = rt.empty((x.rows, weight.n), _EMPTY[dtype])
    kind = _kind(out, dtype)
    addr, _, _, stride = _matrix("out", out, x.rows, weight.n)
    add_addr, add_stride = None, 0
    if add is not None:
        if _kind(add, dtype) != kind:
            raise TypeError("add and out must have one element type")
        add_addr, _, _, add_stride = _matrix("add", add, x.rows, weight.n)
    call("manta_rocm_matmul_q8", rt.handle, weight.handle, x.codes.addr, x.scales.addr, x.rows, kind, add_addr,
         add_stride, addr, stride)
    return out


class Beams:
    """The choice of the next beams (Runtime.beams).  Calls that may overlap
    take one each."""

    def __init__(self, rt, groups: int, beams: int, best: int):
        self.rt = rt
        self.handle = C.c_void_p()
        call("manta_rocm_beams_create", rt.handle, groups, beams, best, C.byref(self.handle))

    def close(self) -> None:
        if self.handle is not None and self.handle.value:
            load().manta_rocm_beams_destroy(self.handle)
        self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def select(self, logits, scores, parents, tokens, totals, ended=None, end_token: int = 0,
               dtype: Optional[str] = None, out_ended=None) -> None:
        """The best continuations: logits [groups, beams, vocab], scores f32
        [groups, beams] (their sums of log probabilities), results [groups,
        best]: parents and tokens int32, totals f32; ended: int32 [groups,
        beams], not 0 for beams whose only continuation is end_token;
        out_ended: the same [groups, best] for the next call."""
        kind = _kind(logits, dtype)
        if len(logits.shape) != 3:
            raise ValueError("logits must be [groups, beams, vocab] (got %s)" % (logits.shape,))
        groups, beams, vocab = logits.shape
        strides = logits.strides
        row = vocab if strides is None else strides[0 if beams == 1 else 1]
        if strides is not None and groups > 1 and strides[0] != beams * row:
            raise ValueError("logits of a group must follow those of the group before (strides %s)" % (strides,))
        if len(parents.shape) != 2 or parents.shape[0] != groups:
            raise ValueError("parents must be [%d, best] (got %s)" % (groups, parents.shape))
        best = parents.shape[1]
        for name, a, shape, dt in (("scores", scores, (groups, beams), np.float32),
                                   ("parents", parents, (groups, best), np.int32),
                                   ("tokens", tokens, (groups, best), np.int32),
                                   ("totals", totals, (groups, best), np.float32),
                                   ("ended", ended, (groups, beams), np.int32),
                                   ("out_ended", out_ended, (groups, best), np.int32)):
            if a is not None and (a.dtype != dt or tuple(a.shape) != shape or a.strides is not None):
                raise ValueError("%s must be a whole %s array %s (got %s %s)"
                                 % (name, np.dtype(dt).name, shape, a.dtype, a.shape))
        call("manta_rocm_beam_select", self.rt.handle, self.handle, kind, logits.addr,
             row, groups, beams, vocab, scores.addr,
             None if ended is None else ended.addr, end_token, best, parents.addr, tokens.addr, totals.addr,
             None if out_ended is None else out_ended.addr)


def beam_inputs(rt, tokens, out, instead: int) -> None:
    for name, a in (("tokens", tokens), ("out", out)):
        if a.dtype != np.int32 or a.strides is not None or a.nbytes != tokens.nbytes:
            raise ValueError("%s must be a whole int32 array, one entry a token (got %s %s)" % (name, a.dtype, a.shape))
    call("manta_rocm_beam_inputs", rt.handle, tokens.addr, tokens.nbytes // 4, instead, out.addr)
