"""Operators of transformers over image and video tokens: rotary positions with
several axes, norms of query and key heads with the rotation in the same pass,
selection of key blocks and attention over them. Thin calls of
libmoebius_hip.so (include/moebius_hip.h); the reference has no counterpart.

    rope = RopeAxes(ctx, (16, 56, 56))                   # time, height, width
    qk_norm_rope(q, k, gamma_q, gamma_k, 1e-6, positions, rope, q_out, k_out)
    block_means(k_out, 64, means)
    block_select(q_out, means, kv_tokens, blocks, q_block=64, kv_block=64)
    block_attention(q_out, k_out, v, blocks, out, q_block=64, kv_block=64)
"""
from __future__ import annotations

import ctypes
import math

import numpy as np

from . import _lib
from ._lib import MoebiusError, check, lib
from .engine import Context, DeviceArray, _ptr

# The calls below are a few microseconds on the host, of single tokens as long as on the
# device: what a view or a table fixes is worked out when it is made.
_F32, _I32 = np.dtype(np.float32), np.dtype(np.int32)
_DTYPE = {_F32: _lib.DTYPE_F32, np.dtype(np.float16): _lib.DTYPE_F16}


class Heads:
    """Heads of tokens [n][tokens][heads][d] over a DeviceArray (f32 or f16), rows
    `ld` elements apart from element `offset` on: the queries, keys or values of a
    fused projection are views of it."""

    def __init__(self, buf: DeviceArray, n: int, tokens: int, heads: int, d: int, ld: int | None = None,
                 offset: int = 0):
        if buf.dtype not in _DTYPE:
            raise MoebiusError(1, "heads are f32 or f16")
        self.buf, self.n, self.tokens, self.heads, self.d = buf, int(n), int(tokens), int(heads), int(d)
        self.ld = int(heads * d if ld is None else ld)
        self.dtype, self.code = buf.dtype, _DTYPE[buf.dtype]
        rows = self.n * self.tokens
        if min(self.n, self.tokens, offset) < 0 or self.ld < heads * d:
            raise MoebiusError(1, "heads: negative size or ld below heads * d")
        if rows and (offset + (rows - 1) * self.ld + heads * d) * self.dtype.itemsize > buf.nbytes:
            raise MoebiusError(1, "heads exceed their buffer")
        self._offset = int(offset) * self.dtype.itemsize
        self.ctx: Context = buf.ctx
        self.rows = rows
        self._kind = (self.code, self.d)
        self._shape = (self.code, self.d, self.n, self.tokens, self.heads)

    @property
    def ptr(self) -> int:
        return self.buf.ptr + self._offset

    def numpy(self) -> np.ndarray:
        """A copy [n, tokens, heads, d]."""
        if not self.rows:
            return np.empty((self.n, self.tokens, self.heads, self.d), self.dtype)
        flat = self.buf.numpy().reshape(-1)[self._offset // self.dtype.itemsize:]
        s = self.dtype.itemsize
        view = np.lib.stride_tricks.as_strided(flat, (self.rows, self.heads, self.d), (self.ld * s, self.d * s, s))
        return view.copy().reshape(self.n, self.tokens, self.heads, self.d)


def _same(a, *heads):
    for b in heads:
        if a._kind != b._kind:
            raise MoebiusError(1, "heads differ in type or channels")
        if a.ctx is not b.ctx:
            raise MoebiusError(1, "heads of different contexts")


def _int32(a, size, what):
    if a is not None and (a.dtype != _I32 or a.nbytes != 4 * size):
        raise MoebiusError(1, f"{what} is int32 of {size} entries")


class RopeAxes:
    """Rotary positions whose axis a turns axis_dims[a] channels of a head with
    frequencies theta^(-2j / axis_dims[a]), or the given ones (radians per position)."""

    def __init__(self, ctx: Context, axis_dims, theta: float = 10000.0, pairing: str = "interleaved", freq=None):
        self.axis_dims = tuple(int(m) for m in axis_dims)
        if not 1 <= len(self.axis_dims) <= 4:
            raise MoebiusError(1, "rope: 1 to 4 axes")
        if pairing not in _lib.ROPE_PAIRING:
            raise MoebiusError(1, f"unknown pairing {pairing!r}")
        self.pairing = _lib.ROPE_PAIRING[pairing]
        pairs = sum(self.axis_dims) // 2
        if freq is None:
            freq = np.empty(pairs, np.float64)
            dims = (ctypes.c_uint32 * len(self.axis_dims))(*self.axis_dims)
            check(lib().mh_rope_frequencies(float(theta), len(self.axis_dims), dims, freq.ctypes.data))
        freq = np.ascontiguousarray(freq, np.float64)
        if freq.shape != (pairs,):
            raise MoebiusError(1, f"rope: {pairs} frequencies")
        self.freq = DeviceArray.from_numpy(ctx, freq)
        self._dims = (ctypes.c_uint32 * 4)(*self.axis_dims)

    def _args(self, positions: DeviceArray, inverse: bool):
        axes, shape = len(self.axis_dims), positions.shape
        if positions.dtype != _I32 or len(shape) != 2 or shape[1] != axes:
            raise MoebiusError(1, f"positions are int32 [rows][{axes}]")
        return ctypes.byref(_lib.Rope(positions.ptr, shape[0], self.freq.ptr, axes, self._dims, self.pairing,
                                      1 if inverse else 0, 0))


def rope_axes(x: Heads, positions: DeviceArray, rope: RopeAxes, out: Heads, inverse: bool = False):
    """out = x turned by its rows' positions [pos_rows, axes] (row r by positions[r % pos_rows]);
    out may be x. inverse: by the negative angles."""
    _same(x, out)
    if x.rows != out.rows or x.heads != out.heads:
        raise MoebiusError(1, "x and out differ in shape")
    st = lib().mh_rope_axes(x.ctx.h, x.ptr, x.code, x.rows, x.heads, x.d, x.ld, rope._args(positions, inverse), out.ptr,
                            out.ld)
    if st:
        check(st)


def qk_norm_rope(q: Heads, k: Heads, gamma_q: DeviceArray | None, gamma_k: DeviceArray | None, eps: float,
                 positions: DeviceArray, rope: RopeAxes, q_out: Heads, k_out: Heads):
    """RMS norm (scales gamma [d], None: ones) of every query and key head, then the rotation,
    in one pass; outputs may be their inputs."""
    _same(q, k, q_out, k_out)
    rows = q.rows
    if not (rows == k.rows == q_out.rows == k_out.rows and q.heads == q_out.heads and k.heads == k_out.heads):
        raise MoebiusError(1, "q, k and their outputs differ in shape")
    for g in (gamma_q, gamma_k):
        if g is not None and (g.dtype != _F32 or g.nbytes != 4 * q.d):
            raise MoebiusError(1, "gamma is f32 of the head's channels")
    st = lib().mh_qk_norm_rope(q.ctx.h, q.ptr, q.ld, q.heads, k.ptr, k.ld, k.heads, q.code, rows, q.d, _ptr(gamma_q),
                               _ptr(gamma_k), eps, rope._args(positions, False), q_out.ptr, q_out.ld, k_out.ptr,
                               k_out.ld)
    if st:
        check(st)


def block_means(x: Heads, block: int, means: DeviceArray, length: DeviceArray | None = None,
                first: DeviceArray | None = None):
    """means [n, ceil(tokens / block), heads, d] f32: every block's mean over its tokens below
    length [n]; blocks at or below first [n] and those behind the length are left as they were."""
    blocks = -(-x.tokens // max(int(block), 1))
    if means.dtype != _F32 or means.nbytes != 4 * x.n * blocks * x.heads * x.d:
        raise MoebiusError(1, "means are f32 [n, blocks, heads, d]")
    _int32(length, x.n, "length")
    _int32(first, x.n, "first")
    check(lib().mh_block_means(x.ctx.h, x.ptr, x.code, x.n, x.tokens, x.heads, x.d, x.ld, _ptr(first), _ptr(length),
                               int(block), means.ptr))


def _shape(q: Heads, kv_tokens, heads_kv, blocks: DeviceArray, q_block, kv_block, causal, q_len, kv_len):
    if blocks.dtype != _I32 or len(blocks.shape) != 4 or \
            blocks.shape[:3] != (q.n, -(-q.tokens // max(int(q_block), 1)), heads_kv):
        raise MoebiusError(1, "blocks are int32 [n, blocks of queries, key heads, top]")
    _int32(q_len, q.n, "q_len")
    _int32(kv_len, q.n, "kv_len")
    return _lib.BlockShape(q.n, q.tokens, int(kv_tokens), q.heads, heads_kv, q.d, int(q_block), int(kv_block),
                           blocks.shape[3], int(causal), _ptr(q_len), _ptr(kv_len))


def block_select(q: Heads, means: DeviceArray, kv_tokens: int, blocks: DeviceArray, q_block: int = 64,
                 kv_block: int = 64, causal: bool = False, q_len: DeviceArray | None = None,
                 kv_len: DeviceArray | None = None):
    """blocks [n, ceil(q_tokens / q_block), key heads, top] int32: for every block of queries and key
    head the key blocks of the largest products of mean query and mean key (means of block_means),
    ascending, -1 behind the last."""
    heads_kv = blocks.shape[2] if len(blocks.shape) == 4 else 0
    s = _shape(q, kv_tokens, heads_kv, blocks, q_block, kv_block, causal, q_len, kv_len)
    nk = -(-int(kv_tokens) // max(int(kv_block), 1))
    if means.dtype != _F32 or means.nbytes != 4 * q.n * nk * heads_kv * q.d:
        raise MoebiusError(1, "means are f32 [n, blocks, key heads, d]")
    check(lib().mh_block_select(q.ctx.h, q.ptr, q.code, q.ld, ctypes.byref(s), means.ptr, blocks.ptr))


def block_attention(q: Heads, k: Heads, v: Heads, blocks: DeviceArray, out: Heads, scale: float | None = None,
                    q_block: int = 64, kv_block: int = 64, causal: bool = False, q_len: DeviceArray | None = None,
                    kv_len: DeviceArray | None = None, scratch: DeviceArray | None = None):
    """out = softmax(scale q . k) v over the keys of every block of queries' listed blocks
    (scale: 1 / sqrt(d) by default). scratch: block_attention_scratch bytes, for calls that are
    captured into a graph."""
    _same(q, k, v, out)
    if (k.n, k.tokens, k.heads) != (v.n, v.tokens, v.heads) or k.n != q.n or \
            (q.n, q.tokens, q.heads) != (out.n, out.tokens, out.heads):
        raise MoebiusError(1, "q, k, v and out differ in shape")
    s = _shape(q, k.tokens, k.heads, blocks, q_block, kv_block, causal, q_len, kv_len)
    check(lib().mh_block_attention(q.ctx.h, q.ptr, q.ld, k.ptr, k.ld, v.ptr, v.ld, q.code, ctypes.byref(s), blocks.ptr,
                                   1.0 / math.sqrt(q.d) if scale is None else float(scale), out.ptr, out.ld,
                                   _ptr(scratch), 0 if scratch is None else scratch.nbytes))


def block_attention_scratch(q: Heads, k: Heads, blocks: DeviceArray, q_block: int = 64, kv_block: int = 64) -> int:
    """Bytes of scratch that block_attention needs for these shapes."""
    s = _shape(q, k.tokens, k.heads, blocks, q_block, kv_block, False, None, None)
    n = ctypes.c_uint64()
    check(lib().mh_block_attention_scratch(q.ctx.h, q.code, ctypes.byref(s), ctypes.byref(n)))
    return int(n.value)
