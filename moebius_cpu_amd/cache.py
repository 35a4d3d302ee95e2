"""A cache of keys and values in 8 bits for streams of tokens, and attention over
it, causal or not, with a sliding window and a few first tokens that stay visible.
Thin calls of libmoebius_hip.so (include/moebius_hip.h mh_cache8_*); the reference
has no counterpart.

    cache = Cache8(ctx, pages=512, heads=8, d=128, block=64)
    table = DeviceArray.from_numpy(ctx, pages_of_each_item)         # int32 [n, blocks], -1: no page
    cache_write(cache, table, k, v, first=lengths)                  # behind the tokens that it holds
    cache_attention(q, cache, table, out, window=4096, sinks=64, kv_len=lengths_with_them)
"""
from __future__ import annotations

import ctypes
import math
import struct

import numpy as np

from . import _lib
from ._lib import MoebiusError, check, lib
from .attention import Heads, _int32, _same
from .engine import Context, DeviceArray, _ptr

_I32 = np.dtype(np.int32)
# _lib.PageTable and _lib.CacheAttention, packed: single tokens take no longer on the device than here.
_TABLE, _SHAPE = struct.Struct("=Q2I").pack, struct.Struct("=6I2Q").pack


class Cache8:
    """Pages of `block` tokens (16, 32, 64 or 128) of `heads` heads of d channels, keys and values in
    8 bits with an f32 scale for each page and head."""

    def __init__(self, ctx: Context, pages: int, heads: int, d: int, block: int = 64):
        codes, scales = ctypes.c_uint64(), ctypes.c_uint64()
        check(lib().mh_cache8_sizes(int(pages), int(heads), int(d), int(block), ctypes.byref(codes),
                                    ctypes.byref(scales)))
        self.ctx, self.pages, self.heads, self.d, self.block = ctx, int(pages), int(heads), int(d), int(block)
        self.k, self.v = (DeviceArray(ctx, (codes.value,), np.uint8) for _ in range(2))
        self.k_scale, self.v_scale = (DeviceArray(ctx, (self.pages, self.heads)) for _ in range(2))
        self.c = _lib.Cache8(self.k.ptr, self.v.ptr, self.k_scale.ptr, self.v_scale.ptr, self.pages, self.heads,
                             self.d, self.block)
        self._ref = ctypes.byref(self.c)

    @property
    def nbytes(self) -> int:
        return 2 * (self.k.nbytes + self.k_scale.nbytes)


def _table(cache: Cache8, table: DeviceArray, n: int):
    if table.dtype != _I32 or len(table.shape) != 2 or table.shape[0] != n:
        raise MoebiusError(1, "table is int32 [n, blocks]")
    if table.ctx is not cache.ctx:
        raise MoebiusError(1, "table and cache of different contexts")
    return _TABLE(table.ptr, n, table.shape[1])


def _rows(cache: Cache8, k: Heads, v: Heads):
    _same(k, v)
    if (k.n, k.tokens, k.heads) != (v.n, v.tokens, v.heads) or k.heads != cache.heads or k.d != cache.d:
        raise MoebiusError(1, "k and v differ from each other or from the cache in heads or channels")
    if k.ctx is not cache.ctx:
        raise MoebiusError(1, "heads and cache of different contexts")


def cache_write(cache: Cache8, table: DeviceArray, k: Heads, v: Heads, first: DeviceArray | None = None,
                length: DeviceArray | None = None):
    """Quantises tokens t < length [n] of k and v into the cache as tokens first [n] + t of each item
    (None: all of them, from 0). A block that holds tokens already keeps the larger scale."""
    _rows(cache, k, v)
    _int32(first, k.n, "first")
    _int32(length, k.n, "length")
    st = lib().mh_cache8_write(cache.ctx.h, cache._ref, _table(cache, table, k.n), k.ptr, k.ld, v.ptr, v.ld, k.code,
                               k.tokens, _ptr(first), _ptr(length))
    if st:
        check(st)


def cache_read(cache: Cache8, table: DeviceArray, k: Heads, v: Heads, first: DeviceArray | None = None,
               length: DeviceArray | None = None):
    """Rows t < length [n] of k and v = what the cache holds of tokens first [n] + t; other rows are
    left as they were."""
    _rows(cache, k, v)
    _int32(first, k.n, "first")
    _int32(length, k.n, "length")
    st = lib().mh_cache8_read(cache.ctx.h, cache._ref, _table(cache, table, k.n), k.ptr, k.ld, v.ptr, v.ld, k.code,
                              k.tokens, _ptr(first), _ptr(length))
    if st:
        check(st)


def _shape(q: Heads, cache: Cache8, causal, window, sinks, q_len, kv_len):
    if q.d != cache.d:
        raise MoebiusError(1, "q and cache differ in channels")
    if q.ctx is not cache.ctx:
        raise MoebiusError(1, "heads and cache of different contexts")
    if not (0 <= window < 1 << 32 and 0 <= sinks < 1 << 32):
        raise MoebiusError(1, "window and sinks are not negative, and below 2^32")
    _int32(q_len, q.n, "q_len")
    _int32(kv_len, q.n, "kv_len")
    return _SHAPE(q.tokens, q.heads, bool(causal), int(window), int(sinks), 0, 0 if q_len is None else q_len.ptr,
                  0 if kv_len is None else kv_len.ptr)


def cache_attention(q: Heads, cache: Cache8, table: DeviceArray, out: Heads, scale: float | None = None,
                    causal: bool = True, window: int = 0, sinks: int = 0, q_len: DeviceArray | None = None,
                    kv_len: DeviceArray | None = None, scratch: DeviceArray | None = None):
    """out = softmax(scale q . k) v over the cache (scale: 1 / sqrt(d) by default). Row t of item i stands
    at t + kv_len[i] - q_len[i]; window 0: no window. scratch: cache_attention_scratch bytes, for calls
    that are captured into a graph."""
    _same(q, out)
    if (q.n, q.tokens, q.heads) != (out.n, out.tokens, out.heads):
        raise MoebiusError(1, "q and out differ in shape")
    s = _shape(q, cache, causal, window, sinks, q_len, kv_len)
    st = lib().mh_cache8_attention(cache.ctx.h, q.ptr, q.ld, q.code, s, cache._ref, _table(cache, table, q.n),
                                   1.0 / math.sqrt(q.d) if scale is None else float(scale), out.ptr, out.ld,
                                   _ptr(scratch), 0 if scratch is None else scratch.nbytes)
    if st:
        check(st)


def cache_attention_scratch(q: Heads, cache: Cache8, table: DeviceArray, window: int = 0, sinks: int = 0) -> int:
    """Bytes of scratch that cache_attention needs for these shapes."""
    n = ctypes.c_uint64()
    check(lib().mh_cache8_attention_scratch(cache.ctx.h, q.code, _shape(q, cache, True, window, sinks, None, None),
                                            cache._ref, _table(cache, table, q.n), ctypes.byref(n)))
    return int(n.value)
