"""Refusals of the cache in 8 bits, its attention and the gated norms, which come before
the context is looked at, so no device is needed; and the sizes' host function."""
from __future__ import annotations

import ctypes

import pytest

from moebius_cpu_amd import _lib

A = 0x1000000  # addresses that the checks read as numbers only
NONE = "context is NULL"  # every check passed


def refused(status, text):
    assert status == _lib.ERR_INVALID_ARGUMENT
    msg = _lib.lib().mh_last_error().decode()
    assert text in msg, msg


def make(cls, base, kw):
    a = {**base, **kw}
    return ctypes.byref(cls(*(a[f] for f, _ in cls._fields_)))


def cache(**kw):
    return make(_lib.Cache8, dict(k=A, v=A + 0x100000, k_scale=A + 0x200000, v_scale=A + 0x201000, pages=8, heads=2, d=40,
                                  block=32), kw)


def table(**kw):
    return make(_lib.PageTable, dict(pages=A + 0x300000, n=2, blocks=4), kw)


BAD_CACHE = [
    (dict(pages=0), "no pages"), (dict(heads=0), "no heads"), (dict(d=0), "no heads"), (dict(d=257), "256"),
    (dict(block=24), "block is 16"), (dict(block=256), "block is 16"), (dict(k=None), "cache k is NULL"),
    (dict(v_scale=None), "v_scale is NULL"), (dict(k=A + 8), "16-byte"), (dict(k_scale=A + 0x200002), "not aligned"),
    (dict(pages=1 << 31), "too large"), (dict(pages=1 << 30, heads=1 << 11), "too large")]
BAD_TABLE = [(dict(pages=None), "table pages is NULL"), (dict(pages=A + 2), "not aligned"), (dict(blocks=1 << 26), "2^30 tokens"),
             (dict(n=1 << 31), "too large")]


@pytest.mark.parametrize("pages,heads,d,block,codes", [(1, 1, 1, 16, 256), (8, 2, 40, 32, 8 * 2 * 32 * 48),
                                                       (1 << 20, 8, 128, 64, 1 << 36)])
def test_sizes(pages, heads, d, block, codes):
    a, b = ctypes.c_uint64(), ctypes.c_uint64()
    _lib.check(_lib.lib().mh_cache8_sizes(pages, heads, d, block, ctypes.byref(a), ctypes.byref(b)))
    assert (a.value, b.value) == (codes, pages * heads * 4)
    refused(_lib.lib().mh_cache8_sizes(pages, heads, d, 8, ctypes.byref(a), ctypes.byref(b)), "block is 16")
    refused(_lib.lib().mh_cache8_sizes(pages, heads, d, block, None, ctypes.byref(b)), "code_bytes is NULL")


def move(fn, c=None, t=None, k=A + 0x400000, ld_k=80, v=A + 0x500000, ld_v=80, dtype=0, tokens=64, first=None, length=None):
    return getattr(_lib.lib(), fn)(None, c or cache(), t or table(), k, ld_k, v, ld_v, dtype, tokens, first, length)


@pytest.mark.parametrize("fn", ["mh_cache8_write", "mh_cache8_read"])
@pytest.mark.parametrize("kw,text", [
    *((dict(c=cache(**c)), m) for c, m in BAD_CACHE), *((dict(t=table(**t)), m) for t, m in BAD_TABLE),
    (dict(dtype=2), "dtype"), (dict(k=None), "k is NULL"), (dict(v=None), "v is NULL"), (dict(ld_k=79), "ld is less"),
    (dict(k=A + 0x400002), "not aligned"), (dict(tokens=1 << 31), "too large"), (dict(first=A + 1), "first is not aligned"),
    (dict(length=A + 1), "len is not aligned"), (dict(k=A + 64), "overlap"), (dict(v=A + 0x200000), "overlap"),
    (dict(), NONE), (dict(k=None, v=None, tokens=0), NONE), (dict(t=table(n=0, pages=None), k=None, v=None), NONE)])
def test_write_and_read_refusals(fn, kw, text):
    refused(move(fn, **kw), text)


def test_write_alone():
    refused(move("mh_cache8_write", c=cache(v=A)), "the arrays of the cache overlap")
    refused(move("mh_cache8_write", c=cache(v_scale=A + 0x200000)), "the arrays of the cache overlap")
    refused(move("mh_cache8_write", first=A + 0x100000), "overlap")
    refused(move("mh_cache8_write", t=table(pages=A)), "overlap")
    refused(move("mh_cache8_write", v=A + 0x400000), NONE)  # both from one tensor


def test_read_alone():
    refused(move("mh_cache8_read", v=A + 0x400000), "k and v overlap")
    refused(move("mh_cache8_read", k=A + 0x300000), "overlap")
    refused(move("mh_cache8_read", first=A + 0x400000), "overlap")


def shape(**kw):
    return make(_lib.CacheAttention, dict(q_tokens=16, heads_q=4, causal=1, window=0, sinks=0, reserved=0, q_len=None,
                                          kv_len=None), kw)


def attend(q=A + 0x400000, ld_q=160, dtype=0, s=None, c=None, t=None, scale=0.1, out=A + 0x500000, ld_out=160, scratch=None,
           size=0):
    return _lib.lib().mh_cache8_attention(None, q, ld_q, dtype, s or shape(), c or cache(), t or table(), scale, out, ld_out,
                                          scratch, size)


@pytest.mark.parametrize("kw,text", [
    *((dict(c=cache(**c)), m) for c, m in BAD_CACHE), *((dict(t=table(**t)), m) for t, m in BAD_TABLE),
    (dict(s=shape(heads_q=3)), "multiple"), (dict(s=shape(heads_q=0)), "no heads"), (dict(s=shape(reserved=1)), "reserved"),
    (dict(s=shape(sinks=4)), "sinks without"), (dict(s=shape(window=1 << 31)), "too large"),
    (dict(s=shape(window=4, sinks=1 << 31)), "too large"), (dict(s=shape(q_len=A + 1)), "q_len is not aligned"),
    (dict(s=shape(kv_len=A + 1)), "kv_len is not aligned"), (dict(s=shape(heads_q=1 << 18)), "65536"),
    (dict(s=shape(q_tokens=1 << 30)), "2^30"), (dict(dtype=3), "dtype"), (dict(q=None), "q is NULL"),
    (dict(out=None), "out is NULL"), (dict(ld_q=100), "ld is less"), (dict(out=A + 0x400000), "overlap"),
    (dict(out=A), "overlap"), (dict(out=A + 0x201000), "overlap"), (dict(out=A + 0x300000), "overlap"),
    (dict(s=shape(kv_len=A + 0x500000)), "overlap"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(), NONE), (dict(s=shape(window=1, sinks=1 << 30)), NONE),
    (dict(s=shape(q_tokens=0), q=None, out=None), NONE)])
def test_attention_refusals(kw, text):
    refused(attend(**kw), text)


def norm(**kw):
    return _lib.Norm(*(kw.get(f, d) for f, d in (("kind", 0), ("eps", 1e-6), ("gamma", None), ("beta", None))))


def gated(**kw):
    a = dict(x=A, branch=A + 0x10000, x_out=A + 0x20000, y=A + 0x30000, ld_x=64, ld_branch=64, ld_x_out=64, ld_y=64, x_dtype=0,
             branch_dtype=0, rows=8, rows_per_item=4, c=64, keep=1.0, post=norm(), pre=norm(kind=2), gate=A + 0x40000,
             scale=A + 0x40100, shift=A + 0x40200, ld_gate=192, ld_scale=192, ld_shift=192)
    a.update(kw)
    return _lib.lib().mh_gated_norm(None, ctypes.byref(_lib.GatedNorm(*(a[f] for f, _ in _lib.GatedNorm._fields_))))


@pytest.mark.parametrize("kw,text", [
    (dict(rows=1 << 31), "2^31 rows"), (dict(rows_per_item=0), "rows_per_item"), (dict(rows_per_item=1 << 31), "rows_per_item"),
    (dict(c=0), "c is 1"), (dict(c=32769, ld_x=1 << 16), "c is 1"), (dict(keep=float("nan")), "keep"),
    (dict(x_dtype=2), "dtype"), (dict(branch_dtype=9), "dtype"), (dict(x=None), "x is NULL"), (dict(ld_y=63), "ld is less"),
    (dict(x=A + 2), "not aligned"), (dict(gate=A + 0x40002), "not aligned"), (dict(ld_gate=8), "ld is less"),
    (dict(post=norm(kind=3)), "unknown norm"), (dict(pre=norm(kind=2, eps=-1.0)), "eps"),
    (dict(pre=norm(kind=1, eps=float("nan"))), "eps"), (dict(post=norm(gamma=A)), "without a norm"),
    (dict(branch=None), "without a branch"), (dict(branch=None, gate=None, post=norm(kind=1)), "without a branch"),
    (dict(y=None), "without y"), (dict(y=None, pre=norm(), scale=None, shift=None, x_out=None), "neither"),
    (dict(y=A + 0x20000), "x_out and y overlap"), (dict(x_out=A + 4), "overlap"), (dict(x_out=A, ld_x_out=65), "overlap"),
    (dict(y=A, branch_dtype=1), "overlap"), (dict(y=A + 0x40000), "overlap"), (dict(x_out=A + 0x40100), "overlap"),
    (dict(pre=norm(kind=2, beta=A + 0x20000)), "overlap"), (dict(), NONE), (dict(x_out=A, y=A + 0x10000), NONE),
    (dict(x_out=A + 0x10000, y=A), NONE), (dict(branch=None, gate=None), NONE),
    (dict(y=None, pre=norm(), scale=None, shift=None), NONE), (dict(rows=0, x=None, branch=None, gate=None), NONE)])
def test_gated_norm_refusals(kw, text):
    refused(gated(**kw), text)
