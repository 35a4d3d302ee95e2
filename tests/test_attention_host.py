"""Refusals of the transformer entry points (include/moebius_hip.h), which come
before the context is looked at, so no device is needed; and the frequencies'
host function."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from moebius_cpu_amd import _lib

A16 = 0x100000  # addresses that the checks read as numbers only


def refused(status, text):
    assert status == _lib.ERR_INVALID_ARGUMENT
    msg = _lib.lib().mh_last_error().decode()
    assert text in msg, msg


def rope(**kw):
    a = dict(positions=A16, pos_rows=4, freq=A16, axes=2, axis_dims=(8, 8, 0, 0), pairing=0, inverse=0, reserved=0)
    a.update(kw)
    a["axis_dims"] = (ctypes.c_uint32 * 4)(*a["axis_dims"])
    return _lib.Rope(*(a[f] for f, _ in _lib.Rope._fields_))


def rope_call(r=None, x=A16, out=A16 + 0x100000, rows=4, heads=2, d=16, ld=32, ld_out=32, dtype=0):
    r = rope() if r is None else r
    return _lib.lib().mh_rope_axes(None, x, dtype, rows, heads, d, ld, ctypes.byref(r), out, ld_out)


@pytest.mark.parametrize("kw,text", [
    (dict(r=rope(axes=0)), "1 to 4 axes"), (dict(r=rope(axes=5)), "1 to 4 axes"),
    (dict(r=rope(axis_dims=(7, 8, 0, 0))), "even"), (dict(r=rope(axis_dims=(0, 8, 0, 0))), "even"),
    (dict(r=rope(axis_dims=(8, 10, 0, 0))), "exceed the head"), (dict(r=rope(pairing=2)), "unknown pairing"),
    (dict(r=rope(pos_rows=0)), "no positions"), (dict(r=rope(positions=None)), "positions is NULL"),
    (dict(r=rope(freq=None)), "freq is NULL"), (dict(r=rope(freq=A16 + 4)), "not aligned"),
    (dict(r=rope(reserved=1)), "reserved"),
    (dict(dtype=2), "dtype"), (dict(heads=0), "no heads"), (dict(d=0), "no heads"), (dict(ld=31), "ld is less"),
    (dict(ld_out=16), "ld is less"), (dict(x=None), "x is NULL"), (dict(out=None), "out is NULL"),
    (dict(x=A16 + 2), "not aligned"), (dict(rows=1 << 31), "2^31"), (dict(ld=1 << 41), "too large"),
    (dict(out=A16 + 64), "overlap"),                 # half a head on
    (dict(out=A16, ld_out=33), "overlap"),           # the same place with another step
    (dict(out=A16 - 32 * 4 * 3), "overlap"),         # one row's reach before
    (dict(), "context is NULL"), (dict(out=A16), "context is NULL"),           # in place: fine
    (dict(ld=96, ld_out=96, out=A16 + 64 * 4), "context is NULL"),             # other columns of the same rows
    (dict(ld=96, ld_out=96, out=A16 + 80 * 4), "overlap"),                     # ... wrapping into the next
])
def test_rope_refusals(kw, text):
    refused(rope_call(**kw), text)


def qk_call(q=A16, k=A16 + 0x10000, qo=A16 + 0x20000, ko=A16 + 0x30000, lds=(32, 16, 32, 16), heads=(2, 1), d=16, rows=4,
            eps=1e-6, dtype=0, r=None, gammas=(None, None)):
    r = rope() if r is None else r
    return _lib.lib().mh_qk_norm_rope(None, q, lds[0], heads[0], k, lds[1], heads[1], dtype, rows, d, *gammas, eps,
                                      ctypes.byref(r), qo, lds[2], ko, lds[3])


@pytest.mark.parametrize("kw,text", [
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"),
    (dict(heads=(0, 1)), "no heads"), (dict(heads=(2, 0)), "no heads"), (dict(qo=A16 + 0x10000), "overlap"),
    (dict(ko=A16), "overlap"), (dict(ko=A16 + 0x20000), "overlap"), (dict(k=None), "k is NULL"),
    (dict(dtype=7), "dtype"), (dict(rows=1 << 31), "2^31"), (dict(r=rope(axis_dims=(16, 16, 0, 0))), "exceed"),
    (dict(gammas=(A16 + 2, None)), "gamma_q is not aligned"), (dict(gammas=(None, A16 + 1)), "gamma_k is not aligned"),
    (dict(), "context is NULL"), (dict(qo=A16, ko=A16 + 0x10000), "context is NULL"),
    # queries and keys of one projection turned where they lie
    (dict(k=A16 + 32 * 4, qo=A16, ko=A16 + 32 * 4, lds=(64, 64, 64, 64)), "context is NULL"),
])
def test_qk_norm_refusals(kw, text):
    refused(qk_call(**kw), text)


def shape(**kw):
    a = dict(n=2, q_tokens=64, kv_tokens=256, heads_q=4, heads_kv=2, d=64, q_block=16, kv_block=32, top=4, causal=0,
             q_len=None, kv_len=None)
    a.update(kw)
    return _lib.BlockShape(*(a[f] for f, _ in _lib.BlockShape._fields_))


SHAPES = [(dict(heads_q=3), "multiple"), (dict(heads_kv=0), "no heads"), (dict(heads_q=0), "no heads"),
          (dict(d=0), "no heads"), (dict(d=257), "256 channels"), (dict(q_block=0), "q_block"),
          (dict(q_block=1025), "q_block"), (dict(kv_block=0), "kv_block"), (dict(kv_block=48), "kv_block"),
          (dict(kv_block=256), "kv_block"), (dict(top=0), "top is"), (dict(top=1025), "top is"),
          (dict(q_len=A16 + 2), "not aligned"), (dict(n=1 << 31), "too large"),
          (dict(heads_q=65537, heads_kv=1, d=1), "65536")]


@pytest.mark.parametrize("kw,text", SHAPES + [
    (dict(kv_tokens=16 * 8193, kv_block=16), "8192 blocks"),
    # 64 tokens lie in two blocks of 32 or, from another first one on, in three
    (dict(causal=1, q_block=64, kv_block=32, top=2), "own tokens"),
    (dict(causal=1, q_block=64, kv_block=32, top=3), "context is NULL"),
    (dict(causal=1, q_block=64, kv_block=32, top=2, kv_tokens=64), "context is NULL"),  # there are no more
    (dict(), "context is NULL")])
def test_select_refusals(kw, text):
    s = shape(**kw)
    ld = max(s.heads_q * s.d, 1) if s.n < 1 << 30 else 256
    refused(_lib.lib().mh_block_select(None, A16, 0, ld, ctypes.byref(s), A16, A16), text)


def test_select_null_arguments():
    s = shape()
    L = _lib.lib()
    refused(L.mh_block_select(None, None, 0, 256, ctypes.byref(s), A16, A16), "q is NULL")
    refused(L.mh_block_select(None, A16, 0, 256, ctypes.byref(s), None, A16), "k_means is NULL")
    refused(L.mh_block_select(None, A16, 0, 256, ctypes.byref(s), A16, None), "blocks is NULL")
    refused(L.mh_block_select(None, A16, 0, 256, None, A16, A16), "shape is NULL")
    refused(L.mh_block_select(None, A16, 0, 255, ctypes.byref(s), A16, A16), "ld is less")
    refused(L.mh_block_select(None, A16, 3, 256, ctypes.byref(s), A16, A16), "dtype")
    refused(L.mh_block_select(None, A16, 0, 256, ctypes.byref(s), A16 + 2, A16), "k_means is not aligned")
    refused(L.mh_block_select(None, A16, 0, 256, ctypes.byref(s), A16, A16 + 2), "blocks is not aligned")


M = 1 << 24


def attend(s=None, q=M, k=2 * M, v=3 * M, out=4 * M, lds=(256, 128, 128, 256), dtype=1, blocks=A16, scale=0.125):
    s = shape() if s is None else s
    return _lib.lib().mh_block_attention(None, q, lds[0], k, lds[1], v, lds[2], dtype, ctypes.byref(s), blocks, scale,
                                         out, lds[3], None, 0)


@pytest.mark.parametrize("kw,text", SHAPES)
def test_attention_shape_refusals(kw, text):
    refused(attend(shape(**kw), lds=(4096,) * 4), text)


@pytest.mark.parametrize("kw,text", [
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(q=None), "q is NULL"), (dict(k=None), "k is NULL"),
    (dict(v=None), "v is NULL"), (dict(out=None), "out is NULL"), (dict(blocks=None), "blocks is NULL"),
    (dict(out=M), "overlap"), (dict(out=2 * M), "overlap"), (dict(out=3 * M + 64), "overlap"),
    (dict(lds=(255, 128, 128, 256)), "ld is less"), (dict(lds=(256, 127, 128, 256)), "ld is less"),
    (dict(lds=(256, 1 << 24, 128, 256)), "32 MiB"), (dict(lds=(256, 128, 1 << 24, 256)), "32 MiB"),
    (dict(dtype=9), "dtype"), (dict(k=2 * M + 1), "not aligned"), (dict(blocks=A16 + 1), "blocks is not aligned"),
    (dict(), "context is NULL")])
def test_attention_refusals(kw, text):
    refused(attend(**kw), text)


@pytest.mark.parametrize("kw,text", [(dict(block=0), "block is"), (dict(block=1025), "block is"), (dict(x=None), "x is NULL"),
                                     (dict(means=None), "means is NULL"), (dict(ld=63), "ld is less"),
                                     (dict(heads=0), "no heads"), (dict(dtype=5), "dtype"),
                                     (dict(first=A16 + 2), "first is not"), (dict(len=A16 + 2), "len is not"),
                                     (dict(means=A16 + 2), "means is not"), (dict(), "context is NULL")])
def test_means_refusals(kw, text):
    a = dict(x=A16, dtype=0, n=1, tokens=10, heads=1, d=64, ld=64, first=None, len=None, block=16, means=A16)
    a.update(kw)
    refused(_lib.lib().mh_block_means(None, *a.values()), text)


def lora_call(ad=None, x=M, out=2 * M, w=3 * M, slot=A16, rows=8, ci=64, co=32, per=1, bias=None, res=None,
              **kw):
    a = dict(a=4 * M, b=5 * M, scale=A16, dtype=0, slots=2, rank=8, reserved=0)
    a.update(kw)
    s = _lib.AdapterSet(*(a[f] for f, _ in _lib.AdapterSet._fields_)) if ad is None else ad
    return _lib.lib().mh_conv1x1_lora(None, x, rows, ci, w, 0, co, bias, res, ctypes.byref(s), slot, per, out, None, 0)


@pytest.mark.parametrize("kw,text", [
    (dict(rank=0), "rank"), (dict(rank=257), "rank"), (dict(a=None), "adapters a"), (dict(b=None), "adapters b"),
    (dict(scale=None), "adapters scale"), (dict(dtype=4), "dtype"), (dict(reserved=1), "reserved"),
    (dict(a=4 * M + 2), "not aligned"), (dict(x=None), "x is NULL"), (dict(out=None), "out is NULL"),
    (dict(w=None), "weight is NULL"), (dict(slot=None), "slot is NULL"), (dict(per=0), "rows_per_slot"),
    (dict(rows=1 << 31), "2^31"), (dict(ci=0), "empty channel"), (dict(co=0), "empty channel"),
    (dict(out=M + 256), "overlap"), (dict(res=2 * M + 64), "overlap"), (dict(res=2 * M), "context is NULL"),
    (dict(w=3 * M + 2), "weight is not aligned"), (dict(ci=(1 << 22) + 1), "2^22 channels"), (dict(co=(1 << 22) + 1), "2^22 channels"),
    *((dict([(f, A16 + 2)]), "x, out, bias") for f in ("x", "out", "bias", "res", "slot", "scale")),
    (dict(), "context is NULL"), (dict(slots=0, a=None, b=None), "context is NULL")])
def test_lora_refusals(kw, text):
    refused(lora_call(**kw), text)


def test_scratch_refusals():
    L, n = _lib.lib(), ctypes.c_uint64()
    refused(L.mh_conv1x1_lora_scratch(None, 8, 64, 32, 0, 0, ctypes.byref(n)), "rank")
    refused(L.mh_conv1x1_lora_scratch(None, 8, 64, 32, 0, 8, None), "bytes is NULL")
    refused(L.mh_conv1x1_lora_scratch(None, 8, 64, 32, 9, 8, ctypes.byref(n)), "dtype")
    refused(L.mh_block_attention_scratch(None, 0, ctypes.byref(shape()), None), "bytes is NULL")
    refused(L.mh_block_attention_scratch(None, 0, ctypes.byref(shape()), ctypes.byref(n)), "context is NULL")


def test_frequencies():
    dims = (ctypes.c_uint32 * 3)(4, 8, 2)
    f = np.zeros(7)
    assert _lib.lib().mh_rope_frequencies(10000.0, 3, dims, f.ctypes.data) == _lib.OK
    want = np.concatenate([10000.0 ** (-np.arange(0, m, 2) / m) for m in (4, 8, 2)])
    assert np.abs(f / want - 1).max() < 1e-14
    L = _lib.lib()
    refused(L.mh_rope_frequencies(0.0, 3, dims, f.ctypes.data), "theta")
    refused(L.mh_rope_frequencies(float("inf"), 3, dims, f.ctypes.data), "theta")
    refused(L.mh_rope_frequencies(1e4, 0, dims, f.ctypes.data), "axes")
    refused(L.mh_rope_frequencies(1e4, 3, (ctypes.c_uint32 * 3)(4, 3, 2), f.ctypes.data), "even")
    refused(L.mh_rope_frequencies(1e4, 3, None, f.ctypes.data), "NULL")
