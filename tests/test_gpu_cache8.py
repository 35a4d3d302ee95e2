"""The cache in 8 bits and the attention over it against their definitions in f64.

Codes and scales are whole results: equal, not near. Attention tolerances, for a row with
scores s_j (natural units) over keys whose values have codes of at most 127 and scales of at
most V (v = 127 V), worst cases of the roundings, u = 2^-24:
  - the f32 sum of a score's 2 d products and its scales: (2 d + 8) u A, A = max_j scale sum |q_i k_ij|;
    two f16 parts of q: u A more, and 2^-39 scale max|q| sum |k_ij| for values far below the largest;
  - the exponent's argument 2^-23 B, B = max |s_j| log2 e + 8, the exponential 2^-22;
  - the sums and their rescales (keys + tiles) u; all of these for numerator and denominator;
  - scales beside the probabilities: 2 u;
  - probabilities in one f16: 2^-11 of themselves, or 2^-24 v where they are below its normal
    range (half a step of 2^-24 at a scale of up to twice V), for every key; in two parts 2^-22 and 2^-35;
  - FAST contexts round q to f16: 2^-11 A, and 2^-25 of its largest;
  - f16 outputs add half a step.
"""
from __future__ import annotations

import numpy as np
import pytest

from moebius_cpu_amd import engine as E
from moebius_cpu_amd._lib import MoebiusError
from moebius_cpu_amd.attention import Heads
from moebius_cpu_amd.cache import Cache8, cache_attention, cache_attention_scratch, cache_read, cache_write
from tests.graph_capture import capture
from tests.test_gpu_block_attention import dev, heads, lens

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32 = np.float32


@pytest.fixture(scope="module")
def ctx():
    return E.Context(0)


# ---------------------------------------------------------------- the definition

class Held:
    """A cache on the host: codes [pages][heads][block][d] and scales [pages][heads], of keys and of values."""

    def __init__(self, pages, h, d, block):
        self.codes = np.zeros((2, pages, h, block, d), np.int64)
        self.scale = np.zeros((2, pages, h), F32)
        self.block, self.pages = block, pages

    def write(self, table, kv, first, length):
        for which, x in enumerate(kv):
            for i in range(x.shape[0]):
                cap = table.shape[1] * self.block
                f = min(max(int(first[i]), 0), cap)
                n = min(max(int(length[i]), 0), x.shape[1], cap - f)
                p = f
                while p < f + n:
                    b, lo = divmod(p, self.block)
                    hi = min(self.block, f + n - b * self.block)
                    page = table[i, b]
                    if 0 <= page < self.pages:
                        self.block_of(which, page, x[i, p - f:p - f + hi - lo], lo)
                    p = b * self.block + hi

    def block_of(self, which, page, x, lo):
        for h in range(x.shape[1]):
            v = x[:, h].astype(np.float64)
            fine = np.isfinite(v)
            s = F32(np.abs(v[fine]).max() if fine.any() else 0) * (F32(1) / F32(127))
            if lo:
                s0 = self.scale[which, page, h]
                s = max(s, s0)
                old = self.codes[which, page, h, :lo]
                if s > s0:
                    old[:] = np.clip(np.rint(old * np.float64(s0) / np.float64(s)), -127, 127)
            self.scale[which, page, h] = s
            with np.errstate(invalid="ignore", divide="ignore"):
                c = np.clip(np.rint(v / np.float64(s)), -127, 127) if s > 0 else np.zeros_like(v)
            self.codes[which, page, h, lo:lo + len(v)] = np.where(np.isnan(c), 0, c)

    def values(self, which, table, item, n):
        """[n][heads][d] f64 and whether each token has a page."""
        v = np.zeros((n, *self.codes.shape[2::2]))
        there = np.zeros(n, bool)
        for p in range(n):
            page = table[item, p // self.block]
            if 0 <= page < self.pages:
                there[p] = True
                v[p] = self.codes[which, page, :, p % self.block] * self.scale[which, page].astype(np.float64)[:, None]
        return v, there


def device_codes(cache):
    dp = -(-cache.d // 16) * 16
    k = cache.k.numpy().reshape(cache.pages, cache.heads, cache.block, dp)
    v = cache.v.numpy().reshape(cache.pages, cache.heads, dp, cache.block).transpose(0, 1, 3, 2)
    return [c[..., :cache.d].astype(np.int64) - 128 for c in (k, v)], [cache.k_scale.numpy(), cache.v_scale.numpy()]


def blank(cache):
    """Codes 128 (0) and scales 0 everywhere, as the host's copy begins."""
    for a in (cache.k, cache.v):
        a.upload(np.full(a.shape, 128, np.uint8))
    for a in (cache.k_scale, cache.v_scale):
        a.upload(np.zeros(a.shape, F32))


def same_state(cache, held, written):
    codes, scales = device_codes(cache)
    for which in (0, 1):
        assert np.array_equal(scales[which], held.scale[which])
        assert np.array_equal(codes[which][written], held.codes[which][written])


def pages(r, n, blocks, extra=3):
    return r.permutation(n * blocks + extra)[:n * blocks].reshape(n, blocks).astype(np.int32)


def mask_of(held, table, lengths):
    """Tokens of every page that have been written [pages][heads][block]."""
    m = np.zeros((held.pages, held.codes.shape[2], held.block), bool)
    for i, n in enumerate(lengths):
        for p in range(n):
            page = table[i, p // held.block]
            if 0 <= page < held.pages:
                m[page, :, p % held.block] = True
    return m


# ---------------------------------------------------------------- writing and reading

@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("n,tokens,h,d,block,pad,offset", [
    (1, 1, 1, 1, 16, 0, 0), (2, 130, 3, 40, 64, 0, 0), (1, 700, 8, 128, 128, 128, 8), (3, 50, 2, 33, 16, 1, 1),
    (1, 257, 4, 64, 32, 0, 0), (2, 129, 1, 256, 128, 8, 0), (5, 7, 2, 80, 32, 0, 8), (1, 300, 2, 72, 64, 4, 4)])
def test_write_and_read(ctx, dtype, n, tokens, h, d, block, pad, offset):
    r = np.random.default_rng(tokens + d)
    blocks = -(-tokens // block) + 1
    table = pages(r, n, blocks)
    length = r.integers(0, tokens + 1, n)
    length[0] = tokens
    kv = [(r.standard_normal((n, tokens, h, d)) * np.exp2(r.integers(-6, 6, (n, tokens, 1, 1)))).astype(dtype) for _ in range(2)]
    for x in kv:
        for i in range(n):
            x[i, length[i]:] = np.nan  # behind the length nothing counts
    cache, held = Cache8(ctx, n * blocks + 3, h, d, block), Held(n * blocks + 3, h, d, block)
    blank(cache)
    t, k, v = dev(ctx, table), *(heads(ctx, x, pad, offset) for x in kv)
    cache_write(cache, t, k, v, length=lens(ctx, length))
    held.write(table, kv, np.zeros(n, int), length)
    same_state(cache, held, mask_of(held, table, length))
    out = [heads(ctx, np.full((n, tokens + 5, h, d), 7, dtype), pad, offset) for _ in range(2)]
    cache_read(cache, t, *out, length=lens(ctx, length))
    for which, o in enumerate(out):
        got = o.numpy()
        flat = o.buf.numpy()
        assert np.isnan(flat[:offset]).all() and (not pad or np.isnan(flat[offset + h * d:offset + h * d + pad]).all())
        for i in range(n):
            want = held.values(which, table, i, length[i])[0].astype(F32).astype(dtype)
            assert np.array_equal(got[i, :length[i]], want)
            assert np.all(got[i, length[i]:] == 7)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("h,d,block", [(2, 40, 16), (1, 128, 64), (3, 65, 32), (2, 80, 128)])
def test_appended_step_by_step(ctx, dtype, h, d, block):
    """Runs of odd lengths behind one another, growing and shrinking in size, and a turn back."""
    r = np.random.default_rng(d)
    n, blocks = 3, 4
    table = pages(r, n, blocks)
    cache, held = Cache8(ctx, n * blocks + 3, h, d, block), Held(n * blocks + 3, h, d, block)
    blank(cache)
    t, at = dev(ctx, table), np.zeros(n, int)
    for step, run in enumerate([1, 1, 3, 1, 5, 1, 2, 17, 1, 40, 1, 1, 64, 1, 2, 1]):
        kv = [(r.standard_normal((n, run, h, d)) * np.exp2(r.integers(-5, 6))).astype(dtype) for _ in range(2)]
        length = r.integers(0, run + 1, n) if step % 3 == 2 else np.full(n, run)
        if step == 10:
            at = at - np.minimum(at, [1, 5, 0])
        cache_write(cache, t, heads(ctx, kv[0]), heads(ctx, kv[1]), first=lens(ctx, at), length=lens(ctx, length))
        held.write(table, kv, at, length)
        at = np.minimum(at + length, blocks * block)
        same_state(cache, held, mask_of(held, table, at))
    first, back = np.maximum(at - [9, 0, 30], 0), 33
    out = [heads(ctx, np.zeros((n, back, h, d), dtype)) for _ in range(2)]
    cache_read(cache, t, *out, first=lens(ctx, first), length=lens(ctx, at - first))
    for which, o in enumerate(out):
        got = o.numpy()
        for i in range(n):
            m = min(at[i] - first[i], back)
            want = held.values(which, table, i, at[i])[0][first[i]:first[i] + m]
            assert np.array_equal(got[i, :m], want.astype(F32).astype(dtype)) and np.all(got[i, m:] == 0)


def test_borders_and_special_values(ctx):
    """Ties between codes, scales whose inverse is inexact, tiny and huge values, infinities, NaN, zeros."""
    d, block = 64, 16
    x = np.zeros((1, 9 * block, 1, d), F32)
    half = np.arange(d) - 31.5
    x[0, :block, 0] = half                                   # scale of a largest value of 127: 1, ties everywhere
    x[0, 0, 0, 0] = 127
    x[0, block:2 * block, 0] = half * 3
    x[0, block, 0, 0] = 381                                   # scale 3
    s = F32(1.7) / F32(127)
    x[0, 2 * block:3 * block, 0] = ((half + 0) * np.float64(s)).astype(F32)
    x[0, 2 * block, 0, 0] = 1.7                               # next to ties on both sides
    x[0, 3 * block:4 * block, 0] = half * F32(1e-42)          # below the normal range
    x[0, 4 * block:5 * block, 0] = half * F32(1e37) / 32
    x[0, 5 * block:6 * block, 0] = half
    x[0, 5 * block, 0, :4] = [np.inf, -np.inf, np.nan, 0]
    x[0, 6 * block, 0, :2] = [np.inf, np.nan]                 # nothing finite but zeros
    x[0, 7 * block:8 * block] = np.nan
    near = np.nextafter(x[0, 2 * block:3 * block, 0], F32(9))
    x[0, 8 * block:9 * block, 0] = near
    x[0, 8 * block, 0, 0] = 1.7
    table = np.arange(9, dtype=np.int32)[None]
    cache, held = Cache8(ctx, 9, 1, d, block), Held(9, 1, d, block)
    blank(cache)
    kv = [x, -x]
    cache_write(cache, dev(ctx, table), heads(ctx, kv[0]), heads(ctx, kv[1]))
    held.write(table, kv, [0], [9 * block])
    same_state(cache, held, np.ones((9, 1, block), bool))


def test_pages_that_are_not_there(ctx):
    """Entries outside the cache: not written, not read, and nothing beside them either."""
    r = np.random.default_rng(1)
    table = np.array([[0, -1, 2, 7], [2**31 - 1, 1, -5, 3]], np.int32)
    x = [r.standard_normal((2, 64, 2, 24)).astype(F32) for _ in range(2)]
    cache, held = Cache8(ctx, 4, 2, 24, 16), Held(4, 2, 24, 16)
    blank(cache)
    t = dev(ctx, table)
    cache_write(cache, t, heads(ctx, x[0]), heads(ctx, x[1]))
    held.write(table, x, [0, 0], [64, 64])
    same_state(cache, held, np.ones((4, 2, 16), bool))
    out = [heads(ctx, np.full((2, 64, 2, 24), 7, F32)) for _ in range(2)]
    cache_read(cache, t, *out)
    for which, o in enumerate(out):
        for i in range(2):
            want, there = held.values(which, table, i, 64)
            assert np.array_equal(o.numpy()[i], np.where(there[:, None, None], want.astype(F32), 7))


def test_positions_out_of_range_are_clamped(ctx):
    r = np.random.default_rng(2)
    table = pages(r, 4, 2, 0)
    x = [r.standard_normal((4, 40, 1, 16)).astype(F32) for _ in range(2)]
    cache, held = Cache8(ctx, 8, 1, 16, 16), Held(8, 1, 16, 16)
    blank(cache)
    first, length = [-7, 30, 2**31 - 1, 5], [2**31 - 1, 40, 40, -9]
    cache_write(cache, dev(ctx, table), heads(ctx, x[0]), heads(ctx, x[1]), first=lens(ctx, first), length=lens(ctx, length))
    held.write(table, x, first, length)
    same_state(cache, held, np.ones((8, 1, 16), bool))


# ---------------------------------------------------------------- attention

def visible(ql, kl, causal, window, sinks):
    at = np.arange(ql)[:, None] + kl - ql
    j = np.arange(kl)[None]
    seen = (j <= at) if causal else np.ones((ql, kl), bool)
    if window:
        seen = seen & ((j > at - window) | (j < sinks))
    return seen


def attention64(q, held, table, scale, causal, window, sinks, q_len, kv_len, fast=False, below=None):
    """out and the bound on its error, NaN where rows are not there; below: the sums' exponent is at most that far
    above those of the values that a row sees."""
    n, qt, hq, d = q.shape
    hk = held.codes.shape[2]
    g, parts2 = hq // hk, q.dtype == F32 and not fast
    out = np.full(q.shape, np.nan)
    tol = np.full(q.shape, np.nan)
    for i in range(n):
        ql, kl = int(q_len[i]), int(kv_len[i])
        k, there = held.values(0, table, i, kl)
        v, _ = held.values(1, table, i, kl)
        seen = visible(ql, kl, causal, window, sinks) & there[None]
        for h in range(hq):
            x, kh, vh = q[i, :ql, h].astype(np.float64), k[:, h // g], v[:, h // g]
            if not kl:
                out[i, :ql, h], tol[i, :ql, h] = 0, 0
                continue
            s = scale * x @ kh.T
            a = (scale * np.abs(x) @ np.abs(kh).T).max(1)
            least = scale * np.abs(x).max(1) * np.abs(kh).sum(1).max()
            b = np.abs(s).max(1) * 1.4427 + 8
            m = np.where(seen, s, -np.inf).max(1, keepdims=True)
            p = np.where(seen, np.exp(s - np.where(np.isfinite(m), m, 0)), 0)
            z = p.sum(1, keepdims=True)
            o = p @ vh / np.where(z > 0, z, 1)
            page = [table[i, t] for t in range(-(-kl // held.block)) if 0 <= table[i, t] < held.pages]
            big = 127 * max([held.scale[1, pg, h // g] for pg in page], default=0)
            e = (2 * d + 9) * U * a + 2.0 ** -39 * least + 2.0 ** -23 * b + 2.0 ** -22 + (kl + kl / 64 + 4) * U
            if q.dtype == F32 and fast:
                e = e + 2.0 ** -11 * a + 2.0 ** -25 * least
            size = (p @ np.abs(vh) / np.where(z > 0, z, 1))  # what relative errors of p are of
            err = np.expm1(2 * e)[:, None] * size + (2.0 ** -22 if parts2 else 2.0 ** -11 * 1.001) * size + \
                kl * (2.0 ** -35 if parts2 else 2.0 ** -24) * big
            if below is not None:
                of = np.array([held.scale[1, pg, h // g] if 0 <= pg < held.pages else 0 for pg in table[i, np.arange(kl) // held.block]])
                big, keys = 127 * np.where(seen, of, 0).max(1) * 2.0 ** below, seen.sum(1)
                err = np.expm1(2 * e)[:, None] * size + (2.0 ** -22 if parts2 else 2.0 ** -11 * 1.001) * size + \
                    (keys * (2.0 ** -35 if parts2 else 2.0 ** -24) * big)[:, None]
            if q.dtype == np.float16:
                err = err + 2.0 ** -11 * (np.abs(o) + err) + 2.0 ** -25
            else:
                err = err + U * np.abs(o)
            out[i, :ql, h], tol[i, :ql, h] = o, err
    return out, tol


class Case:
    def __init__(self, ctx, dtype, n, q, kv, hq, hk, d, block, causal=True, window=0, sinks=0, q_len=None, kv_len=None, pad=0,
                 offset=0, absent=(), seed=0, std=1.5):
        r = np.random.default_rng(seed + kv + d)
        self.ctx, self.blocks = ctx, -(-kv // block)
        self.table = pages(r, n, self.blocks)
        for i, b in absent:
            self.table[i, b] = -1
        self.q_len = np.full(n, q) if q_len is None else np.asarray(q_len)
        self.kv_len = np.full(n, kv) if kv_len is None else np.asarray(kv_len)
        x = [(r.standard_normal((n, kv, hk, d)) * np.exp2(r.integers(-3, 3, (n, 1, hk, 1)))).astype(dtype) for _ in range(2)]
        self.held = Held(n * self.blocks + 3, hk, d, block)
        self.held.write(self.table, x, np.zeros(n, int), self.kv_len)
        self.cache = Cache8(ctx, n * self.blocks + 3, hk, d, block)
        for a in (self.cache.k, self.cache.v):  # what was never written is anything
            a.upload(r.integers(0, 256, a.shape).astype(np.uint8))
        for a in (self.cache.k_scale, self.cache.v_scale):
            a.upload(np.where(r.random(a.shape) < 0.5, np.nan, 3e38).astype(F32))
        self.dtable = dev(ctx, self.table)
        cache_write(self.cache, self.dtable, heads(ctx, x[0]), heads(ctx, x[1]), length=lens(ctx, self.kv_len))
        self.qh = (r.standard_normal((n, q, hq, d)) * std).astype(dtype)
        for i in range(n):
            self.qh[i, self.q_len[i]:] = np.nan
        self.q = heads(ctx, self.qh, pad, offset)
        self.out = heads(ctx, np.full(self.qh.shape, 7, dtype), pad, offset)
        self.kw = dict(causal=causal, window=window, sinks=sinks)
        self.lens = dict(q_len=lens(ctx, self.q_len), kv_len=lens(ctx, self.kv_len))

    def run(self, scratch=None, scale=None):
        cache_attention(self.q, self.cache, self.dtable, self.out, scale=scale, scratch=scratch, **self.kw, **self.lens)

    def check(self, fast=False, scale=None):
        want, tol = attention64(self.qh, self.held, self.table, 1 / np.sqrt(self.qh.shape[3]) if scale is None else scale,
                                *self.kw.values(), self.q_len, self.kv_len, fast)
        got = self.out.numpy().astype(np.float64)
        there = ~np.isnan(want)
        assert np.all(got[~there] == 7)  # behind the lengths: as they were
        off = np.abs(got - want)[there]
        assert np.all(off <= tol[there]), (off / np.maximum(tol[there], 1e-300)).max()


CASES = [
    dict(n=1, q=1, kv=1, hq=1, hk=1, d=1, block=16), dict(n=1, q=1, kv=300, hq=8, hk=8, d=80, block=32),
    dict(n=3, q=1, kv=2000, hq=8, hk=2, d=128, block=64, kv_len=[2000, 1, 777]),
    dict(n=2, q=1, kv=515, hq=32, hk=1, d=64, block=128, kv_len=[515, 0]),
    dict(n=2, q=5, kv=400, hq=6, hk=2, d=40, block=16, q_len=[5, 0], kv_len=[400, 33]),
    dict(n=1, q=3, kv=2, hq=2, hk=1, d=96, block=16, q_len=[3], kv_len=[2]),  # rows before the first token
    dict(n=2, q=70, kv=200, hq=4, hk=4, d=160, block=32, q_len=[70, 41], kv_len=[200, 41]),
    dict(n=1, q=33, kv=130, hq=3, hk=1, d=256, block=64), dict(n=1, q=9, kv=100, hq=2, hk=2, d=33, block=64, pad=1, offset=1),
    dict(n=1, q=130, kv=700, hq=4, hk=2, d=64, block=64, causal=False),
    dict(n=2, q=40, kv=500, hq=4, hk=2, d=72, block=32, window=100, sinks=10, q_len=[40, 7], kv_len=[500, 290]),
    dict(n=1, q=300, kv=900, hq=2, hk=1, d=128, block=128, window=1), dict(n=1, q=1, kv=3000, hq=4, hk=1, d=64, block=16, window=70, sinks=1),
    dict(n=1, q=64, kv=400, hq=2, hk=2, d=80, block=16, window=33, sinks=390, causal=False),
    dict(n=2, q=20, kv=300, hq=2, hk=1, d=48, block=16, absent=[(0, 0), (0, 3), (1, 17), (1, 18)]),
    dict(n=1, q=200, kv=333, hq=8, hk=1, d=128, block=32, pad=8, offset=8, window=128, sinks=64),
    dict(n=1, q=600, kv=1300, hq=2, hk=2, d=112, block=64), dict(n=1, q=257, kv=257, hq=4, hk=4, d=16, block=16),
    dict(n=1, q=150, kv=1000, hq=2, hk=1, d=200, block=128, causal=False, window=300, sinks=4),
]


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v) for v in c.values()).replace(" ", ""))
def test_attention(ctx, dtype, case):
    c = Case(ctx, dtype, **case)
    c.run()
    c.check()


# Rows enough to fill the card, so that waves share chunks: four waves (up to 128 rows of a key head, heads
# of 64 channels or of more than 128), and eight.
SHARED = [
    *(dict(n=64, q=70, kv=80, hq=4, hk=4, d=d, block=b, causal=c) for d, b, c in (
        (33, 16, True), (64, 64, False), (80, 32, True), (128, 128, True), (160, 16, False), (256, 64, True))),
    dict(n=64, q=35, kv=200, hq=8, hk=4, d=64, block=32, window=40, sinks=20, q_len=[35, 0, 7, 35] * 16, kv_len=[200, 90, 131, 35] * 16),
    dict(n=64, q=90, kv=150, hq=4, hk=4, d=96, block=64, window=64, absent=[(3, 1), (5, 0), (5, 1), (5, 2)], pad=8, offset=8),
    *(dict(n=32, q=130, kv=200, hq=8, hk=8, d=d, block=b, causal=c, window=w, sinks=s) for d, b, c, w, s in (
        (72, 16, True, 0, 0), (80, 64, True, 100, 9), (96, 32, False, 50, 70), (112, 128, True, 1, 0), (128, 64, True, 0, 0))),
    dict(n=32, q=70, kv=260, hq=16, hk=8, d=128, block=16, q_len=[70, 1, 33, 70] * 8, kv_len=[260, 1, 200, 70] * 8, absent=[(0, 3), (2, 0)]),
    dict(n=32, q=140, kv=64, hq=8, hk=8, d=65, block=64, pad=1, offset=1, kv_len=[64, 0, 1, 63] * 8, q_len=[140, 140, 1, 63] * 8),
    # few rows over many tokens: split
    dict(n=1, q=80, kv=4200, hq=2, hk=2, d=64, block=64, kv_len=[4001]), dict(n=2, q=90, kv=4500, hq=2, hk=1, d=80, block=32, kv_len=[4500, 333]),
    dict(n=1, q=200, kv=5000, hq=1, hk=1, d=128, block=128, window=4100, sinks=30), dict(n=2, q=70, kv=4200, hq=1, hk=1, d=200, block=16, kv_len=[700, 0]),
]


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("case", SHARED, ids=lambda c: "-".join(str(c[k]) for k in ("n", "q", "kv", "hk", "d", "block")))
def test_attention_of_many_rows(ctx, dtype, case):
    c = Case(ctx, dtype, **case)
    c.run()
    c.check()


@pytest.mark.parametrize("case", CASES[1:5] + CASES[9:11] + SHARED[1:4] + SHARED[9:12])
def test_attention_fast(case):
    ctx = E.Context(0)
    ctx.set_precision(True)
    c = Case(ctx, np.float32, **case)
    c.run()
    c.check(fast=True)
    ctx.close()


@pytest.mark.parametrize("n,q,kv_len", [(5, 1, [4000, 0, 1, 700, 3999]), (64, 1, list(range(1, 641, 10))), (65, 1, list(range(0, 650, 10))),
                                        (3, 3, [2, 1500, 64]), (2, 1, [0, 0]), (33, 2, [2000] + 32 * [5])])
@pytest.mark.parametrize("window,sinks", [(0, 0), (600, 70)])
def test_lengths_far_apart(ctx, n, q, kv_len, window, sinks):
    """Single tokens of items whose caches are empty, short and long: shares of very different numbers."""
    c = Case(ctx, np.float16, n=n, q=q, kv=4096 if n < 64 else 1024, hq=2, hk=1, d=40, block=64, kv_len=kv_len, window=window, sinks=sinks)
    c.run()
    c.check()


@pytest.mark.parametrize("n,q,d", [(1, 1, 64), (2, 9, 80), (64, 70, 64), (32, 130, 128)])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_scores_beyond_any_exponent(ctx, dtype, n, q, d):
    """Scores of 10^7 and more: each row is the value of its largest key, where the next one is far behind."""
    h = 1 if n < 32 else 4 if n == 64 else 8
    c = Case(ctx, dtype, n=n, q=q, kv=200, hq=h, hk=h, d=d, block=64, causal=False)
    c.run(scale=1e6)
    got = c.out.numpy().astype(np.float64)
    checked = 0
    for i in range(n):
        k, v = (c.held.values(w, c.table, i, 200)[0] for w in (0, 1))
        for x in range(h):
            s = 1e6 * c.qh[i, :, x].astype(np.float64) @ k[:, x].T
            two = np.sort(s, 1)[:, -2:]
            far = two[:, 1] - two[:, 0] > 1e-5 * np.abs(s).max(1) + 100  # beyond the f32 sums' own error
            want = v[s.argmax(1), x]
            assert np.all(np.abs(got[i, far, x] - want[far]) <= 2.0 ** (-10 if dtype == np.float16 else -20) * np.abs(want[far]) + 1e-7)
            checked += far.sum()
    assert checked >= 0.9 * n * q * h


@pytest.mark.parametrize("q,cap", [(1, 512), (150, 512), (150, 4200)])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_scores_and_values_of_very_different_size(ctx, dtype, q, cap):
    """Values of blocks 2^20 apart, keys that make the softmax nearly one token, queries with a few large channels."""
    r = np.random.default_rng(5)
    c = Case(ctx, dtype, n=1, q=q, kv=cap, hq=2, hk=2, d=64, block=16, kv_len=[512])
    size = np.exp2(np.where(np.arange(32) % 5 == 1, -14, 0) + np.where(np.arange(32) % 7 == 3, 6, 0))
    kv = [np.repeat(r.choice([0.25, 30.0], 32), 16)[None, :, None, None] * r.standard_normal((1, 512, 2, 64)),
          np.repeat(size, 16)[None, :, None, None] * r.standard_normal((1, 512, 2, 64))]
    kv = [x.astype(dtype) for x in kv]
    kv[1][:, 64:80] = 0  # a block of zeros
    cache_write(c.cache, c.dtable, heads(ctx, kv[0]), heads(ctx, kv[1]))
    c.held.write(c.table, kv, [0], [512])
    c.run()
    c.check()


@pytest.mark.parametrize("n,q,cap,hk", [(3, 1, 512, 2), (2, 5, 300, 2), (1, 150, 512, 2), (1, 150, 4200, 2), (64, 70, 200, 4), (4, 300, 300, 2)])
@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("window", [0, 8])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_rows_that_see_only_small_values(ctx, dtype, window, block, n, q, cap, hk):
    """Neighbouring blocks of values 2^21 apart, tokens that are alike: rows that see only small ones keep their bits.

    The sums' exponent is at most 2^10 above that of any value that a row sees, if it sees those of one block;
    the larger ones of others only make the bound's terms larger."""
    r = np.random.default_rng(cap + q)
    blocks = -(-cap // block)
    kv_len = [min(300, cap) - (i * 37) % 150 for i in range(n)]
    q_len = [min(q, x) for x in kv_len]
    c = Case(ctx, dtype, n=n, q=q, kv=cap, hq=2 * hk, hk=hk, d=64, block=block, q_len=q_len, kv_len=kv_len, window=window, std=0.25)
    size = np.repeat(np.exp2(r.choice([9, -2, -12, -12], blocks)), block)[None, :cap, None, None]
    kv = [0.25 * r.standard_normal((n, cap, hk, 64)), size * r.standard_normal((n, cap, hk, 64))]
    kv = [x.astype(dtype) for x in kv]
    c.held.write(c.table, kv, np.zeros(n, int), kv_len)
    cache_write(c.cache, c.dtable, heads(ctx, kv[0]), heads(ctx, kv[1]), length=lens(ctx, kv_len))
    c.run()
    want, tol = attention64(c.qh, c.held, c.table, 0.125, True, window, 0, q_len, kv_len, below=10)
    there = ~np.isnan(want)
    off = np.abs(c.out.numpy().astype(np.float64) - want)[there]
    assert np.all(off <= tol[there]), (off / tol[there]).max()


def test_probabilities_in_two_parts(ctx):
    """Few keys of nearly equal weight: no term of the bound hides a probability whose parts do not belong together."""
    c = Case(ctx, F32, n=2, q=256, kv=64, hq=8, hk=4, d=32, block=16, causal=False)
    c.run(scale=2.0 ** -6)
    c.check(scale=2.0 ** -6)


@pytest.mark.parametrize("n,q,hq,hk,d,kv,window", [(2, 1, 8, 4, 64, 16, 0), (1, 5, 8, 2, 128, 300, 26), (3, 1, 4, 4, 80, 2000, 0), (1, 20, 2, 1, 200, 900, 40)])
def test_f16_rows_alone_round_once(ctx, n, q, hq, hk, d, kv, window):
    """f16 calls whose rows share no tokens hold probabilities in two parts: off as f32 ones, and half a step of the output."""
    c = Case(ctx, np.float16, n=n, q=q, kv=kv, hq=hq, hk=hk, d=d, block=32, window=window)
    c.run()
    want, tol = attention64(c.qh.astype(F32), c.held, c.table, 1 / np.sqrt(d), True, window, 0, c.q_len, c.kv_len)
    off = np.abs(c.out.numpy().astype(np.float64) - want)
    tol = tol + 2.0 ** -11 * (np.abs(want) + tol) + 2.0 ** -25
    assert np.all(off <= tol), (off / tol).max()


@pytest.mark.parametrize("n,block", [(1, 16), (2, 32)])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_blocks_of_small_values_in_splits(ctx, dtype, n, block):
    """Single tokens over a long cache whose shares and blocks of values lie far apart, with a page missing between them."""
    kv_len = [3900, 2117][:n]
    c = Case(ctx, dtype, n=n, q=1, kv=4000, hq=4, hk=2, d=80, block=block, kv_len=kv_len, absent=[(0, 61), (0, 62)])
    r = np.random.default_rng(block)
    size = np.repeat(np.exp2(r.choice([9, -2, -12], c.blocks)), block)[None, :4000, None, None]
    kv = [(0.25 * r.standard_normal((n, 4000, 2, 80))).astype(dtype), (size * r.standard_normal((n, 4000, 2, 80))).astype(dtype)]
    c.held.write(c.table, kv, np.zeros(n, int), kv_len)
    cache_write(c.cache, c.dtable, heads(ctx, kv[0]), heads(ctx, kv[1]), length=lens(ctx, kv_len))
    c.run()
    c.check()


@pytest.mark.parametrize("q,cap", [(8, 200), (80, 4200)])
def test_queries_of_any_size(ctx, q, cap):
    """f32 queries far outside f16 in both directions, and rows that are not finite beside others."""
    c = Case(ctx, F32, n=1, q=q, kv=cap, hq=1, hk=1, d=64, block=64, causal=False, kv_len=[200])
    for i, e in enumerate([-126, -60, -20, 0, 10]):
        c.qh[0, i] = (c.qh[0, i].astype(np.float64) * 2.0 ** e).astype(F32)
    c.qh[0, 5] = np.nan
    c.qh[0, 6, 0, 3] = np.inf
    c.qh[0, 7] = 0
    c.q.buf.upload(c.qh)
    c.run()
    got = c.out.numpy()
    assert np.isnan(got[0, 5:7]).all()
    rows = [i for i in range(q) if i not in (5, 6)]
    want, tol = attention64(c.qh[:, rows], c.held, c.table, 0.125, False, 0, 0, [len(rows)], [200])
    assert np.all(np.abs(got[0, rows] - want[0]) <= tol[0])


@pytest.mark.parametrize("q,kv", [(1, 3000), (200, 1000), (100, 4300)])
def test_captured_and_replayed(ctx, q, kv):
    """Two graphs with scratch of their own beside eager calls; a write and the attention over it in each."""
    cases = [Case(ctx, np.float16, n=2, q=q, kv=kv, hq=8, hk=2, d=64, block=32, seed=s) for s in (1, 2)]
    new = [[heads(ctx, np.random.default_rng(s + w).standard_normal((2, 1, 2, 64)).astype(np.float16)) for w in (0, 9)] for s in (1, 2)]
    at = lens(ctx, [kv - 1, kv - 1])

    def step(c, x, scratch=None):
        cache_write(c.cache, c.dtable, *x, first=at)
        c.run(scratch)

    wants = []
    for c, x in zip(cases, new):
        step(c, x)
        wants.append(c.out.numpy())
    need = [cache_attention_scratch(c.q, c.cache, c.dtable) for c in cases]
    if need[0]:
        with pytest.raises(MoebiusError, match="scratch of its own"):
            capture(ctx, lambda: step(cases[0], new[0]))
        with pytest.raises(MoebiusError, match="smaller"):
            cases[0].run(E.DeviceArray(ctx, (need[0] - 16,), np.uint8))
    scratch = [E.DeviceArray(ctx, (max(b, 16),), np.uint8) for b in need]
    graphs = [capture(ctx, lambda c=c, x=x, s=s: step(c, x, s)) for c, x, s in zip(cases, new, scratch)]
    for turn in range(4):
        for c in cases:
            c.out.buf.upload(np.zeros(c.out.buf.shape, np.float16))
        for launch, _ in graphs:
            launch()
        ctx.synchronize()
        for c, want in zip(cases, wants):
            assert np.array_equal(c.out.numpy(), want)
        step(cases[turn % 2], new[turn % 2])
        assert np.array_equal(cases[turn % 2].out.numpy(), wants[turn % 2])
    for _, destroy in graphs:
        destroy()
