"""Block means, the selection of key blocks and the attention over them, against
the definitions in f64.

Attention tolerances, for a row with scores s_j and values v_j (m = max |v| over
the keys it sees; all bounds are worst cases of the roundings):
  - a score is off by (d + 2) u A with u = 2^-24 and A = max_j scale sum |q_i k_ij|
    (f32 sums of exact or once rounded products), the exponent's argument by 2^-23 B
    more with B = max |s_j| log2 e, the hardware's exponential by 2^-22, the running
    rescales and the two sums by (2 tiles + keys) u, all twice (numerator and denominator);
  - f32 products formed from operands in two f16 parts leave 3 u of each product out (two
    roundings of 2^-24 and the product of the small parts), of a score and of p v;
  - f16 products round each probability by 2^-11;
  - FAST contexts round q, k and v too: 2 x 2^-11 A per score, twice, and 2^-11 for v;
  - f16 outputs add half a step.
"""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from moebius_cpu_amd import _lib
from moebius_cpu_amd import engine as E
from moebius_cpu_amd._lib import MoebiusError
from moebius_cpu_amd.attention import (Heads, RopeAxes, block_attention, block_attention_scratch, block_means,
                                       block_select, qk_norm_rope)
from tests.graph_capture import capture

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    return E.Context(0)


def dev(ctx, a):
    return E.DeviceArray.from_numpy(ctx, np.ascontiguousarray(a))


def lens(ctx, a):
    return None if a is None else dev(ctx, np.asarray(a, np.int32))


def heads(ctx, x, pad=0, offset=0):
    """x [n][tokens][heads][d] with rows `pad` elements longer, NaN between them."""
    n, t, h, d = x.shape
    if not pad and not offset:
        return Heads(dev(ctx, x), n, t, h, d)
    flat = np.full(offset + n * t * (h * d + pad), np.nan, x.dtype)
    rows = np.lib.stride_tricks.as_strided(flat[offset:], (n * t, h * d),
                                           ((h * d + pad) * x.itemsize, x.itemsize))
    rows[:] = x.reshape(n * t, h * d)
    return Heads(dev(ctx, flat), n, t, h, d, ld=h * d + pad, offset=offset)


# ---------------------------------------------------------------- means

@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("n,tokens,h,d,block,pad,offset", [
    (1, 1, 1, 1, 16, 0, 0), (2, 130, 3, 40, 64, 0, 0), (1, 1000, 8, 128, 128, 128, 8), (3, 50, 2, 33, 16, 1, 1),
    (1, 257, 16, 64, 32, 0, 0), (2, 7, 2, 80, 1, 0, 0), (1, 2050, 1, 72, 1024, 0, 0)])
def test_means(ctx, dtype, n, tokens, h, d, block, pad, offset):
    """Off by one f32 rounding of the f64 mean (and f64's own, 10^-13 of the largest term)."""
    r = np.random.default_rng(tokens)
    x = r.standard_normal((n, tokens, h, d)).astype(dtype)
    length = r.integers(0, tokens + 1, n)
    length[0] = tokens
    for i in range(n):
        x[i, length[i]:] = np.nan  # behind the length nothing counts
    nb = -(-tokens // block)
    means = dev(ctx, np.full((n, nb, h, d), 7, np.float32))
    block_means(heads(ctx, x, pad, offset), block, means, length=lens(ctx, length))
    got = means.numpy().astype(np.float64)
    for i in range(n):
        for b in range(nb):
            part = x[i, b * block:min((b + 1) * block, length[i])].astype(np.float64)
            if len(part):
                want = part.mean(0)
                assert np.all(np.abs(got[i, b] - want) <= U * np.abs(want) + 1e-13 * np.abs(part).max())
            else:
                assert np.all(got[i, b] == 7)  # left as it was


def test_means_of_new_tokens_only(ctx):
    """first leaves the blocks below it alone; the result is that of the whole pass."""
    x = np.random.default_rng(0).standard_normal((3, 200, 2, 40)).astype(np.float32)
    h = heads(ctx, x)
    whole, step = dev(ctx, np.zeros((3, 7, 2, 40), np.float32)), dev(ctx, np.zeros((3, 7, 2, 40), np.float32))
    old, new = np.array([0, 64, 95]), np.array([40, 65, 200])
    block_means(h, 32, whole, length=lens(ctx, new))
    block_means(h, 32, step, length=lens(ctx, old))
    marked = step.numpy()
    marked[1, :2] += 1  # blocks that end at or below `first`
    marked[2, :2] += 1
    step.upload(marked)
    block_means(h, 32, step, length=lens(ctx, new), first=lens(ctx, old))
    want = whole.numpy()
    want[1, :2] += 1
    want[2, :2] += 1
    assert np.array_equal(step.numpy(), want)


def test_lengths_out_of_range_are_clamped(ctx):
    x = np.random.default_rng(0).standard_normal((2, 40, 1, 8)).astype(np.float32)
    m = dev(ctx, np.full((2, 3, 1, 8), 5, np.float32))
    block_means(heads(ctx, x), 16, m, length=lens(ctx, [-3, 2**31 - 1]))
    assert np.all(m.numpy()[0] == 5)
    assert np.abs(m.numpy()[1, 2] - x[1, 32:].mean(0)).max() < 1e-6


# ---------------------------------------------------------------- selection

def selected(q, means, qb, kb, top, causal, q_len, kv_len):
    """The definition: f64 scores of the f32 means, a stable order by (forced, score, lower index)."""
    n, qt, hq, d = q.shape
    hk, g = means.shape[2], hq // means.shape[2]
    nq = -(-qt // qb)
    out = np.full((n, nq, hk, top), -1, np.int32)
    for i in range(n):
        ql = qt if q_len is None else q_len[i]
        kl = kv_len[i]
        for b in range(nq):
            rows = q[i, b * qb:min((b + 1) * qb, ql)].astype(np.float64)
            if not len(rows):
                continue
            last = kl - 1
            if causal:
                last = min(last, kl - ql + min((b + 1) * qb, ql) - 1)
            seen = last // kb + 1 if last >= 0 else 0
            lo = max(kl - ql + b * qb, 0) // kb if causal else seen
            for h in range(hk):
                mean = rows[:, h * g:(h + 1) * g].mean((0, 1)).astype(np.float32).astype(np.float64)
                s = means[i, :seen, h].astype(np.float64) @ mean
                s = np.where(np.isnan(s), -np.inf, s)
                keys = sorted(range(seen), key=lambda j: (j < lo, -s[j], j))[:top]
                out[i, b, h, :len(keys)] = sorted(keys)
    return out


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("n,qt,kt,hq,hk,d,qb,kb,top,causal", [
    (1, 1, 40, 1, 1, 8, 1, 16, 2, False), (3, 1, 3000, 8, 2, 128, 1, 16, 20, True), (2, 200, 200, 4, 4, 40, 64, 16, 5, False),
    (2, 130, 700, 6, 2, 72, 16, 32, 6, True), (1, 1024, 1024, 2, 1, 80, 128, 64, 4, True), (1, 37, 555, 3, 3, 33, 5, 128, 2, True),
    (2, 300, 90, 2, 2, 64, 32, 16, 7, True), (1, 700, 9000, 1, 1, 256, 1, 32, 64, False), (1, 64, 64, 2, 2, 96, 64, 128, 3, False),
    (1, 3, 60000, 2, 1, 16, 1, 16, 900, False)])
def test_select(ctx, dtype, n, qt, kt, hq, hk, d, qb, kb, top, causal):
    r = np.random.default_rng(kt)
    q = r.standard_normal((n, qt, hq, d)).astype(dtype)
    nk = -(-kt // kb)
    means = r.standard_normal((n, nk, hk, d)).astype(np.float32)
    kv_len = r.integers(0, kt + 1, n)
    q_len = r.integers(0, qt + 1, n)
    kv_len[0], q_len[0] = kt, qt
    blocks = dev(ctx, np.full((n, -(-qt // qb), hk, top), 77, np.int32))
    block_select(heads(ctx, q, pad=8, offset=16), dev(ctx, means), kt, blocks, q_block=qb, kv_block=kb, causal=causal,
                 q_len=lens(ctx, q_len), kv_len=lens(ctx, kv_len))
    assert np.array_equal(blocks.numpy(), selected(q, means, qb, kb, top, causal, q_len, kv_len))


def test_select_ties_nan_and_infinity(ctx):
    """Equal scores go to the lower index, zeros of either sign are equal, NaN is lowest, infinity highest."""
    means = np.zeros((1, 200, 1, 8), np.float32)
    means[0, 3::7, 0, 0] = 1
    means[0, 5, 0, 0] = np.nan
    means[0, 6, 0, 0] = -np.inf
    means[0, 190, 0, 0] = np.inf
    means[0, 8, 0, 0] = -0.0
    q = np.zeros((1, 1, 1, 8), np.float32)
    q[..., 0] = 1
    for top in (1, 5, 29, 30, 31, 40, 198, 199, 200):
        blocks = dev(ctx, np.zeros((1, 1, 1, top), np.int32))
        block_select(heads(ctx, q), dev(ctx, means), 3200, blocks, q_block=1, kv_block=16)
        s = means[0, :, 0, 0] + 0.0
        order = sorted(range(200), key=lambda j: (np.isnan(s[j]), -s[j] if not np.isnan(s[j]) else 0, j))[:top]
        assert blocks.numpy().ravel().tolist() == sorted(order), top


def test_select_reads_nothing_behind_the_lengths(ctx):
    """Means of blocks that there are not, and queries behind q_len, may hold anything."""
    r = np.random.default_rng(4)
    q, means = r.standard_normal((1, 64, 2, 40)).astype(np.float32), r.standard_normal((1, 32, 2, 40)).astype(np.float32)
    got = []
    for fill in (0.0, np.nan):
        q[0, 40:], means[0, 10:] = fill, fill
        blocks = dev(ctx, np.zeros((1, 4, 2, 6), np.int32))
        block_select(heads(ctx, q), dev(ctx, means), 512, blocks, q_block=16, kv_block=16, q_len=lens(ctx, [40]),
                     kv_len=lens(ctx, [150]))
        got.append(blocks.numpy())
    assert np.array_equal(got[0], got[1])
    assert (got[0][0, 3] == -1).all() and got[0].max() < 10


# ---------------------------------------------------------------- attention

def reference(q, k, v, blocks, scale, qb, kb, causal, q_len, kv_len):
    """The definition in f64, and what the tolerance of a row goes by: (out, seen keys, A, B, m), rows not there NaN."""
    n, qt, hq, d = q.shape
    hk, g = k.shape[2], hq // k.shape[2]
    out = np.full((n, qt, hq, d), np.nan)
    tol = np.zeros((n, qt, hq, 4))
    for i in range(n):
        ql = qt if q_len is None else min(max(q_len[i], 0), qt)
        kl = k.shape[1] if kv_len is None else min(max(kv_len[i], 0), k.shape[1])
        for t in range(ql):
            for h in range(hq):
                picked = sorted({int(b) for b in blocks[i, t // qb, h // g] if 0 <= int(b) * kb < kl})
                keys = [j for b in picked for j in range(b * kb, min((b + 1) * kb, kl)) if not causal or j <= t + kl - ql]
                if not keys:
                    out[i, t, h] = 0
                    continue
                kk, vv = k[i, keys, h // g].astype(np.float64), v[i, keys, h // g].astype(np.float64)
                qq = q[i, t, h].astype(np.float64)
                s = kk @ qq * scale
                p = np.exp(s - s.max())
                out[i, t, h] = p @ vv / p.sum()
                tol[i, t, h] = len(keys), (np.abs(kk) @ np.abs(qq)).max() * scale, np.abs(s).max() * 1.4427, np.abs(vv).max()
    return out, tol


def tolerance(out, tol, d, dtype, fast):
    keys, A, B, m = (tol[..., i] for i in range(4))
    e = 2 * ((d + 5) * U * A + 2 * U * B + 4 * U) + (keys + keys / 8 + 3) * U
    if dtype == np.float16 or fast:
        e = e + 2.0 ** -11
    if fast:
        e = e + 2 * 2 * 2.0 ** -11 * A + 2.0 ** -11
    t = (e * m)[..., None] + 1e-30
    return t + (np.abs(out) * 2.0 ** -11 + 2.0 ** -25 if dtype == np.float16 else np.abs(out) * U)


def lists(r, n, nq, hk, top, nk):
    """Distinct blocks in any order, some places empty."""
    out = np.full((n, nq, hk, top), -1, np.int32)
    for i in np.ndindex(n, nq, hk):
        pick = r.permutation(nk)[:top]
        out[i][:len(pick)] = np.sort(pick) if r.random() < 0.5 else pick
        out[i][r.random(top) < 0.1] = -1
    return out


def run(ctx, q, k, v, blocks, qb, kb, causal=False, q_len=None, kv_len=None, scale=None, pad=0, offset=0, fill=np.nan):
    """The call on rows `pad` apart; rows that it leaves alone come back as `fill`."""
    out = heads(ctx, np.full(q.shape, fill, q.dtype), pad, offset)
    block_attention(heads(ctx, q, pad, offset), heads(ctx, k, pad, offset), heads(ctx, v, pad, offset), dev(ctx, blocks),
                    out, scale=scale, q_block=qb, kv_block=kb, causal=causal, q_len=lens(ctx, q_len), kv_len=lens(ctx, kv_len))
    return out.numpy()


CASES = [  # n, q, kv, hq, hk, d, qb, kb, top, causal
    (1, 1, 1, 1, 1, 8, 1, 16, 1, False),        # one token, one key
    (2, 1, 300, 4, 1, 64, 1, 16, 12, True),     # single tokens, lists split over workgroups
    (3, 1, 1000, 8, 2, 128, 1, 64, 9, True),
    (1, 3, 2100, 2, 2, 40, 1, 128, 10, False),
    (2, 70, 70, 2, 2, 40, 32, 16, 4, False),    # one wave of rows
    (1, 128, 200, 1, 1, 80, 64, 32, 5, False),  # two
    (1, 150, 333, 2, 1, 72, 64, 64, 4, True),   # four, ragged
    (2, 100, 250, 4, 2, 96, 16, 16, 8, True),
    (1, 260, 260, 1, 1, 128, 128, 64, 3, False),
    (1, 140, 140, 1, 1, 160, 100, 128, 2, True),  # blocks of queries that are no power of two
    (1, 40, 200, 3, 1, 256, 16, 32, 4, True),
    (1, 130, 300, 1, 1, 200, 128, 32, 6, False),
    (1, 20, 90, 2, 1, 33, 8, 16, 4, True),      # no wide loads
    (1, 70, 90, 1, 1, 7, 70, 64, 2, False),
    (1, 10, 100, 2, 2, 130, 4, 16, 5, True),
    (1, 9, 50, 36, 1, 32, 2, 16, 3, False),     # 72 rows of one key head
    (1, 5, 64, 70, 2, 16, 5, 16, 3, True),
    # keys read by many rows: f32 operands in two parts
    (2, 256, 256, 2, 2, 80, 64, 32, 8, False),
    (1, 300, 400, 2, 1, 40, 64, 16, 20, True),
    (1, 128, 500, 4, 2, 128, 64, 64, 8, True),
    (1, 200, 300, 1, 1, 160, 100, 32, 9, False),
    (1, 130, 140, 1, 1, 33, 70, 16, 8, True),
    (2, 256, 300, 1, 1, 64, 128, 128, 3, True),
    (1, 140, 170, 1, 1, 134, 70, 16, 11, False),
    # the same with a wave of rows and one without, and lists of few keys split over workgroups
    (2, 300, 300, 2, 2, 80, 16, 32, 8, False), (1, 640, 320, 1, 1, 160, 32, 64, 5, True),
    (1, 200, 96, 2, 2, 128, 8, 16, 6, True), (1, 330, 120, 1, 1, 33, 16, 16, 8, True),
    (1, 3, 290, 2, 1, 96, 128, 32, 10, True), (2, 1, 310, 4, 4, 160, 1, 16, 20, True),
    (1, 70, 400, 1, 1, 160, 64, 64, 6, False),
]


@pytest.mark.parametrize("kind", ["f16", "f32", "fast"])
@pytest.mark.parametrize("case", CASES)
def test_attention(ctx, case, kind):
    n, qt, kt, hq, hk, d, qb, kb, top, causal = case
    dtype = np.float16 if kind == "f16" else np.float32
    r = np.random.default_rng(qt * 7 + kt + d)
    q, k, v = (r.standard_normal(s).astype(dtype) for s in ((n, qt, hq, d), (n, kt, hk, d), (n, kt, hk, d)))
    kv_len, q_len = r.integers(kt // 2, kt + 1, n), r.integers((qt + 1) // 2, qt + 1, n)
    kv_len[0], q_len[0] = kt, qt
    for i in range(n):  # behind the lengths lies anything
        q[i, q_len[i]:], k[i, kv_len[i]:], v[i, kv_len[i]:] = np.nan, np.nan, np.inf
    blocks = lists(r, n, -(-qt // qb), hk, top, -(-kt // kb))
    scale = 1 / np.sqrt(d)
    pad, offset = (8, 16) if d % 8 == 0 else (1, 3)
    ctx.set_precision(kind == "fast")
    try:
        got = run(ctx, q, k, v, blocks, qb, kb, causal, q_len, kv_len, None, pad, offset, fill=3).astype(np.float64)
    finally:
        ctx.set_precision(False)
    want, tol = reference(q, k, v, blocks, scale, qb, kb, causal, q_len, kv_len)
    there = ~np.isnan(want)
    assert np.all(got[~there] == 3)  # rows at or above q_len: left as they were
    err, bound = np.abs(got - want)[there], tolerance(want, tol, d, dtype, kind == "fast")[there]
    assert np.all(err <= bound), (err / bound).max()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_rows_that_see_nothing_are_zero(ctx, dtype):
    """No key at all, empty lists, lists of blocks that are not there, causal rows before the first key."""
    r = np.random.default_rng(0)
    q, k, v = (r.standard_normal((4, t, 2, 64)).astype(dtype) for t in (40, 96, 96))
    blocks = lists(r, 4, 3, 2, 6, 6)
    blocks[1] = -1
    blocks[2] = np.array([6, 7, -5, 2**31 - 1, -2**31, 1000])
    got = run(ctx, q, k, v, blocks, 16, 16, True, [40, 40, 40, 40], [0, 96, 96, 10])
    assert not got[:3].any()
    assert not got[3, :30].any()  # query i sees keys up to i - 30
    want, tol = reference(q, k, v, blocks, 1 / 8, 16, 16, True, [40] * 4, [0, 96, 96, 10])
    assert np.all(np.abs(got[3].astype(np.float64) - want[3]) <= tolerance(want, tol, 64, dtype, False)[3])
    # no keys in the tensor either
    none = np.zeros((1, 0, 2, 64), dtype)
    got = run(ctx, q[:1], none, none, np.zeros((1, 3, 2, 1), np.int32), 16, 16)
    assert not got.any()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("q_block", [1, 16])
def test_lists_are_sets(ctx, dtype, q_block):
    """An index listed twice counts once, in any order; ascending lists and their shuffles of one tile agree in bits."""
    r = np.random.default_rng(1)
    q, k, v = (r.standard_normal((1, t, 1, 40)).astype(dtype) for t in (16, 640, 640))
    nq = 16 // q_block
    base = np.tile(np.array([3, 7, 20, 39], np.int32), (1, nq, 1, 1))
    twice = np.tile(np.array([3, 7, 20, 39, -1, 7, 3, 39, 20, 3, 50, -7], np.int32), (1, nq, 1, 1))
    a, b = run(ctx, q, k, v, base, q_block, 16), run(ctx, q, k, v, twice, q_block, 16)
    want, tol = reference(q, k, v, base, 1 / np.sqrt(40), q_block, 16, False, None, None)
    bound = tolerance(want, tol, 40, dtype, False)
    assert np.all(np.abs(a - want) <= bound) and np.all(np.abs(b - want) <= bound)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("q_block", [1, 16, 64, 128])
def test_what_a_row_does_not_see_does_not_reach_it(ctx, dtype, q_block):
    """Causal rows whose tile holds keys and values of later tokens that are NaN or infinite."""
    r = np.random.default_rng(2)
    q, k, v = (r.standard_normal((1, 128, 2, 48)).astype(dtype) for _ in range(3))
    blocks = np.tile(np.arange(4, dtype=np.int32), (1, -(-128 // q_block), 2, 1))
    clean, tol = reference(q, k, v, blocks, 1 / np.sqrt(48), q_block, 32, True, None, None)
    v[0, 70, 0, 5], v[0, 100, :, :], k[0, 90] = np.inf, np.nan, np.nan
    got = run(ctx, q, k, v, blocks, q_block, 32, True).astype(np.float64)
    bound = tolerance(clean, tol, 48, dtype, False)
    ok = np.abs(got - clean) <= bound
    assert ok[0, :70].all()
    assert ok[0, 70:90, 0, :5].all() and ok[0, 70:90, 0, 6:].all() and np.isposinf(got[0, 70:90, 0, 5]).all()
    assert ok[0, 70:90, 1].all()
    assert np.isnan(got[0, 90:]).all()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_blocks_not_listed_are_not_read(ctx, dtype):
    r = np.random.default_rng(3)
    q, k, v = (r.standard_normal((1, t, 1, 64)).astype(dtype) for t in (64, 512, 512))
    blocks = np.array([1, 4, 6], np.int32).reshape(1, 1, 1, 3)
    a = run(ctx, q, k, v, blocks, 64, 64)
    mask = np.ones(512, bool)
    for b in (1, 4, 6):
        mask[b * 64:(b + 1) * 64] = False
    k[0, mask], v[0, mask] = np.nan, np.nan
    assert np.array_equal(run(ctx, q, k, v, blocks, 64, 64), a)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_large_and_infinite_scores(ctx, dtype):
    """Scores of thousands keep the softmax finite; equal scores give the mean; a masked lowest value gives nothing."""
    q, k, v = np.zeros((1, 4, 1, 8), dtype), np.zeros((1, 64, 1, 8), dtype), np.zeros((1, 64, 1, 8), dtype)
    v[0, :, 0, 0] = np.arange(64)
    q[0, 1, 0, 0], k[0, 17, 0, 0] = 200, 200     # one score of 40 000 above the others
    q[0, 2, 0, 1], k[0, 33, 0, 1] = 200, -200    # one far below
    q[0, 3, 0, 2], k[0, 50:, 0, 2] = -1, np.finfo(dtype).max if dtype == np.float16 else 1e30
    wants = (31.5, 17.0, (2016 - 33) / 63, 24.5)
    listed = np.arange(4, dtype=np.int32).reshape(1, 1, 1, 4)
    for rows in (1, 16):  # one wave of rows, and keys read by many
        qq, li = np.tile(q, (1, rows, 1, 1)), np.tile(listed, (1, max(1, rows // 16), 1, 1))
        got = run(ctx, qq, k, v, li, 4 * rows, 16, scale=1.0)[0, :, 0, 0]
        for g, want in zip(got, wants * rows):
            assert abs(float(g) - want) <= want * (2.0 ** -10 if dtype == np.float16 else 1e-6)
    # scores of 10^9 and more, of which those of the largest key are the largest (f16: 200 x 200 x 10^5)
    big = 1e5 if dtype == np.float16 else 1e20
    for rows in (1, 16):
        qq = np.tile(q[:, 1:2], (1, 4 * rows, 1, 1))
        got = run(ctx, qq, k, v, listed, 4 * rows, 16, scale=big)[0, :, 0, 0]
        assert np.array_equal(got, np.full(4 * rows, 17, dtype))


@pytest.mark.parametrize("d", [64, 80])
def test_f32_ranges(ctx, d):
    """Blocks of keys and values, and rows of queries, of sizes far from each other and from f16's range:
    the errors stay relative to the products a row forms and to the largest value it sees."""
    r = np.random.default_rng(d)
    q, k, v = (r.standard_normal((1, t, 1, d)).astype(np.float32) for t in (192, 192, 192))
    for b, f in enumerate((1e-30, 1e-6, 1.0, 1e4, 3e8, 1e-42)):
        k[0, b * 32:(b + 1) * 32] *= np.float32(f)
        v[0, b * 32:(b + 1) * 32] *= np.float32((1e30, 1e-20, 1e10, 1.0, 0.0, 1e20)[b])
        q[0, b * 32:(b + 1) * 32] *= np.float32((1.0, 1e-9, 1e-4, 1e3, 1e20, 1e-38)[b])
    v[0, :, 0, :8] *= np.float32(2.0 ** -20)
    for blocks in ([0, 1, 2], [1, 2, 3], [3, 4], [5], [1], [2, 5], [4], [1, 5]):
        li = np.tile(np.array(blocks + [-1] * (6 - len(blocks)), np.int32), (1, 2, 1, 1))
        got = run(ctx, q, k, v, li, 96, 32, scale=0.125).astype(np.float64)
        want, tol = reference(q, k, v, li, 0.125, 96, 32, False, None, None)
        ok = tol[..., 2] < 1e4  # beyond it an exponent's rounding is larger than a score's part
        bound = tolerance(want, tol, d, np.float32, False)
        assert ok.any() and np.all((np.abs(got - want) <= bound)[ok]), blocks
        assert np.isfinite(got).all()


def test_row_results_do_not_depend_on_the_batch(ctx):
    """The same item alone and among others, and the same call twice: the same bits."""
    r = np.random.default_rng(6)
    q, k, v = (r.standard_normal((3, t, 2, 64)).astype(np.float16) for t in (64, 320, 320))
    blocks = lists(r, 3, 1, 2, 4, 5)
    a = run(ctx, q, k, v, blocks, 64, 64)
    assert np.array_equal(a, run(ctx, q, k, v, blocks, 64, 64))


def test_scratch_is_checked(ctx):
    r = np.random.default_rng(7)
    q, k, v = (heads(ctx, r.standard_normal((1, t, 2, 64)).astype(np.float16)) for t in (1, 2048, 2048))
    out, blocks = Heads(E.DeviceArray(ctx, (1, 1, 2, 64), "f2"), 1, 1, 2, 64), dev(ctx, np.arange(32, dtype=np.int32).reshape(1, 1, 2, 16))
    size = block_attention_scratch(q, k, blocks, 1, 64)
    assert size > 0
    with pytest.raises(MoebiusError, match="smaller"):
        block_attention(q, k, v, blocks, out, q_block=1, scratch=E.DeviceArray(ctx, (size - 1,), np.uint8))
    block_attention(q, k, v, blocks, out, q_block=1, scratch=E.DeviceArray(ctx, (size,), np.uint8))
    a = out.numpy()
    block_attention(q, k, v, blocks, out, q_block=1)
    assert np.array_equal(out.numpy(), a)
    with pytest.raises(MoebiusError, match="captured call needs scratch"):
        capture(ctx, lambda: block_attention(q, k, v, blocks, out, q_block=1))
    ctx.synchronize()
    few = dev(ctx, np.arange(4, dtype=np.int32).reshape(1, 1, 2, 2))  # lists that are not split need none
    assert block_attention_scratch(q, k, few, 1, 64) == 0
    launch, destroy = capture(ctx, lambda: block_attention(q, k, v, few, out, q_block=1))
    block_attention(q, k, v, few, out, q_block=1)
    a = out.numpy()
    out.buf.upload(np.zeros_like(a))
    launch()
    ctx.synchronize()
    assert np.array_equal(out.numpy(), a)
    destroy()


def test_a_layer_step_captured_and_replayed(ctx):
    """Norm and rotation, means, selection and attention of single tokens as one run, eager and as
    two graphs with scratch of their own, replayed in turn among eager calls; against the definitions."""
    r = np.random.default_rng(8)
    n, kt, hq, hk, d, kb, top = 2, 1024, 4, 2, 64, 32, 8
    rope = RopeAxes(ctx, (16, 24, 24))
    g = dev(ctx, (1 + 0.1 * r.standard_normal(d)).astype(np.float32))
    cache_v = heads(ctx, r.standard_normal((n, kt, hk, d)).astype(np.float16))
    ql, kl = lens(ctx, [1, 1]), lens(ctx, [1000, 513])

    def state(seed):
        r = np.random.default_rng(seed)
        x = r.standard_normal((n, hq + hk, d)).astype(np.float16)
        buf = dev(ctx, x)
        st = dict(q=Heads(buf, n, 1, hq, d, ld=(hq + hk) * d), kn=Heads(buf, n, 1, hk, d, ld=(hq + hk) * d, offset=hq * d),
                  pos=dev(ctx, r.integers(0, 1000, (n, 3)).astype(np.int32)), k=heads(ctx, r.standard_normal((n, kt, hk, d)).astype(np.float16)),
                  qo=Heads(E.DeviceArray(ctx, (n, 1, hq, d), "f2"), n, 1, hq, d), ko=Heads(E.DeviceArray(ctx, (n, 1, hk, d), "f2"), n, 1, hk, d),
                  means=dev(ctx, np.zeros((n, kt // kb, hk, d), np.float32)), blocks=dev(ctx, np.zeros((n, 1, hk, top), np.int32)),
                  out=Heads(E.DeviceArray(ctx, (n, 1, hq, d), "f2"), n, 1, hq, d))
        st["scratch"] = E.DeviceArray(ctx, (block_attention_scratch(st["qo"], st["k"], st["blocks"], 1, kb),), np.uint8)
        return st

    def step(st, scratch):
        qk_norm_rope(st["q"], st["kn"], g, g, 1e-6, st["pos"], rope, st["qo"], st["ko"])
        block_means(st["k"], kb, st["means"], length=kl)
        block_select(st["qo"], st["means"], kt, st["blocks"], q_block=1, kv_block=kb, causal=True, q_len=ql, kv_len=kl)
        block_attention(st["qo"], st["k"], cache_v, st["blocks"], st["out"], q_block=1, kv_block=kb, causal=True, q_len=ql,
                        kv_len=kl, scratch=scratch)

    states = [state(1), state(2)]
    wants = []
    for st in states:
        step(st, None)
        q, k, blocks = st["qo"].numpy(), st["k"].numpy(), st["blocks"].numpy()
        assert np.array_equal(blocks, selected(q, st["means"].numpy(), 1, kb, top, True, [1, 1], [1000, 513]))
        want, tol = reference(q, k, cache_v.numpy(), blocks, 1 / 8, 1, kb, True, [1, 1], [1000, 513])
        got = st["out"].numpy()
        assert np.all(np.abs(got - want) <= tolerance(want, tol, d, np.float16, False))
        wants.append(got)
    graphs = [capture(ctx, lambda st=st: step(st, st["scratch"])) for st in states]
    for turn in range(4):
        for st in states:
            st["out"].buf.upload(np.zeros((n, 1, hq, d), np.float16))
        for launch, _ in graphs:
            launch()
        if turn % 2:
            block_attention(states[0]["qo"], states[0]["k"], cache_v, states[1]["blocks"], Heads(E.DeviceArray(ctx, (n, 1, hq, d), "f2"), n, 1, hq, d),
                            q_block=1, kv_block=kb)  # eager work between replays, in the context's own workspace
        ctx.synchronize()
        for st, want in zip(states, wants):
            assert np.array_equal(st["out"].numpy(), want)
    for _, destroy in graphs:
        destroy()


def test_cache_beyond_32_bit_offsets(ctx):
    """Blocks at the far end of a cache of more than 2^32 bytes and 2^31 elements."""
    kt, hk, d, kb = 1_100_000, 16, 128, 128
    k, v = (E.DeviceArray(ctx, (1, kt, hk, d), "f2") for _ in range(2))
    r = np.random.default_rng(9)
    small = r.standard_normal((2, 2 * kb, hk, d)).astype(np.float16)
    picked = np.array([3, kt // kb - 1], np.int32)
    for buf, src in ((k, small[0]), (v, small[1])):
        for i, b in enumerate(picked):
            part = np.ascontiguousarray(src[i * kb:(i + 1) * kb])
            _lib.check(_lib.lib().mh_memcpy_h2d(ctx.h, buf.ptr + int(b) * kb * hk * d * 2, part.ctypes.data, part.nbytes))
    q = r.standard_normal((1, 1, hk, d)).astype(np.float16)
    blocks = np.tile(picked, (1, 1, hk, 1))
    out = Heads(E.DeviceArray(ctx, q.shape, "f2"), 1, 1, hk, d)
    block_attention(heads(ctx, q), Heads(k, 1, kt, hk, d), Heads(v, 1, kt, hk, d), dev(ctx, blocks), out, q_block=1, kv_block=kb)
    want, tol = reference(q, small[:1], small[1:], np.tile(np.arange(2, dtype=np.int32), (1, 1, hk, 1)), d ** -0.5, 1, kb, False, None, None)
    assert np.all(np.abs(out.numpy() - want) <= tolerance(want, tol, d, np.float16, False))
    k.free(), v.free()


def test_python_refusals(ctx):
    z = lambda *s: Heads(E.DeviceArray(ctx, s, "f2"), *s)  # noqa: E731
    q, k, v, out = z(1, 4, 2, 8), z(1, 32, 1, 8), z(1, 32, 1, 8), z(1, 4, 2, 8)
    blocks = E.DeviceArray(ctx, (1, 1, 1, 2), "i4")
    with pytest.raises(MoebiusError, match="blocks are int32"):
        block_attention(q, k, v, E.DeviceArray(ctx, (1, 2, 1, 2), "i4"), out)
    with pytest.raises(MoebiusError, match="blocks are int32"):
        block_attention(q, k, v, E.DeviceArray(ctx, (1, 1, 1, 2)), out)
    with pytest.raises(MoebiusError, match="differ in shape"):
        block_attention(q, k, z(1, 31, 1, 8), blocks, out)
    with pytest.raises(MoebiusError, match="differ in type"):
        block_attention(q, k, v, blocks, Heads(E.DeviceArray(ctx, (1, 4, 2, 8)), 1, 4, 2, 8))
    with pytest.raises(MoebiusError, match="kv_len is int32"):
        block_attention(q, k, v, blocks, out, kv_len=E.DeviceArray(ctx, (2,), "i4"))
    with pytest.raises(MoebiusError, match="means are f32"):
        block_select(q, E.DeviceArray(ctx, (1, 2, 1, 8)), 32, blocks, kv_block=64)
    with pytest.raises(MoebiusError, match="means are f32"):
        block_means(k, 16, E.DeviceArray(ctx, (1, 1, 1, 8)))


@pytest.mark.parametrize("size", [1.0, 1e-4, 1e-8, 1e-20])
def test_blocks_of_zero_values_leave_small_ones_their_bits(ctx, size):
    """f32 values of any size beside listed blocks whose values are zero, or zero and infinite."""
    r = np.random.default_rng(10)
    q, k, v = (r.standard_normal((1, t, 1, 64)).astype(np.float32) for t in (192, 192, 192))
    v *= np.float32(size)
    v[0, 32:64], v[0, 96:128] = 0, 0
    for blocks in ([0, 1], [1, 2, 4], [1, 3], [0, 1, 2, 3, 4, 5]):
        li = np.tile(np.array(blocks + [-1] * (6 - len(blocks)), np.int32), (1, 2, 1, 1))
        want, tol = reference(q, k, v, li, 0.125, 96, 32, False, None, None)
        bound = tolerance(want, tol, 64, np.float32, False)
        got = run(ctx, q, k, v, li, 96, 32, scale=0.125)
        assert np.all(np.abs(got - want) <= bound), (blocks, (np.abs(got - want) / bound).max())
        inf = v.copy()
        inf[0, 40, 0, 7] = np.inf  # of block 1, which every list holds
        got = run(ctx, q, k, inf, li, 96, 32, scale=0.125)
        assert np.isposinf(got[..., 7]).all()
        assert np.all(np.delete(np.abs(got - want) <= bound, 7, axis=3)), blocks


@pytest.mark.parametrize("big", [1e8, 1e12, 1e30])
@pytest.mark.parametrize("d", [48, 33])
@pytest.mark.parametrize("q_block", [1, 16, 64, 128])
def test_large_values_of_unseen_keys_do_not_reach_a_row(ctx, q_block, d, big):
    """Causal f32 rows whose listed blocks hold keys and values of later tokens that are far larger than theirs."""
    r = np.random.default_rng(11)
    q, k, v = (r.standard_normal((1, 128, 2, d)).astype(np.float32) for _ in range(3))
    blocks = np.tile(np.arange(4, dtype=np.int32), (1, -(-128 // q_block), 2, 1))
    clean, tol = reference(q, k, v, blocks, d ** -0.5, q_block, 32, True, None, None)
    v[0, 40, 0, 5], v[0, 71:75, 1], v[0, 100] = big, -big, big
    k[0, 90, 0], k[0, 101, 1, 3] = big, -big
    got = run(ctx, q, k, v, blocks, q_block, 32, True).astype(np.float64)
    ok = np.abs(got - clean) <= tolerance(clean, tol, d, np.float32, False)
    assert ok[0, :40].all() and ok[0, :71, 1].all()
    # rows that see the large values: within the largest's roundings
    want, tol = reference(q, k, v, blocks, d ** -0.5, q_block, 32, True, None, None)
    ok = np.abs(got - want) <= tolerance(want, tol, d, np.float32, False)
    assert ok[0, :90].all() and ok[0, :101, 1].all()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [8, 64, 80, 160])
@pytest.mark.parametrize("q_block", [1, 64])
def test_tokens_of_sizes_far_apart(ctx, q_block, d, causal):
    """f32 keys and values that differ from token to token by more than the sixteen around them share, some
    of them zero; values grow along the cache, so causal rows see only what is small beside the rest."""
    r = np.random.default_rng(17)
    q, k, v = (r.standard_normal((2, t, 2, d)).astype(np.float32) for t in (160, 200, 200))
    k *= (10.0 ** r.uniform(-9, 0, (2, 200, 2, 1))).astype(np.float32)
    v *= (10.0 ** (np.arange(200) / 8 - 12)).astype(np.float32)[None, :, None, None]
    k[:, 5:90:11], v[:, 3:150:13] = 0, 0
    blocks = lists(r, 2, -(-160 // q_block), 2, 10, 13)
    got = run(ctx, q, k, v, blocks, q_block, 16, causal, [160, 130], [200, 187])
    want, tol = reference(q, k, v, blocks, d ** -0.5, q_block, 16, causal, [160, 130], [200, 187])
    there = ~np.isnan(want)
    bound = tolerance(want, tol, d, np.float32, False)
    assert np.all((np.abs(got - want) <= bound)[there]), (np.abs(got - want) / bound)[there].max()


@pytest.mark.parametrize("kind", ["f16", "f32", "fast"])
@pytest.mark.parametrize("q_block", [1, 64, 128])
def test_keys_of_infinite_score(ctx, q_block, kind):
    """A key whose score is -inf has no weight, one of +inf or NaN makes its rows NaN."""
    dtype = np.float16 if kind == "f16" else np.float32
    r = np.random.default_rng(13)
    q, k, v = (r.standard_normal((1, 128, 2, 40)).astype(dtype) for _ in range(3))
    q[..., 2:5] = np.abs(q[..., 2:5]) + 0.5
    q[0, ::3, :, 2:5] = 1  # exact in f16: low parts of zero
    blocks = np.tile(np.arange(4, dtype=np.int32), (1, -(-128 // q_block), 2, 1))
    k[0, 3, 0, 2] = k[0, 70, 0, 3] = k[0, 100:110, 0, 4] = -np.inf
    k[0, 33, 1, 2], k[0, 33, 1, 3] = -np.inf, -np.inf
    ctx.set_precision(kind == "fast")
    try:
        got = run(ctx, q, k, v, blocks, q_block, 32).astype(np.float64)
        k2 = k.copy()
        k2[0, 50, 0, 2], k2[0, 60, 1, 2], k2[0, 61, 1, 3] = np.inf, np.nan, -np.inf
        bad = run(ctx, q, k2, v, blocks, q_block, 32)
    finally:
        ctx.set_precision(False)
    k[~np.isfinite(k)] = -1e4  # as far below all others as makes no difference
    want, tol = reference(q, k, v, blocks, 40 ** -0.5, q_block, 32, False, None, None)
    tol[..., 1:3] = 20  # (the seen keys' own scores: |q| |k| scale stays below)
    assert np.all(np.abs(got - want) <= tolerance(want, tol, 40, dtype, kind == "fast"))
    assert np.isnan(bad).all() or kind == "fast" and np.isnan(bad[..., 1, :]).all()


@pytest.mark.parametrize("q_block", [1, 16, 128])
def test_infinite_values_on_fast_contexts(ctx, q_block):
    """Infinite f32 operands are taken as f16's largest, as finite ones beyond it are, by every row that sees
    them, whichever rows share its workgroup; NaN stays NaN."""
    r = np.random.default_rng(14)
    q, k, v = (r.standard_normal((1, 128, 1, 64)).astype(np.float32) for _ in range(3))
    blocks = np.tile(np.arange(4, dtype=np.int32), (1, -(-128 // q_block), 1, 1))
    v[0, 0, 0, 3], v[0, 70, 0, 5], v[0, 100, 0, 6], v[0, 90, 0, 7] = -np.inf, np.inf, 1e9, np.nan
    k[0, 110, 0, 9] = np.inf
    clean, tol = reference(q, np.clip(k, -65504, 65504), np.nan_to_num(np.clip(v, -65504, 65504)), blocks, 0.125, q_block, 32, True, None, None)
    ctx.set_precision(True)
    try:
        got = run(ctx, q, k, v, blocks, q_block, 32, True)
    finally:
        ctx.set_precision(False)
    assert np.isnan(got[0, 90:, 0, 7]).all()
    ok = np.abs(got - clean) <= tolerance(clean, tol, 64, np.float32, True)
    ok[0, 90:, 0, 7] = True
    assert ok.all()


@pytest.mark.parametrize("nk", [5900, 6007, 6100, 6144, 6145, 8192])
def test_select_of_many_blocks(ctx, nk):
    """Scores of single queries over as many blocks as the selection takes."""
    r = np.random.default_rng(nk)
    q, means = r.standard_normal((1, 1, 1, 8)).astype(np.float32), r.standard_normal((1, nk, 1, 8)).astype(np.float32)
    blocks = dev(ctx, np.zeros((1, 1, 1, 1000), np.int32))
    block_select(heads(ctx, q), dev(ctx, means), nk * 16, blocks, q_block=1, kv_block=16)
    assert np.array_equal(blocks.numpy(), selected(q, means, 1, 16, 1000, False, None, [nk * 16]))


@pytest.mark.parametrize("kind", ["f16", "f32", "fast"])
@pytest.mark.parametrize("case", [CASES[3], CASES[12], CASES[17], CASES[24]])
def test_items_alone_and_in_a_batch(ctx, case, kind):
    """Each item of a batch by itself: equal within both sides' roundings (lists are split by the work that there is)."""
    _, qt, kt, hq, hk, d, qb, kb, top, causal = case
    dtype = np.float16 if kind == "f16" else np.float32
    r = np.random.default_rng(15)
    q, k, v = (r.standard_normal(s).astype(dtype) for s in ((3, qt, hq, d), (3, kt, hk, d), (3, kt, hk, d)))
    blocks, kl, ql = lists(r, 3, -(-qt // qb), hk, top, -(-kt // kb)), [kt, kt // 2, kt - 1], [qt, qt, max(qt - 1, 1)]
    want, tol = reference(q, k, v, blocks, d ** -0.5, qb, kb, causal, ql, kl)
    bound = tolerance(want, tol, d, dtype, kind == "fast")
    ctx.set_precision(kind == "fast")
    try:
        whole = run(ctx, q, k, v, blocks, qb, kb, causal, ql, kl)
        for i in range(3):
            one = run(ctx, q[i:i + 1], k[i:i + 1], v[i:i + 1], blocks[i:i + 1], qb, kb, causal, ql[i:i + 1], kl[i:i + 1])
            there = ~np.isnan(want[i])
            diff = np.abs(one[0].astype(np.float64) - whole[i])
            assert np.all(diff[there] <= 2 * bound[i][there])
    finally:
        ctx.set_precision(False)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("q_block", [1, 16])
def test_lists_of_the_same_order_agree_in_bits(ctx, dtype, q_block):
    """Places that are empty, outside or listed before change nothing of a list, in bits."""
    r = np.random.default_rng(16)
    q, k, v = (r.standard_normal((1, t, 1, 40)).astype(dtype) for t in (16, 640, 640))
    tile = lambda b: np.tile(np.array(b, np.int32), (1, 16 // q_block, 1, 1))  # noqa: E731
    a = run(ctx, q, k, v, tile([20, 3, 39, 7, -1, -1, -1, -1]), q_block, 16)
    b = run(ctx, q, k, v, tile([-1, 20, 3, 20, 50, 39, 3, 7]), q_block, 16)
    assert np.array_equal(a, b)


def test_split_operands_captured_and_replayed(ctx):
    """Two graphs of f32 calls whose keys are split, lists too, with scratch of their own, replayed among eager
    calls in the context's workspace."""
    r = np.random.default_rng(19)
    blocks = dev(ctx, np.tile(np.arange(20, dtype=np.int32), (1, 2, 1, 1)))
    calls, wants = [], []
    for _ in range(2):
        q, k, v = (heads(ctx, r.standard_normal((1, t, 1, 72)).astype(np.float32)) for t in (128, 640, 640))
        out = heads(ctx, np.zeros((1, 128, 1, 72), np.float32))
        scratch = E.DeviceArray(ctx, (block_attention_scratch(q, k, blocks, 64, 32),), np.uint8)
        assert scratch.nbytes >= 640 * 72 * 8
        calls.append((q, k, v, out, scratch))
        block_attention(q, k, v, blocks, out, q_block=64, kv_block=32)
        wants.append(out.numpy())
    with pytest.raises(MoebiusError, match="captured call needs scratch"):
        capture(ctx, lambda: block_attention(*calls[0][:3], blocks, calls[0][3], q_block=64, kv_block=32))
    graphs = [capture(ctx, lambda c=c: block_attention(*c[:3], blocks, c[3], q_block=64, kv_block=32, scratch=c[4])) for c in calls]
    eager = heads(ctx, np.zeros((1, 128, 1, 72), np.float32))
    for turn in range(4):
        for c in calls:
            c[3].buf.upload(np.zeros((1, 128, 1, 72), np.float32))
        for launch, _ in graphs:
            launch()
        block_attention(*calls[turn % 2][:3], blocks, eager, q_block=64, kv_block=32)
        ctx.synchronize()
        for c, want in zip(calls, wants):
            assert np.array_equal(c[3].numpy(), want)
        assert np.array_equal(eager.numpy(), wants[turn % 2])
    for _, destroy in graphs:
        destroy()
