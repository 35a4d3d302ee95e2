"""What the attention over a cache in 8 bits makes of probabilities far below a row's largest, of
scales of values far apart, and of values near the end of f32.

Bounds, beside those of test_gpu_cache8 (e below, from the f32 sums, exponents and FAST queries), for a
row with probabilities p_j relative to its largest, z = sum p_j, over values v_j = code_j s_j that it
sees, |code_j| <= 127:
  - a probability in one f16 is off by 2^-11 of itself, in two by 2^-22;
  - or by half of f16's last step, 2^-25, of what it is stored against: p_j s_j 2^(L - E) with the sums'
    exponent E at most 4 above that of s_j (3, and s_j may be half of its power of two), L = 7 for one
    part and 12 for two. That is 2^-28 or 2^-33 of 127 s_j, for every key, over z;
  - f16 outputs add half a step.
"""
from __future__ import annotations

import numpy as np
import pytest

from moebius_cpu_amd import engine as E
from moebius_cpu_amd.cache import cache_attention, cache_attention_scratch, cache_write
from tests.test_gpu_block_attention import dev, heads, lens
from tests.test_gpu_cache8 import F32, SHARED, U, Case, attention64, visible

pytestmark = pytest.mark.gpu
F16 = np.float16
# type, FAST
KINDS = [(F32, False), (F16, False), (F32, True), (F16, True)]
NAMES = ["f32", "f16", "f32-fast", "f16-fast"]


@pytest.fixture(scope="module")
def contexts():
    exact, fast = E.Context(0), E.Context(0)
    fast.set_precision(True)
    return exact, fast


def row_bound(q, k, v, scales, seen, scale, fast):
    """Of one item and key head: q [ql][d], k and v [kl][d] as the cache holds them, the scales [kl] of the
    values' blocks. out [ql][d] and the bound on its error."""
    dtype, x = q.dtype, q.astype(np.float64)
    d, kl = x.shape[1], len(k)
    s = scale * x @ k.T
    a = np.where(seen, scale * np.abs(x) @ np.abs(k).T, 0).max(1)
    least = scale * np.abs(x).max(1) * np.where(seen, np.abs(k).sum(1), 0).max(1)
    b = np.where(seen, np.abs(s), 0).max(1) * 1.4427 + 8
    m = np.where(seen, s, -np.inf).max(1, keepdims=True)
    p = np.where(seen, np.exp(s - np.where(np.isfinite(m), m, 0)), 0)
    z = np.where(p.sum(1, keepdims=True) > 0, p.sum(1, keepdims=True), 1)
    o, size = p @ v / z, p @ np.abs(v) / z
    e = (2 * d + 9) * U * a + 2.0 ** -39 * least + 2.0 ** -23 * b + 2.0 ** -22 + (kl + kl / 64 + 4) * U
    if dtype == F32 and fast:
        e = e + 2.0 ** -11 * a + 2.0 ** -25 * least
    err = (np.expm1(2 * e)[:, None] + (2.0 ** -11 * 1.001 if fast else 2.0 ** -22)) * size
    err = err + 2.0 ** (-28 if fast else -33) * 127 * (seen * scales).sum(1, keepdims=True) / z
    if dtype == F16:
        return o, err + 2.0 ** -11 * (np.abs(o) + err) + 2.0 ** -25
    return o, err + U * np.abs(o)


def check(c, scale, fast):
    """Every row of a Case against row_bound."""
    got = c.out.numpy().astype(np.float64)
    n, _, hq, _ = c.qh.shape
    hk = c.held.codes.shape[2]
    for i in range(n):
        ql, kl = int(c.q_len[i]), int(c.kv_len[i])
        if not ql or not kl:
            continue
        (k, there), (v, _) = (c.held.values(w, c.table, i, kl) for w in (0, 1))
        seen = visible(ql, kl, *c.kw.values()) & there[None]
        page = c.table[i, np.arange(kl) // c.held.block]
        for h in range(hq):
            x = h // (hq // hk)
            scales = np.where(there, c.held.scale[1, np.where(there, page, 0), x], 0).astype(np.float64)
            want, tol = row_bound(c.qh[i, :ql, h], k[:, x], v[:, x], scales, seen, scale, fast)
            off = np.abs(got[i, :ql, h] - want)
            assert np.isfinite(got[i, :ql, h]).all() and np.all(off <= tol), (i, h, (off / np.maximum(tol, 1e-300)).max())


# ---------------------------------------------------------------- f16 rows that share tokens

@pytest.mark.parametrize("case", [SHARED[i] for i in (1, 3, 4, 6, 8, 12, 13, 15, 16, 18)],
                         ids=lambda c: "-".join(str(c[k]) for k in ("n", "q", "kv", "hk", "d", "block")))
def test_f16_rows_that_share_tokens_round_once(contexts, case):
    """As rows alone: off by what f32 calls are, and half a step of the output."""
    c = Case(contexts[0], F16, **case)
    c.run()
    want, tol = attention64(c.qh.astype(F32), c.held, c.table, 1 / np.sqrt(case["d"]), *c.kw.values(), c.q_len, c.kv_len)
    there = ~np.isnan(want)
    off, tol = np.abs(c.out.numpy().astype(np.float64) - want)[there], tol[there]
    tol = tol + 2.0 ** -11 * (np.abs(want[there]) + tol) + 2.0 ** -25
    assert np.all(off <= tol), (off / tol).max()


@pytest.mark.parametrize("d,hq,hk", [(64, 2, 1), (128, 4, 2)])
def test_f16_rows_alone_and_shared_agree(contexts, d, hq, hk):
    """The rows of one item are the same numbers, but for rounding, whether other items fill the card or not."""
    n, q, kv = 64, 140, 300
    c = Case(contexts[0], F16, n=n, q=q, kv=kv, hq=hq * 4, hk=hk * 4, d=d, block=64)
    c.run()
    one = c.out.numpy()[:1].astype(np.float64)
    own = heads(contexts[0], np.zeros((1, q, hq * 4, d), F16))
    cache_attention(heads(contexts[0], c.qh[:1]), c.cache, dev(contexts[0], c.table[:1]), own,
                    kv_len=lens(contexts[0], [kv]))
    alone = own.numpy().astype(np.float64)
    # each is the rounding of a value that is off by about 2^-21 of the probabilities' weights
    assert np.all(np.abs(alone - one) <= 2.0 ** -10 * np.abs(alone) + 2.0 ** -24 + 2.0 ** -18 * np.abs(c.held.scale).max() * 127)
    assert np.mean(alone != one) < 0.02  # few of them lie that near to a border of two f16


@pytest.mark.parametrize("case", [SHARED[i] for i in (1, 3, 8, 12, 16)], ids=lambda c: "-".join(str(c[k]) for k in ("n", "q", "kv", "hk", "d", "block")))
def test_f16_rows_that_share_tokens_fast(contexts, case):
    c = Case(contexts[1], F16, **case)
    c.run()
    c.check()


# ---------------------------------------------------------------- probabilities far below the largest

def tail_case(ctx, dtype, block, n, q, hk, d, hidden, kv):
    """A block of values 2^9.9 larger that the window hides or that has no weight; then keys that are alike, and one whose
    score is 2^14.5 times theirs and whose value is zero."""
    k, v = np.zeros((1, kv, hk, d)), np.zeros((1, kv, hk, d))
    k[..., 0] = -14.5 * np.log(2.0) / 8
    k[:, kv - 1] = 0
    if not hidden:
        k[:, :block, :, 0] = -60 / 8
    v[:] = np.where(np.arange(d) % 3 == 1, -0.5, 1.0)
    v[:, :block] *= 2.0 ** 9.9
    v[:, kv - 1] = 0
    c = Case(ctx, dtype, n=n, q=q, kv=kv, hq=hk, hk=hk, d=d, block=block, window=kv - q - block + 1 if hidden else 0, causal=False)
    c.table[:] = c.table[:1]  # every item reads the same pages
    c.dtable = dev(ctx, c.table)
    x = [y.astype(dtype) for y in (k, v)]
    c.held.write(c.table[:1], x, [0], [kv])
    cache_write(c.cache, dev(ctx, c.table[:1]), heads(ctx, x[0]), heads(ctx, x[1]))
    c.qh[:] = 0
    c.qh[..., 0] = 8
    c.q = heads(ctx, c.qh)
    return c


TAILS = [  # n, q, key heads, d, tokens: few rows, few rows split, rows that share tokens in workgroups of four and of eight waves
    (2, 9, 2, 80, 500), (1, 3, 1, 128, 4000), (64, 70, 4, 64, 500), (16, 70, 16, 160, 500), (32, 130, 8, 128, 500), (1, 80, 1, 64, 4300)]


@pytest.mark.parametrize("dtype,fast", KINDS, ids=NAMES)
@pytest.mark.parametrize("block,hidden", [(16, True), (16, False), (64, False)])
@pytest.mark.parametrize("n,q,hk,d,kv", TAILS)
def test_many_small_probabilities_behind_large_values(contexts, dtype, fast, block, hidden, n, q, hk, d, kv):
    c = tail_case(contexts[fast], dtype, block, n, q, hk, d, hidden, kv)
    c.run(scale=1.0)
    if not hidden:  # all rows and items are alike
        got = c.out.numpy()
        assert np.all(got == got[:1, :1])
    c.q_len = np.array([q if i in (0, n - 1) else 0 for i in range(n)])
    check(c, 1.0, fast)


# ---------------------------------------------------------------- scales of values far apart

@pytest.mark.parametrize("dtype,fast", KINDS, ids=NAMES)
@pytest.mark.parametrize("block", [16, 64, 128])
@pytest.mark.parametrize("n,q,cap,hk,d,window", [(3, 1, 512, 2, 64, 40), (2, 5, 300, 2, 80, 8), (64, 70, 200, 4, 64, 8), (32, 130, 260, 8, 80, 40),
                                                 (32, 130, 260, 8, 128, 0), (1, 150, 4200, 2, 128, 0)])
def test_rows_beside_a_jump_in_scale(contexts, dtype, fast, block, n, q, cap, hk, d, window):
    """Blocks of values up to 2^21 apart: rows of one tile on both sides of a jump, and rows that see one block alone."""
    r = np.random.default_rng(cap + q + block)
    blocks = -(-cap // block)
    kv_len = [min(300, cap) - (i * 37) % 150 for i in range(n)]
    q_len = [min(q, x) for x in kv_len]
    ctx = contexts[fast]
    c = Case(ctx, dtype, n=n, q=q, kv=cap, hq=2 * hk, hk=hk, d=d, block=block, q_len=q_len, kv_len=kv_len, window=window, std=0.25)
    exps = r.choice([9, 2, 0, -2, -12], blocks)
    exps[:3] = [9, -12, -2][:blocks]  # a jump among the first tokens
    size = np.repeat(np.exp2(exps), block)[None, :cap, None, None]
    x = [(0.25 * r.standard_normal((n, cap, hk, d))).astype(dtype), (size * r.standard_normal((n, cap, hk, d))).astype(dtype)]
    c.held.write(c.table, x, np.zeros(n, int), kv_len)
    cache_write(c.cache, c.dtable, heads(ctx, x[0]), heads(ctx, x[1]), length=lens(ctx, kv_len))
    c.run()
    c.q_len = np.array([q_len[i] if i in (0, 1, n - 1) else 0 for i in range(n)])
    check(c, 1 / np.sqrt(d), fast)


@pytest.mark.parametrize("dtype,fast", KINDS, ids=NAMES)
@pytest.mark.parametrize("block", [16, 64])
def test_windows_of_small_values_in_splits(contexts, dtype, fast, block):
    """Single tokens that give weight to small values alone, among the first tokens and in their window, over so many that
    they are split, with large ones between them and, without weight, inside the window."""
    kv, window, sinks, d = 4096, 1024, 128, 80
    ctx = contexts[fast]
    c = Case(ctx, dtype, n=2, q=1, kv=kv, hq=4, hk=2, d=d, block=block, window=window, sinks=sinks)
    assert cache_attention_scratch(c.q, c.cache, c.dtable, window, sinks) > 0
    r, at = np.random.default_rng(block), np.arange(kv)
    large = ((at >= sinks) & (at < kv - window)) | ((at >= 3328) & (at < 3456))
    k, v = 0.25 * r.standard_normal((2, kv, 2, d)), np.where(large, 1, 2.0 ** -13)[None, :, None, None] * r.standard_normal((2, kv, 2, d))
    k[..., 0] = np.where(large, -60 * np.sqrt(d) / 16, 0)[None, :, None]
    c.qh[..., 0] = 16
    c.q = heads(ctx, c.qh)
    x = [k.astype(dtype), v.astype(dtype)]
    c.held.write(c.table, x, [0, 0], [kv, kv])
    cache_write(c.cache, c.dtable, heads(ctx, x[0]), heads(ctx, x[1]))
    c.run()
    check(c, 1 / np.sqrt(d), fast)


# ---------------------------------------------------------------- values near the end of f32

@pytest.mark.parametrize("fast", [False, True])
@pytest.mark.parametrize("block", [16, 64])
@pytest.mark.parametrize("n,q,hq,hk,d,kv", [(1, 1, 4, 2, 80, 300), (2, 40, 4, 2, 64, 200), (1, 1, 2, 1, 128, 4000), (64, 70, 4, 4, 64, 300),
                                            (32, 130, 8, 8, 128, 300), (1, 80, 2, 2, 80, 4300)])
def test_values_near_the_end_of_the_range(contexts, fast, block, n, q, hq, hk, d, kv):
    """Means of values of up to 3.4e38 are finite: no sum leaves its power of two before it is divided."""
    ctx = contexts[fast]
    c = Case(ctx, F32, n=n, q=q, kv=kv, hq=hq, hk=hk, d=d, block=block, std=0.25)
    r = np.random.default_rng(kv)
    x = [r.standard_normal((n, kv, hk, d)).astype(F32), ((0.9 + 0.1 * r.random((n, kv, hk, d))) * np.finfo(F32).max).astype(F32)]
    c.held.write(c.table, x, np.zeros(n, int), c.kv_len)
    cache_write(c.cache, c.dtable, heads(ctx, x[0]), heads(ctx, x[1]))
    c.run()
    keep = {0, n - 1}
    c.q_len = np.array([c.q_len[i] if i in keep else 0 for i in range(n)])
    check(c, 1 / np.sqrt(d), fast)


# ---------------------------------------------------------------- scores whose steps are coarse

@pytest.mark.parametrize("dtype,fast", KINDS, ids=NAMES)
@pytest.mark.parametrize("block", [16, 64])
@pytest.mark.parametrize("factor", [8, 32])
@pytest.mark.parametrize("n,q,hk", [(1, 2, 1), (64, 70, 4), (32, 130, 8)])
def test_maxima_that_grow_by_steps_of_large_scores(contexts, dtype, fast, block, factor, n, q, hk):
    """Scores of 2^26 and 2^28 whose maximum grows by a step or two of f32 from chunk to chunk: probabilities stay within f16.
    All values are the same, and so is their mean, whatever the weights."""
    ctx, kv, d = contexts[fast], 640, 64 if hk < 8 else 128
    c = Case(ctx, dtype, n=n, q=q, kv=kv, hq=hk, hk=hk, d=d, block=block, causal=False)
    c.table[:] = c.table[:1]
    c.dtable = dev(ctx, c.table)
    k = np.zeros((1, kv, hk, d))
    k[..., 0], k[..., 1] = 127, (np.arange(kv) // 64)[None, :, None]
    v = np.full((1, kv, hk, d), 127 * (1 - 2.0 ** -10))  # a scale just below a power of two
    x = [k.astype(dtype), v.astype(dtype)]
    cache_write(c.cache, dev(ctx, c.table[:1]), heads(ctx, x[0]), heads(ctx, x[1]))
    c.qh[:] = 0
    c.qh[..., 0], c.qh[..., 1] = 65504, 0.5
    c.q = heads(ctx, c.qh)
    c.run(scale=factor / 1.4426950408889634)
    want = float(x[1].flat[0])
    # f32 sums of kv products and of the probabilities, the codes' scale, and the output's rounding
    tol = want * ((2.0 ** -11 * 1.001 if fast else 2.0 ** -22) + 2 * (kv + 16) * U + (2.0 ** -11 if dtype == F16 else U))
    got = c.out.numpy().astype(np.float64)
    assert np.isfinite(got).all() and np.all(np.abs(got - want) <= tol), np.abs(got - want).max() / tol
