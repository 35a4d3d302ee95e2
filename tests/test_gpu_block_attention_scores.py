"""Attention over listed blocks where a row's scores are so large that f32 holds them in steps of 4 and 16."""
from __future__ import annotations

import numpy as np
import pytest

from moebius_cpu_amd import engine as E
from moebius_cpu_amd.attention import block_attention
from tests.test_gpu_block_attention import dev, heads

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,fast", [(np.float32, False), (np.float32, True), (np.float16, False)])
@pytest.mark.parametrize("factor", [8, 32])
@pytest.mark.parametrize("q_block,hk,d", [(1, 2, 64), (32, 4, 64), (64, 8, 128)])
def test_maxima_that_grow_by_steps_of_large_scores(dtype, fast, factor, q_block, hk, d):
    """Scores of 2^26 and 2^28 whose maximum grows by a step or two of f32 from block to block: probabilities stay within
    f16. All values are the same, and so is their mean, whatever the weights."""
    ctx, n, qt, kv = E.Context(0), 2, 256, 640
    ctx.set_precision(fast)
    q, k = np.zeros((n, qt, 2 * hk, d), dtype), np.zeros((n, kv, hk, d), dtype)
    q[..., 0], q[..., 1] = 65504, 0.5
    k[..., 0], k[..., 1] = 128, (np.arange(kv) // 64)[:, None]
    v = np.full((n, kv, hk, d), 1 - 2.0 ** -10, dtype)
    blocks = dev(ctx, np.broadcast_to(np.arange(10, dtype=np.int32), (n, -(-qt // q_block), hk, 10)))
    out = heads(ctx, np.zeros_like(q))
    block_attention(heads(ctx, q), heads(ctx, k), heads(ctx, v), blocks, out, scale=factor / 1.4426950408889634,
                    q_block=q_block, kv_block=64)
    got, want = out.numpy().astype(np.float64), float(v.flat[0])
    # f32 sums of kv products and of the probabilities, those in one part or two, and the output's rounding
    one = fast or dtype == np.float16
    tol = want * ((2.0 ** -11 * 1.001 if one else 2.0 ** -22) + 2 * (kv + 16) * 2.0 ** -24 + (2.0 ** -11 if dtype == np.float16 else 2.0 ** -24))
    assert np.isfinite(got).all() and np.all(np.abs(got - want) <= tol), np.abs(got - want).max() / tol
    ctx.close()
