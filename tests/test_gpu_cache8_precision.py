"""What the attention over a cache in 8 bits makes of probabilities."""
from __future__ import annotations

import numpy as np
import pytest

from moebius_cpu_amd import engine as E
from moebius_cpu_amd.cache import cache_attention
from tests.test_gpu_block_attention import dev, heads, lens
from tests.test_gpu_cache8 import F32, SHARED, Case, attention64

pytestmark = pytest.mark.gpu
F16 = np.float16


@pytest.fixture(scope="module")
def contexts():
    exact, fast = E.Context(0), E.Context(0)
    fast.set_precision(True)
    return exact, fast


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
