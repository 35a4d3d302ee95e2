"""The token operators as an attention block of image tokens uses them: projections
with adapters, norms and rotation where the projection left queries and keys, block
means, selection and attention, over a padded batch; every stage against its
definition in f64 of what it read on the device, within its own tests' tolerances,
eager and as two graphs."""
from __future__ import annotations

import numpy as np
import pytest

from moebius_cpu_amd import engine as E
from moebius_cpu_amd.adapters import Adapters
from moebius_cpu_amd.attention import (Heads, RopeAxes, block_attention, block_attention_scratch, block_means,
                                       block_select, qk_norm_rope)
from tests import test_gpu_block_attention as A
from tests import test_gpu_lora as L
from tests import test_gpu_rope as R
from tests.graph_capture import capture

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    return E.Context(0)


class Block:
    """n requests of at most `tokens` tokens of c channels."""
    def __init__(self, ctx, n, tokens, c, hq, hk, d, kb, top, qb, causal, lengths, seed):
        r = np.random.default_rng(seed)
        self.ctx, self.n, self.tokens, self.c, self.hq, self.hk, self.d = ctx, n, tokens, c, hq, hk, d
        self.kb, self.top, self.qb, self.causal, self.lengths = kb, top, qb, causal, lengths
        wide, rank, slots = (hq + 2 * hk) * d, 8, 3
        self.h = dict(x=r.standard_normal((n, 1, tokens, c)).astype(np.float32),
                      gq=(1 + 0.2 * r.standard_normal(d)).astype(np.float32), gk=(1 + 0.2 * r.standard_normal(d)).astype(np.float32),
                      pos=np.stack([np.arange(tokens) // 20, np.arange(tokens) % 20], 1).astype(np.int32),
                      slot=(np.arange(n) % (slots + 1) - 1).astype(np.int32))
        self.layers = []
        for ci, co in ((c, wide), (hq * d, c)):
            p = dict(w=(r.standard_normal((co, ci)) / np.sqrt(ci)).astype(np.float16), bias=r.standard_normal(co).astype(np.float32),
                     a=(r.standard_normal((slots, rank, ci)) / np.sqrt(ci)).astype(np.float16),
                     b=(0.3 * r.standard_normal((slots, co, rank))).astype(np.float16), scale=r.uniform(0.5, 2, slots).astype(np.float32))
            conv = E.Conv1x1(ctx, ci, co, E.Param(ctx, p["w"], f16=True), p["bias"])
            self.layers.append((conv, Adapters(ctx, E.Param(ctx, p["a"], f16=True), E.Param(ctx, p["b"], f16=True), p["scale"], ci, co, rank), p))
        dev = lambda a: E.DeviceArray.from_numpy(ctx, a)  # noqa: E731
        self.x, self.slot, self.pos, self.gq, self.gk = E.Tensor.from_numpy(ctx, self.h["x"]), *(dev(self.h[k]) for k in ("slot", "pos", "gq", "gk"))
        self.len = dev(np.asarray(lengths, np.int32))
        self.rope = RopeAxes(ctx, (d // 2, d // 2))
        self.qkv = E.Tensor(ctx, n, 1, tokens, wide)
        self.q, self.k, self.v = (Heads(self.qkv, n, tokens, h, d, ld=wide, offset=o * d) for h, o in ((hq, 0), (hk, hq), (hk, hq + hk)))
        self.mixed = E.Tensor.from_numpy(ctx, np.zeros((n, 1, tokens, hq * d)))
        self.out = E.Tensor(ctx, n, 1, tokens, c)
        self.means = dev(np.zeros((n, -(-tokens // kb), hk, d), np.float32))
        self.blocks = dev(np.zeros((n, -(-tokens // qb), hk, top), np.int32))
        rows = n * tokens
        self.scratch = [E.DeviceArray(ctx, (max(b, 16),), np.uint8) for b in (
            *(ad.scratch(rows, conv.weight) for conv, ad, _ in self.layers), block_attention_scratch(self.q, self.k, self.blocks, qb, kb))]

    def project(self, scratch):
        self.layers[0][0].forward_adapted(self.x, self.layers[0][1], self.slot, self.qkv, scratch=scratch)

    def turn(self):
        qk_norm_rope(self.q, self.k, self.gq, self.gk, 1e-6, self.pos, self.rope, self.q, self.k)

    def select(self):
        block_means(self.k, self.kb, self.means, length=self.len)
        block_select(self.q, self.means, self.tokens, self.blocks, self.qb, self.kb, self.causal, self.len, self.len)

    def attend(self, scratch):
        block_attention(self.q, self.k, self.v, self.blocks, Heads(self.mixed, self.n, self.tokens, self.hq, self.d), None,
                        self.qb, self.kb, self.causal, self.len, self.len, scratch)

    def finish(self, scratch):
        self.layers[1][0].forward_adapted(self.mixed, self.layers[1][1], self.slot, self.out, residual=self.x, scratch=scratch)

    def run(self, scratch=(None, None, None)):
        self.project(scratch[0])
        self.turn()
        self.select()
        self.attend(scratch[2])
        self.finish(scratch[1])

    def check_projection(self, x, layer, got, res):
        p = self.layers[layer][2]
        co, ci = p["w"].shape
        y, base, low = L.reference(x.reshape(-1, ci), p["w"], p["bias"], res, p["a"], p["b"], p["scale"], self.h["slot"], self.tokens)
        bound = 1e-5 * base + (ci + 16) * U * low + U * np.abs(y)
        assert np.all(np.abs(got.reshape(-1, co) - y) <= bound)


@pytest.mark.parametrize("shape", [
    dict(n=2, tokens=300, c=320, hq=8, hk=2, d=40, kb=32, top=5, qb=64, causal=False, lengths=[300, 217]),
    dict(n=4, tokens=256, c=640, hq=8, hk=8, d=80, kb=64, top=3, qb=128, causal=True, lengths=[256, 1, 0, 129]),
    dict(n=3, tokens=20, c=96, hq=4, hk=1, d=64, kb=16, top=2, qb=4, causal=False, lengths=[20, 17, 3])])
def test_block(ctx, shape):
    states = [Block(ctx, **shape, seed=s) for s in (1, 2)]
    for b in states:
        b.project(None)
        raw = b.qkv.numpy()
        b.check_projection(b.h["x"], 0, raw, None)
        b.turn()
        heads = raw.reshape(b.n * b.tokens, -1, b.d).astype(np.float64)
        for got, part, g in ((b.q, heads[:, :b.hq], b.h["gq"]), (b.k, heads[:, b.hq:b.hq + b.hk], b.h["gk"])):
            want, size = R.turn64(R.norm64(part, g.astype(np.float64), np.float64(np.float32(1e-6))), b.h["pos"],
                                  (b.d // 2, b.d // 2), 10000.0, False)
            assert np.all(np.abs(got.numpy().reshape(want.shape) - want) <= 5e-7 * size)
        q, k, v = b.q.numpy(), b.k.numpy(), b.v.numpy()
        assert np.array_equal(v.reshape(-1), raw.reshape(b.n * b.tokens, -1, b.d)[:, b.hq + b.hk:].reshape(-1))
        b.select()
        means, blocks = b.means.numpy(), b.blocks.numpy()
        for i, n in enumerate(b.lengths):
            for j in range(-(-n // b.kb)):
                part = k[i, j * b.kb:min((j + 1) * b.kb, n)].astype(np.float64)
                assert np.all(np.abs(means[i, j] - part.mean(0)) <= U * np.abs(part.mean(0)) + 1e-13 * np.abs(part).max())
        assert np.array_equal(blocks, A.selected(q, means, b.qb, b.kb, b.top, b.causal, b.lengths, b.lengths))
        b.attend(None)
        mixed = b.mixed.numpy().reshape(q.shape)
        want, tol = A.reference(q, k, v, blocks, 1 / np.sqrt(b.d), b.qb, b.kb, b.causal, b.lengths, b.lengths)
        there = ~np.isnan(want)
        assert np.all(mixed[~there] == 0)  # behind the lengths: as they were
        assert np.all(np.abs(mixed - want)[there] <= A.tolerance(want, tol, b.d, np.float32, False)[there])
        b.finish(None)
        b.check_projection(b.mixed.numpy(), 1, b.out.numpy(), b.h["x"].reshape(-1, b.c))
    wants = [b.out.numpy() for b in states]
    graphs = [capture(ctx, lambda b=b: b.run(b.scratch)) for b in states]
    for turn in range(4):
        for b in states:
            b.out.upload(np.zeros(b.out.shape, np.float32))
        for launch, _ in graphs:
            launch()
        ctx.synchronize()
        for b, want in zip(states, wants):
            assert np.array_equal(b.out.numpy(), want)
        states[turn % 2].run()  # eager, in the context's workspace
        assert np.array_equal(states[turn % 2].out.numpy(), wants[turn % 2])
    for _, destroy in graphs:
        destroy()
