"""The operators of a stream as a block of a token transformer uses them: modulated norm, projection,
norms and rotation of its heads, keys and values into the cache, attention over it with a window and
first tokens, projection, gated residual with the next norm; a prompt, then token after token for
requests of different lengths. Every stage against its definition in f64 of what it read on the
device, within its own tests' tolerances, eager and as two graphs replayed token after token."""
from __future__ import annotations

import numpy as np
import pytest

from moebius_cpu_amd import engine as E
from moebius_cpu_amd._lib import MoebiusError
from moebius_cpu_amd.attention import Heads, RopeAxes, qk_norm_rope
from moebius_cpu_amd.cache import Cache8, cache_attention, cache_attention_scratch, cache_read, cache_write
from moebius_cpu_amd.gated_norm import Norm, gated_norm
from tests import test_gpu_cache8 as K
from tests import test_gpu_gated_norm as G
from tests import test_gpu_rope as R
from tests.graph_capture import capture

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    return E.Context(0)


class Stream:
    """n requests; one call takes `tokens` new tokens of c channels of each."""
    def __init__(self, ctx, n, tokens, c, hq, hk, d, block, window, sinks, blocks, seed):
        r = np.random.default_rng(seed)
        self.ctx, self.n, self.tokens, self.c, self.hq, self.hk, self.d = ctx, n, tokens, c, hq, hk, d
        self.window, self.sinks, wide = window, sinks, (hq + 2 * hk) * d
        dev = lambda a: E.DeviceArray.from_numpy(ctx, np.ascontiguousarray(a))  # noqa: E731
        self.dev = dev
        self.table = K.pages(r, n, blocks)
        self.cache, self.held = Cache8(ctx, n * blocks + 3, hk, d, block), K.Held(n * blocks + 3, hk, d, block)
        K.blank(self.cache)
        self.dtable = dev(self.table)
        self.w = [(r.standard_normal((co, ci)) / np.sqrt(ci)).astype(np.float32) for ci, co in ((c, wide), (hq * d, c))]
        self.conv = [E.Conv1x1(ctx, w.shape[1], w.shape[0], E.Param(ctx, w), None) for w in self.w]
        self.g = [(1 + 0.2 * r.standard_normal(k)).astype(np.float32) for k in (d, d, c)]
        self.dg = [dev(g) for g in self.g]
        self.mod = (0.4 * r.standard_normal((n, 5 * c))).astype(np.float32)
        self.dmod = dev(self.mod)
        self.vec = [Heads(self.dmod, n, 1, 1, c, ld=5 * c, offset=i * c) for i in range(5)]
        self.rope, self.pre, self.post = RopeAxes(ctx, (d,)), Norm("layer", eps=1e-6), Norm("rms", self.dg[2], None, 1e-6)
        self.x, self.y, self.out = (E.Tensor.from_numpy(ctx, np.zeros((n, 1, tokens, c), np.float32)) for _ in range(3))
        self.branch = E.Tensor.from_numpy(ctx, np.zeros((n, 1, tokens, c), np.float32))
        self.qkv = E.Tensor(ctx, n, 1, tokens, wide)
        self.q, self.k, self.v = (Heads(self.qkv, n, tokens, h, d, ld=wide, offset=o * d) for h, o in ((hq, 0), (hk, hq), (hk, hq + hk)))
        self.mixed = E.Tensor.from_numpy(ctx, np.zeros((n, 1, tokens, hq * d), np.float32))
        self.pos, self.first, self.kv_len, self.q_len = (dev(np.zeros(s, np.int32)) for s in ((n * tokens, 1), n, n, n))
        self.rows = lambda t: Heads(t, n, tokens, 1, c)  # noqa: E731
        self.heads = Heads(self.mixed, n, tokens, hq, d)
        need = cache_attention_scratch(self.q, self.cache, self.dtable, window, sinks)
        self.scratch = E.DeviceArray(ctx, (max(need, 16),), np.uint8)

    def feed(self, x, at, new):
        """New tokens x behind `at` [n], `new` [n] of them there."""
        self.at, self.new = np.asarray(at), np.asarray(new)
        self.x.upload(x.reshape(self.x.shape))
        self.pos.upload((self.at[:, None] + np.arange(self.tokens)).reshape(-1, 1))
        self.first.upload(self.at), self.q_len.upload(self.new), self.kv_len.upload(self.at + self.new)

    def stages(self, scratch=None):
        yield gated_norm(self.rows(self.x), pre=self.pre, scale=self.vec[0], shift=self.vec[1], y=self.rows(self.y))
        yield self.conv[0].forward(self.y, self.qkv)
        yield qk_norm_rope(self.q, self.k, self.dg[0], self.dg[1], 1e-6, self.pos, self.rope, self.q, self.k)
        yield cache_write(self.cache, self.dtable, self.k, self.v, first=self.first, length=self.q_len)
        yield cache_attention(self.q, self.cache, self.dtable, self.heads, window=self.window, sinks=self.sinks,
                              q_len=self.q_len, kv_len=self.kv_len, scratch=scratch)
        yield self.conv[1].forward(self.mixed, self.branch)
        yield gated_norm(self.rows(self.x), branch=self.rows(self.branch), post=self.post, gate=self.vec[2], x_out=self.rows(self.out),
                         pre=self.pre, scale=self.vec[3], shift=self.vec[4], y=self.rows(self.y))

    def run(self, scratch=None):
        for _ in self.stages(scratch):
            pass

    def vectors(self, *which):
        return [None if i is None else self.mod[:, i * self.c:(i + 1) * self.c] for i in which]

    def project(self, x, w, got):
        x = x.reshape(-1, w.shape[1]).astype(np.float64)
        want, size = x @ w.T.astype(np.float64), np.abs(x) @ np.abs(w.T.astype(np.float64))
        assert np.all(np.abs(got.reshape(want.shape) - want) <= 1e-5 * size)

    def checked(self):
        c, eps = self.c, np.float64(np.float32(1e-6))
        run, x = self.stages(), self.x.numpy()[:, 0]
        next(run)
        y = self.y.numpy()
        layer, none = ("layer", None, None, eps), ("none", None, None, eps)
        _, _, want, e = G.reference(x, None, none, None, 1.0, layer, *self.vectors(0, 1))
        G.near(y[:, 0], want, e, np.float32)
        next(run)
        raw = self.qkv.numpy()
        self.project(y, self.w[0], raw)
        next(run)
        heads = raw.reshape(self.n * self.tokens, -1, self.d).astype(np.float64)
        pos = self.pos.numpy()
        for got, part, g in ((self.q, heads[:, :self.hq], self.g[0]), (self.k, heads[:, self.hq:self.hq + self.hk], self.g[1])):
            want, size = R.turn64(R.norm64(part, g.astype(np.float64), eps), pos, (self.d,), 10000.0, False)
            assert np.all(np.abs(got.numpy().reshape(want.shape) - want) <= 5e-7 * size)
        next(run)
        self.held.write(self.table, [self.k.numpy(), self.v.numpy()], self.at, self.new)
        K.same_state(self.cache, self.held, K.mask_of(self.held, self.table, self.at + self.new))
        before = self.mixed.numpy()
        next(run)
        q, mixed = self.q.numpy(), self.mixed.numpy().reshape(self.n, self.tokens, self.hq, self.d)
        want, tol = K.attention64(q, self.held, self.table, 1 / np.sqrt(self.d), True, self.window, self.sinks, self.new,
                                  self.at + self.new)
        there = ~np.isnan(want)
        assert np.all(np.abs(mixed - want)[there] <= tol[there])
        assert np.array_equal(mixed[~there], before.reshape(mixed.shape)[~there])  # behind the new tokens: as they were
        next(run)
        h = self.branch.numpy()
        self.project(mixed, self.w[1], h)
        next(run)
        s, es, want, e = G.reference(x, h[:, 0], ("rms", self.g[2], None, eps), self.vectors(2)[0], 1.0, layer, *self.vectors(3, 4))
        G.near(self.out.numpy()[:, 0], s, es, np.float32)
        G.near(self.y.numpy()[:, 0], want, e, np.float32)
        assert next(run, "end") == "end"


SHAPES = [dict(n=3, c=160, hq=4, hk=2, d=40, block=16, window=0, sinks=0, blocks=12),
          dict(n=2, c=256, hq=8, hk=1, d=64, block=64, window=50, sinks=5, blocks=4),
          dict(n=4, c=320, hq=4, hk=4, d=80, block=32, window=33, sinks=0, blocks=6)]


@pytest.mark.parametrize("shape", SHAPES)
def test_prompt_then_tokens(ctx, shape):
    r = np.random.default_rng(4)
    n, c = shape["n"], shape["c"]
    prompt, one = Stream(ctx, tokens=70, seed=1, **shape), Stream(ctx, tokens=1, seed=1, **shape)
    for a in ("cache", "held", "dtable", "table"):
        setattr(one, a, getattr(prompt, a))
    new = r.integers(30, 71, n)
    new[0] = 70
    prompt.feed(r.standard_normal((n, 70, c)).astype(np.float32), np.zeros(n, int), new)
    prompt.checked()
    at = new.copy()
    for step in range(40):
        here = np.ones(n, int) if step != 5 else (np.arange(n) != 1).astype(int)  # once a request has none
        one.feed(r.standard_normal((n, 1, c)).astype(np.float32), at, here)
        one.checked()
        at += here
    prompt.feed(r.standard_normal((n, 70, c)).astype(np.float32), at, np.full(n, 20))  # and a turn of several
    prompt.checked()


def test_two_graphs_token_after_token(ctx):
    """Each graph holds the whole block of its own stream; lengths and positions move between replays."""
    r = np.random.default_rng(5)
    shape = dict(n=2, c=128, hq=4, hk=2, d=64, block=32, window=600, sinks=8, blocks=40)
    streams = [[Stream(ctx, tokens=1, seed=s, **shape) for _ in range(2)] for s in (1, 2)]  # eager and captured
    for pair in streams:
        x = r.standard_normal((2, 700, 2, 64)).astype(np.float32)
        for s in pair:
            cache_write(s.cache, s.dtable, *(Heads(s.dev(x), 2, 700, 2, 64) for _ in range(2)))
    graphs = []
    for _, s in streams:
        s.feed(np.zeros((2, 1, 128), np.float32), [700, 700], [1, 1])
        s.run(s.scratch)
        graphs.append(capture(ctx, lambda s=s: s.run(s.scratch)))
    for step in range(70):
        for eager, s in streams:
            x = r.standard_normal((2, 1, 128)).astype(np.float32)
            for one in (eager, s):
                one.feed(x, [700 + step, 650 + step], [1, 1])
        for launch, _ in graphs:
            launch()
        for eager, s in streams:
            eager.run()
            assert np.array_equal(eager.y.numpy(), s.y.numpy()) and np.array_equal(eager.out.numpy(), s.out.numpy())
    for _, destroy in graphs:
        destroy()


def test_python_refusals(ctx):
    other = E.Context(0)
    cache = Cache8(ctx, 4, 2, 32, 16)
    t = E.DeviceArray.from_numpy(ctx, np.zeros((2, 2), np.int32))
    h = lambda n=2, tokens=3, heads=2, d=32, c=ctx, dtype=np.float32: Heads(  # noqa: E731
        E.DeviceArray(c, (n, tokens, heads, d), dtype), n, tokens, heads, d)
    bad = [lambda: cache_write(cache, t, h(), h(tokens=2)), lambda: cache_write(cache, t, h(heads=1), h(heads=1)),
           lambda: cache_write(cache, t, h(n=3), h(n=3)), lambda: cache_write(cache, t, h(d=16), h(d=16)),
           lambda: cache_write(cache, t, h(), h(dtype=np.float16)), lambda: cache_write(cache, t, h(c=other), h(c=other)),
           lambda: cache_write(cache, E.DeviceArray(other, (2, 2), np.int32), h(), h()),
           lambda: cache_write(cache, E.DeviceArray(ctx, (2, 2)), h(), h()),
           lambda: cache_write(cache, t, h(), h(), first=E.DeviceArray(ctx, (3,), np.int32)),
           lambda: cache_read(cache, t, h(), h(), length=E.DeviceArray(ctx, (2,), np.float32)),
           lambda: cache_attention(h(heads=3), cache, t, h(heads=3)), lambda: cache_attention(h(), cache, t, h(tokens=2)),
           lambda: cache_attention(h(d=16), cache, t, h(d=16)), lambda: cache_attention(h(), cache, t, h(), sinks=3),
           lambda: cache_attention(h(), cache, t, h(), window=-1), lambda: cache_attention(h(), cache, t, h(), window=1 << 40),
           lambda: cache_attention(h(), cache, t, h(), scale=0.0), lambda: Cache8(ctx, 4, 2, 300), lambda: Cache8(ctx, 0, 2, 32),
           lambda: Norm("batch"), lambda: gated_norm(h(), y=h(tokens=2)), lambda: gated_norm(h(), y=h(c=other)),
           lambda: gated_norm(h(), branch=h(), y=h(dtype=np.float16)), lambda: gated_norm(h(), x_out=h(dtype=np.float16)),
           lambda: gated_norm(h(), y=h(), scale=h()), lambda: gated_norm(h(), y=h(), scale=h(tokens=1, dtype=np.float16)),
           lambda: gated_norm(h(), y=h(), pre=Norm("rms", E.DeviceArray(ctx, (8,)))), lambda: gated_norm(h()),
           lambda: gated_norm(h(), y=h(), gate=h(tokens=1)), lambda: gated_norm(h(), x_out=h(), pre=Norm("rms"))]
    for call in bad:
        with pytest.raises(MoebiusError):
            call()
    other.close()


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_nothing_to_do(ctx, dtype):
    """No items, no tokens, tables without blocks: calls that leave everything as it was."""
    cache = Cache8(ctx, 4, 2, 32, 16)
    K.blank(cache)
    for n, tokens, blocks in ((0, 3, 2), (2, 0, 2), (2, 3, 0)):
        t = E.DeviceArray.from_numpy(ctx, np.zeros((n, blocks), np.int32))
        k, v, q = (Heads(E.DeviceArray.from_numpy(ctx, np.full((n, tokens, 2, 32), 7, dtype)), n, tokens, 2, 32) for _ in range(3))
        cache_write(cache, t, k, v)
        cache_read(cache, t, k, v)
        assert np.all(k.numpy() == 7) and np.all(cache.k.numpy() == 128) and np.all(cache.k_scale.numpy() == 0)
        out = Heads(E.DeviceArray.from_numpy(ctx, np.full((n, tokens, 2, 32), 7, dtype)), n, tokens, 2, 32)
        cache_attention(q, cache, t, out)
        assert np.all(out.numpy() == 0)  # rows that see no token
        gated_norm(Heads(q.buf, n, tokens, 1, 64), pre=Norm("layer"), y=Heads(q.buf, n, tokens, 1, 64))
