"""Gated residuals and modulated norms against their definition in f64.

Tolerances, u = 2^-24, worst cases of the roundings: s = keep x + gate n is off by
2 u (|keep x| + |gate n|) + |gate| e with e the error of n. A norm's n = (v - mean) inv gamma + beta
has v - mean off by a few u of max |v| (the mean's sum of c values in a tree of depth log2 c + 16 in
the lane: (log2 c + 20) u mean |v|), and inv by (log2 c + 24) u; an error e of v goes into n as up to
2 e inv (its own, and its share in the sums; more only where all of the row is off one way).
Outputs are rounded once.
"""
from __future__ import annotations

import numpy as np
import pytest

from moebius_cpu_amd import engine as E
from moebius_cpu_amd.attention import Heads
from moebius_cpu_amd.gated_norm import Norm, gated_norm
from tests.graph_capture import capture
from tests.test_gpu_block_attention import dev, heads

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {np.dtype(np.float32): (U, 0), np.dtype(np.float16): (2.0 ** -11, 2.0 ** -25)}


@pytest.fixture(scope="module")
def ctx():
    return E.Context(0)


def norm64(v, e, kind, gamma, beta, eps):
    """The norm and its error from values v that are off by e."""
    if kind == "none":
        return v, e
    c = v.shape[-1]
    depth = np.log2(c) + 24
    if kind == "layer":
        mean = v.mean(-1, keepdims=True)
        e = e + e.mean(-1, keepdims=True) + depth * U * np.abs(v).mean(-1, keepdims=True) + U * np.abs(v - mean)
        v = v - mean
    ms = (v * v).mean(-1, keepdims=True)
    inv = 1 / np.sqrt(ms + eps)
    # the root mean square is off by at most the errors' own root mean square
    rel = depth * U + np.sqrt((e * e).mean(-1, keepdims=True)) * inv
    y = v * inv
    err = e * inv + np.abs(y) * rel + 2 * U * np.abs(y)
    if gamma is not None:
        y, err = y * gamma, err * np.abs(gamma)
    if beta is not None:
        y = y + beta
    return y, err + 2 * U * np.abs(y)


def reference(x, h, post, gate, keep, pre, scale, shift):
    s, e = x.astype(np.float64), np.zeros(x.shape)
    if h is not None:
        n, en = norm64(h.astype(np.float64), e, *post)
        g = 1.0 if gate is None else gate.astype(np.float64)[:, None]
        e = 3 * U * (np.abs(keep * s) + np.abs(g * n)) + np.abs(g) * en
        s = np.float64(np.float32(keep)) * s + g * n
    y, ey = norm64(s, e, *pre)
    if scale is not None:
        m = 1 + scale.astype(np.float64)[:, None]
        y, ey = y * m, ey * np.abs(m) + 3 * U * np.abs(y * m)
    if shift is not None:
        y = y + shift.astype(np.float64)[:, None]
        ey = ey + 2 * U * np.abs(y)
    return s, e, y, ey


def near(got, want, e, dtype):
    step, least = HALF[np.dtype(dtype)]
    assert np.all(np.abs(got.astype(np.float64) - want) <= e + step * (np.abs(want) + e) + least)


class Case:
    def __init__(self, ctx, n, rows, c, xt=np.float32, ht=np.float32, post="none", pre="layer", affine=False, mod=True,
                 branch=True, pad=0, offset=0, mean=0.3, keep=0.75, seed=0):
        r = np.random.default_rng(seed + c)
        self.ctx, self.n, self.rows, self.c, self.xt, self.ht = ctx, n, rows, c, xt, ht
        self.x = (1.5 * r.standard_normal((n, rows, 1, c)) + mean).astype(xt)
        self.h = (0.7 * r.standard_normal((n, rows, 1, c)) - mean).astype(ht) if branch else None
        eps = 1e-6
        vec = lambda: (1 + 0.2 * r.standard_normal(c)).astype(np.float32) if affine else None  # noqa: E731
        self.v = [vec() for _ in range(4)]
        self.mods = [(0.4 * r.standard_normal((n, c))).astype(np.float32) if mod else None for _ in range(3)]
        if not branch:
            self.mods[0], post = None, "none"
        dv = [None if a is None else dev(ctx, a) for a in self.v]
        self.post, self.pre = (post, *(self.v[:2] if post != "none" else (None, None)), np.float64(np.float32(eps))), \
            (pre, *(self.v[2:] if pre != "none" else (None, None)), np.float64(np.float32(eps)))
        rows_of = lambda a: heads(ctx, a, pad, offset)  # noqa: E731
        wide = None
        if mod:  # one projection's three vectors
            wide = dev(ctx, np.concatenate([np.zeros((n, c), np.float32) if m is None else m for m in self.mods], 1))
        views = [None if m is None else Heads(wide, n, 1, 1, c, ld=3 * c, offset=i * c) for i, m in enumerate(self.mods)]
        self.dx, self.dh = rows_of(self.x), None if self.h is None else rows_of(self.h)
        self.xo, self.y = rows_of(np.zeros_like(self.x)), rows_of(np.zeros((n, rows, 1, c), ht))
        self.kw = dict(branch=self.dh, post=Norm(post, dv[0], dv[1], eps) if post != "none" else None, gate=views[0],
                       keep=keep, pre=Norm(pre, dv[2], dv[3], eps) if pre != "none" else None, scale=views[1], shift=views[2])

    def check(self, xo, y):
        h = None if self.h is None else self.h[:, :, 0]
        s, e, want, ey = reference(self.x[:, :, 0], h, self.post, self.mods[0], self.kw["keep"], self.pre, *self.mods[1:])
        if xo is not None:
            near(xo.numpy()[:, :, 0], s, e, self.xt)
        if y is not None:
            near(y.numpy()[:, :, 0], want, ey, self.ht)


F, H = np.float32, np.float16


@pytest.mark.parametrize("xt,ht", [(F, F), (F, H), (H, H), (H, F)])
@pytest.mark.parametrize("post,pre", [("none", "layer"), ("rms", "rms"), ("layer", "none"), ("layer", "layer"), ("none", "rms")])
@pytest.mark.parametrize("n,rows,c", [(1, 1, 1), (3, 5, 40), (2, 3, 1280), (1, 7, 333)])
def test_kinds_and_types(ctx, xt, ht, post, pre, n, rows, c):
    k = Case(ctx, n, rows, c, xt, ht, post, pre, affine=c % 3 == 0)
    gated_norm(k.dx, x_out=k.xo, y=k.y, **k.kw)
    k.check(k.xo, k.y)


@pytest.mark.parametrize("c", [2, 64, 255, 256, 257, 512, 516, 768, 1023, 1028, 1284, 2048, 2052, 4096, 4100, 8192, 8196,
                               8193, 32768])
@pytest.mark.parametrize("ht", [F, H])
def test_widths(ctx, c, ht):
    k = Case(ctx, 2, 9, c, F, ht, "rms", "layer", affine=True)
    gated_norm(k.dx, x_out=k.xo, y=k.y, **k.kw)
    k.check(k.xo, k.y)


@pytest.mark.parametrize("pad,offset", [(4, 4), (1, 3), (8, 0)])
@pytest.mark.parametrize("xt,ht", [(F, H), (H, H)])
def test_strides(ctx, pad, offset, xt, ht):
    k = Case(ctx, 3, 4, 100, xt, ht, "layer", "rms", pad=pad, offset=offset)
    gated_norm(k.dx, x_out=k.xo, y=k.y, **k.kw)
    k.check(k.xo, k.y)
    for o in (k.xo, k.y):
        gaps = o.buf.numpy()[offset:].reshape(-1)[:(k.n * k.rows - 1) * o.ld].reshape(-1, o.ld)[:, 100:]
        assert np.isnan(gaps).all()


@pytest.mark.parametrize("mod", [False, True])
@pytest.mark.parametrize("branch", [False, True])
def test_parts_alone(ctx, mod, branch):
    """Only the sum, only the norm, and in place."""
    k = Case(ctx, 2, 6, 320, F, F, "rms" if branch else "none", "layer", mod=mod, branch=branch)
    gated_norm(k.dx, y=k.y, **k.kw)
    k.check(None, k.y)
    only = {**k.kw, "pre": None, "scale": None, "shift": None}
    gated_norm(k.dx, x_out=k.xo, **only)
    k.check(k.xo, None)
    gated_norm(k.dx, x_out=k.dx, **k.kw, y=k.dh if branch else k.y)
    k.check(k.dx, k.dh if branch else k.y)


def test_a_large_mean_costs_no_bits(ctx):
    k = Case(ctx, 1, 4, 640, F, F, "none", "layer", mod=False, branch=False, mean=3000.0)
    gated_norm(k.dx, y=k.y, **k.kw)
    k.check(None, k.y)


def test_constant_and_non_finite_rows(ctx):
    k = Case(ctx, 1, 4, 256, F, F, "none", "layer", mod=False, branch=False)
    k.x[0, 0] = 4.0
    k.x[0, 1, 0, 7] = np.nan
    k.x[0, 2, 0, 7] = np.inf
    k.dx.buf.upload(k.x)
    gated_norm(k.dx, y=k.y, **k.kw)
    got = k.y.numpy()[0, :, 0]
    assert np.all(got[0] == 0) and np.isnan(got[1]).all() and np.isnan(got[2]).all()
    assert abs(got[3].std() - 1) < 1e-5


def test_captured_and_replayed(ctx):
    cases = [Case(ctx, 2, 50, c, F, H, "rms", "layer", seed=c) for c in (1280, 5000)]
    wants = []
    for k in cases:
        gated_norm(k.dx, x_out=k.xo, y=k.y, **k.kw)
        wants.append((k.xo.numpy(), k.y.numpy()))
    graphs = [capture(ctx, lambda k=k: gated_norm(k.dx, x_out=k.xo, y=k.y, **k.kw)) for k in cases]
    for _ in range(3):
        for k in cases:
            k.xo.buf.upload(np.zeros_like(k.x).reshape(k.xo.buf.shape))
        for launch, _ in graphs:
            launch()
        ctx.synchronize()
        for k, (xo, y) in zip(cases, wants):
            assert np.array_equal(k.xo.numpy(), xo) and np.array_equal(k.y.numpy(), y)
        gated_norm(cases[0].dx, x_out=cases[0].xo, y=cases[0].y, **cases[0].kw)
        assert np.array_equal(cases[0].y.numpy(), wants[0][1])
    for _, destroy in graphs:
        destroy()
