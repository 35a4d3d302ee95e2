"""Rotary positions with several axes, alone and behind the norms of query and
key heads, against the formulas in f64.

Tolerances: the kernel's sine and cosine are off by at most 1.5e-7 (the remainder
of the angle rounded to f32, 2.3e-8 rad, the series and its roundings), a turned
value by two f32 roundings more: 3e-7 (|x0| + |x1|). The norm adds three relative
roundings of 2^-24 for f32 rows (the scale, its product, gamma's: 1.8e-7) and for
f16 rows the f32 sum of squares of up to 22 roundings, halved by the root, and four
more (16 x 2^-24 = 1e-6). f16 outputs add half a step: |y| 2^-11, at least 2^-25."""
from __future__ import annotations

import numpy as np
import pytest

from moebius_cpu_amd import engine as E
from moebius_cpu_amd._lib import MoebiusError
from moebius_cpu_amd.attention import Heads, RopeAxes, qk_norm_rope, rope_axes

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return E.Context(0)


def turn64(x, pos, dims, theta, halves, inverse=False, freq=None):
    """x [rows][heads][d] in f64 turned, and |x0| + |x1| for every channel of a pair."""
    rows, _, d = x.shape
    if freq is None:
        freq = np.concatenate([theta ** (-np.arange(0, m, 2) / m) for m in dims])
    axis = np.repeat(np.arange(len(dims)), np.array(dims) // 2)
    a = pos.astype(np.float64)[np.arange(rows) % len(pos)][:, axis] * freq * (-1 if inverse else 1)
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    n = sum(dims) // 2
    i0, i1 = (np.arange(n), n + np.arange(n)) if halves else (2 * np.arange(n), 2 * np.arange(n) + 1)
    y, size = x.copy(), np.abs(x)
    y[..., i0] = x[..., i0] * c - x[..., i1] * s
    y[..., i1] = x[..., i0] * s + x[..., i1] * c
    size[..., i0] = size[..., i1] = np.abs(x[..., i0]) + np.abs(x[..., i1])
    return y, size


def half_step(y, dtype):
    return np.abs(y) * 2.0 ** -11 + 2.0 ** -25 if dtype == np.float16 else 0.0


def strided(ctx, x, ld, offset):
    """x [rows][heads][d] with rows ld apart from element `offset` on, NaN in between."""
    rows, heads, d = x.shape
    flat = np.full(offset + rows * ld, np.nan, x.dtype)
    for r in range(rows):
        flat[offset + r * ld: offset + r * ld + heads * d] = x[r].ravel()
    return Heads(E.DeviceArray.from_numpy(ctx, flat), 1, rows, heads, d, ld=ld, offset=offset)


CASES = [  # rows, pos_rows, heads, d, dims, extra ld, offset
    (1, 1, 1, 2, (2,), 0, 0), (7, 7, 3, 40, (20, 20), 0, 0), (64, 32, 8, 40, (20, 20), 0, 0),
    (130, 65, 5, 64, (16, 24, 24), 0, 0), (9, 3, 2, 72, (36, 36), 0, 0), (33, 33, 2, 80, (40, 40), 80, 160),
    (17, 17, 16, 128, (32, 48, 48), 128, 64), (5, 5, 2, 128, (8, 8, 8, 8), 0, 0), (6, 6, 3, 160, (64, 32), 0, 0),
    (4, 2, 2, 256, (128, 64, 64), 0, 0), (11, 11, 2, 38, (18, 20), 1, 1), (3, 3, 1, 7, (4, 2), 0, 3),
    (257, 257, 33, 96, (32, 32, 32), 0, 0), (2, 2, 2, 514, (256, 256), 0, 0), (3, 3, 2, 256, (4, 4), 0, 0),
]


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("pairing", ["interleaved", "halves"])
@pytest.mark.parametrize("case", CASES)
def test_rope_against_the_formula(ctx, case, pairing, dtype):
    rows, pos_rows, heads, d, dims, pad, offset = case
    r = np.random.default_rng(rows * 1000 + d)
    x = r.standard_normal((rows, heads, d)).astype(dtype)
    pos = r.integers(-50, 100_000, (pos_rows, len(dims))).astype(np.int32)
    rope = RopeAxes(ctx, dims, theta=10000.0, pairing=pairing)
    xh = strided(ctx, x, heads * d + pad, offset)
    out = Heads(E.DeviceArray.from_numpy(ctx, np.full((rows, heads, d), np.nan, dtype)), 1, rows, heads, d)
    p = E.DeviceArray.from_numpy(ctx, pos)
    for inverse in (False, True):
        rope_axes(xh, p, rope, out, inverse=inverse)
        want, size = turn64(x.astype(np.float64), pos, dims, 10000.0, pairing == "halves", inverse)
        got = out.numpy()[0].astype(np.float64)
        assert np.all(np.abs(got - want) <= 3e-7 * size + half_step(want, dtype)), np.abs(got - want).max()
        rest = slice(sum(dims), d)
        assert np.array_equal(out.numpy()[0][..., rest], x[..., rest])  # channels behind the pairs pass through


@pytest.mark.parametrize("pairing", ["interleaved", "halves"])
@pytest.mark.parametrize("d,dims", [(64, (32, 32)), (13, (6, 4))])
def test_rope_in_place_and_back(ctx, pairing, d, dims):
    """In place gives the bits of the call out of place; the inverse undoes it."""
    r = np.random.default_rng(5)
    x = r.standard_normal((20, 4, d)).astype(np.float32)
    p = E.DeviceArray.from_numpy(ctx, r.integers(0, 1000, (20, 2)).astype(np.int32))
    rope = RopeAxes(ctx, dims, pairing=pairing)
    a = Heads(E.DeviceArray.from_numpy(ctx, x), 1, 20, 4, d)
    b = Heads(E.DeviceArray(ctx, x.shape), 1, 20, 4, d)
    rope_axes(a, p, rope, b)
    rope_axes(a, p, rope, a)
    assert np.array_equal(a.numpy(), b.numpy())
    rope_axes(a, p, rope, a, inverse=True)
    n = sum(dims)
    assert np.abs(a.numpy()[0] - x)[..., :n].max() <= 2 * 3e-7 * 2 * np.abs(x).max() * 2 ** 0.5
    assert np.array_equal(a.numpy()[0][..., n:], x[..., n:])


def test_rope_far_positions(ctx):
    """Positions to the ends of int32: f64 turns are off by less than 1e-6 rad on either side."""
    dims, pos = (64,), np.array([[2**31 - 1], [-2**31], [2**31 - 2], [123456789], [0]], np.int32)
    x = np.random.default_rng(1).standard_normal((5, 2, 64)).astype(np.float32)
    out = Heads(E.DeviceArray(ctx, x.shape), 1, 5, 2, 64)
    rope_axes(Heads(E.DeviceArray.from_numpy(ctx, x), 1, 5, 2, 64), E.DeviceArray.from_numpy(ctx, pos),
              RopeAxes(ctx, dims), out)
    want, size = turn64(x.astype(np.float64), pos, dims, 10000.0, False)
    assert np.all(np.abs(out.numpy()[0] - want) <= (3e-7 + 2e-6) * size)
    assert np.array_equal(out.numpy()[0][4], x[4])  # position 0: unchanged


def test_rope_quarter_turns_are_exact(ctx):
    """With a frequency of a quarter turn the sines are 0, 1, 0, -1 but for the rounding of pi / 2 in f64."""
    x = np.random.default_rng(2).standard_normal((8, 1, 2)).astype(np.float32)
    pos = np.arange(-4, 4, dtype=np.int32)[:, None]
    out = Heads(E.DeviceArray(ctx, x.shape), 1, 8, 1, 2)
    rope_axes(Heads(E.DeviceArray.from_numpy(ctx, x), 1, 8, 1, 2), E.DeviceArray.from_numpy(ctx, pos),
              RopeAxes(ctx, (2,), freq=[np.pi / 2]), out)
    z = (x[:, 0, 0] + 1j * x[:, 0, 1]) * np.array([1, 1j, -1, -1j] * 2)
    got = out.numpy()[0][:, 0]
    assert np.abs(got[:, 0] - z.real).max() <= 1e-14 and np.abs(got[:, 1] - z.imag).max() <= 1e-14


def test_rope_does_not_write_between_rows(ctx):
    x = np.random.default_rng(3).standard_normal((6, 2, 40)).astype(np.float32)
    out = strided(ctx, np.zeros_like(x), 100, 4)
    p = E.DeviceArray.from_numpy(ctx, np.zeros((6, 2), np.int32))
    rope_axes(Heads(E.DeviceArray.from_numpy(ctx, x), 1, 6, 2, 40), p, RopeAxes(ctx, (20, 20)), out)
    flat = out.buf.numpy()
    for r in range(6):
        assert np.array_equal(flat[4 + r * 100: 84 + r * 100], x[r].ravel())
        assert np.isnan(flat[84 + r * 100: 104 + r * 100]).all()
    assert np.isnan(flat[:4]).all()


def norm64(x, gamma, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gamma


QK = [  # rows, pos_rows, hq, hk, d, dims
    (1, 1, 1, 1, 8, (4, 4)), (8, 8, 32, 8, 128, (32, 48, 48)), (50, 25, 8, 8, 160, (80, 80)), (13, 13, 6, 2, 72, (36, 36)),
    (100, 100, 3, 1, 80, (40, 40)), (5, 5, 4, 2, 256, (64, 64, 64, 64)), (9, 9, 2, 1, 30, (14, 10)), (300, 300, 16, 4, 64, (64,)),
    (4, 4, 2, 2, 96, (32, 16)), (3, 3, 5, 5, 33, (16, 16)),
]


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("pairing", ["interleaved", "halves"])
@pytest.mark.parametrize("case", QK)
@pytest.mark.parametrize("inplace", [False, True])
def test_qk_norm_rope_against_the_formula(ctx, case, pairing, dtype, inplace):
    """Queries and keys as columns of one projection, turned where they lie or into arrays of their own."""
    rows, pos_rows, hq, hk, d, dims = case
    r = np.random.default_rng(rows + d)
    qkv = (r.standard_normal((rows, hq + 2 * hk, d)) * 2 + 0.2).astype(dtype)
    pos = r.integers(0, 5000, (pos_rows, len(dims))).astype(np.int32)
    gq, gk = (1 + 0.2 * r.standard_normal(d)).astype(np.float32), (1 + 0.2 * r.standard_normal(d)).astype(np.float32)
    buf, ld = E.DeviceArray.from_numpy(ctx, qkv), (hq + 2 * hk) * d
    q, k = Heads(buf, 1, rows, hq, d, ld=ld), Heads(buf, 1, rows, hk, d, ld=ld, offset=hq * d)
    if inplace:
        qo, ko = q, k
    else:
        qo = Heads(E.DeviceArray(ctx, (rows, hq, d), dtype), 1, rows, hq, d)
        ko = Heads(E.DeviceArray(ctx, (rows, hk, d), dtype), 1, rows, hk, d)
    qk_norm_rope(q, k, E.DeviceArray.from_numpy(ctx, gq), E.DeviceArray.from_numpy(ctx, gk), 1e-6,
                 E.DeviceArray.from_numpy(ctx, pos), RopeAxes(ctx, dims, pairing=pairing), qo, ko)
    e = 5e-7 if dtype == np.float32 else 3e-7 + 1e-6
    for got, x, g in ((qo, qkv[:, :hq], gq), (ko, qkv[:, hq:hq + hk], gk)):
        want, size = turn64(norm64(x.astype(np.float64), g.astype(np.float64), np.float64(np.float32(1e-6))), pos, dims,
                            10000.0, pairing == "halves")
        err = np.abs(got.numpy()[0].astype(np.float64) - want)
        assert np.all(err <= e * size + half_step(want, dtype)), (err / size).max()
    assert np.array_equal(buf.numpy()[:, hq + hk:], qkv[:, hq + hk:])  # the values are not touched
    if not inplace:
        assert np.array_equal(buf.numpy(), qkv)


def test_qk_norm_without_gamma_and_extreme_rows(ctx):
    """Zero rows stay zero, rows of the type's largest and smallest values are normed in range (their
    squares leave f32), NaN and infinity stay in their own head."""
    d = 64
    x = np.zeros((6, 2, d), np.float32)
    x[1] = 3e38
    x[2] = 1e-38
    x[3, 0, 5] = np.nan
    x[3, 1] = 1.0
    x[4, 0, 0] = np.inf
    x[4, 1] = 2.0
    x[5] = -1e30
    out = [Heads(E.DeviceArray(ctx, x.shape), 1, 6, 2, d) for _ in range(2)]
    h = Heads(E.DeviceArray.from_numpy(ctx, x), 1, 6, 2, d)
    qk_norm_rope(h, h, None, None, 0.0, E.DeviceArray.from_numpy(ctx, np.zeros((1, 1), np.int32)), RopeAxes(ctx, (d,)),
                 out[0], out[1])
    for o in out:
        y = o.numpy()[0]
        assert np.isnan(y[0]).all()  # 0 / 0 without eps
        for r, v in ((1, 1.0), (2, 1.0), (5, -1.0)):
            assert np.abs(y[r] - v).max() <= 3e-7
        assert np.isnan(y[3, 0]).all() and np.abs(y[3, 1] - 1).max() <= 3e-7
        assert np.isnan(y[4, 0, :2]).any() and np.abs(y[4, 1] - 1).max() <= 3e-7
    qk_norm_rope(h, h, None, None, 1e-6, E.DeviceArray.from_numpy(ctx, np.zeros((1, 1), np.int32)), RopeAxes(ctx, (d,)),
                 out[0], out[1])
    assert not out[0].numpy()[0][0].any()


def test_no_rows(ctx):
    h = Heads(E.DeviceArray(ctx, (0, 2, 8)), 0, 5, 2, 8)
    p = E.DeviceArray.from_numpy(ctx, np.zeros((1, 1), np.int32))
    rope_axes(h, p, RopeAxes(ctx, (8,)), h)
    qk_norm_rope(h, h, None, None, 1e-6, p, RopeAxes(ctx, (8,)), h, h)
    ctx.synchronize()


def test_python_refusals(ctx):
    h = Heads(E.DeviceArray(ctx, (4, 2, 8)), 1, 4, 2, 8)
    p = E.DeviceArray.from_numpy(ctx, np.zeros((4, 1), np.int32))
    with pytest.raises(MoebiusError, match="exceed their buffer"):
        Heads(h.buf, 1, 5, 2, 8)
    with pytest.raises(MoebiusError, match="exceed their buffer"):
        Heads(h.buf, 1, 4, 2, 8, offset=1)
    with pytest.raises(MoebiusError, match="ld below"):
        Heads(h.buf, 1, 4, 2, 8, ld=15)
    with pytest.raises(MoebiusError, match="f32 or f16"):
        Heads(p, 1, 4, 1, 1)
    with pytest.raises(MoebiusError, match="int32"):
        rope_axes(h, E.DeviceArray(ctx, (4, 1)), RopeAxes(ctx, (8,)), h)
    with pytest.raises(MoebiusError, match="int32"):
        rope_axes(h, p, RopeAxes(ctx, (4, 4)), h)
    with pytest.raises(MoebiusError, match="differ in type"):
        rope_axes(h, p, RopeAxes(ctx, (8,)), Heads(E.DeviceArray(ctx, (4, 2, 8), "f2"), 1, 4, 2, 8))
    with pytest.raises(MoebiusError, match="gamma"):
        qk_norm_rope(h, h, E.DeviceArray(ctx, (4,)), None, 1e-6, p, RopeAxes(ctx, (8,)), h, h)
    with pytest.raises(MoebiusError, match="frequencies"):
        RopeAxes(ctx, (8,), freq=[1.0])
    with pytest.raises(MoebiusError, match="pairing"):
        RopeAxes(ctx, (8,), pairing="spiral")
