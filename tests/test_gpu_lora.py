"""Low-rank adapters beside a shared projection, against f64.

Tolerance: the projection's own (1e-5 of the sum of its terms' sizes in EXACT, as the
f32 parity tests take; f16 operand roundings 2^-10 of them in FAST), and for the
adapter (c_in + rank + 8) roundings of 2^-24 of scale sum |b| sum |a x|, worst case."""
from __future__ import annotations

import numpy as np
import pytest

from moebius_cpu_amd import engine as E
from moebius_cpu_amd._lib import MoebiusError
from moebius_cpu_amd.adapters import Adapters
from tests.graph_capture import capture

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    return E.Context(0)


def reference(x, w, bias, res, a, b, scale, slot, per):
    """y and its tolerances' scale: the projection's and the adapter's sums of sizes."""
    x, w, a, b = (t.astype(np.float64) for t in (x, w, a, b))
    y, base = x @ w.T, np.abs(x) @ np.abs(w).T
    if bias is not None:
        y, base = y + bias, base + np.abs(bias)
    if res is not None:
        y, base = y + res, base + np.abs(res)
    low = np.zeros_like(y)
    for r in range(len(x)):
        s = slot[r // per]
        if 0 <= s < len(scale):
            y[r] += float(scale[s]) * (b[s] @ (a[s] @ x[r]))
            low[r] = abs(float(scale[s])) * (np.abs(b[s]) @ (np.abs(a[s]) @ np.abs(x[r])))
    return y, base, low


CASES = [  # n, h, w, ci, co, rank, slots, per pixel
    (1, 1, 1, 64, 64, 8, 1, False), (16, 1, 1, 320, 320, 16, 32, False), (3, 5, 7, 100, 52, 4, 5, False),
    (1, 1, 40, 1280, 256, 32, 4, True), (2, 16, 16, 320, 640, 64, 2, False), (1, 9, 9, 33, 45, 3, 7, True),
    (5, 1, 1, 2500, 70, 10, 3, False), (1, 20, 20, 64, 128, 256, 2, True), (1, 3, 11, 16, 4, 100, 3, True),
    (17, 1, 3, 640, 1100, 7, 40, False),
    # enough rows and columns for the product of operands in two f16 parts
    (4, 32, 32, 320, 640, 16, 3, False), (3, 23, 29, 333, 1030, 12, 4, False), (1, 50, 43, 100, 1281, 40, 9, True),
    (5, 20, 21, 64, 1280, 72, 2, False), (2, 20, 25, 1400, 1300, 24, 3, False),
    # its tiles, and the groups of waves that share the long axis
    (1, 27, 30, 1100, 320, 12, 3, True), (2, 19, 23, 2600, 330, 40, 3, False), (1, 27, 30, 333, 321, 33, 5, True),
    (1, 64, 65, 72, 1100, 20, 4, True), (1, 4100, 1, 33, 1030, 16, 2, True), (1, 20, 20, 40, 600, 256, 2, True),
    (1, 75, 74, 72, 1100, 20, 4, True), (1, 5600, 1, 33, 1030, 16, 2, True),
    # rows and ranks shorter than a load
    (1, 1, 3, 1, 5, 1, 2, True), (2, 3, 3, 3, 7, 2, 2, False), (1, 40, 40, 3, 700, 2, 3, True), (1, 90, 80, 5, 97, 3, 4, True),
    (2, 50, 50, 1, 130, 1, 2, False),
]


def make(ctx, case, f16, seed=0):
    n, h, w, ci, co, rank, slots, pixel = case
    r = np.random.default_rng(seed + ci)
    store = np.float16 if f16 else np.float32
    d = dict(x=r.standard_normal((n, h, w, ci)).astype(np.float32), w=(r.standard_normal((co, ci)) / np.sqrt(ci)).astype(store),
             a=(r.standard_normal((slots, rank, ci)) / np.sqrt(ci)).astype(store), b=(r.standard_normal((slots, co, rank)) * 0.3).astype(store),
             scale=r.uniform(0.3, 2, slots).astype(np.float32), bias=r.standard_normal(co).astype(np.float32),
             res=r.standard_normal((n, h, w, co)).astype(np.float32))
    d["slot"] = r.integers(-1, slots, n * h * w if pixel else n).astype(np.int32)
    return d


def layer(ctx, case, d, f16, bias=True):
    _, _, _, ci, co, rank, _, _ = case
    conv = E.Conv1x1(ctx, ci, co, E.Param(ctx, d["w"], f16=f16), d["bias"] if bias else None)
    return conv, Adapters(ctx, E.Param(ctx, d["a"], f16=f16), E.Param(ctx, d["b"], f16=f16), d["scale"], ci, co, rank)


@pytest.mark.parametrize("fast", [False, True])
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("extra", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_against_the_formula(ctx, case, f16, extra, fast):
    n, h, w, ci, co, rank, slots, pixel = case
    d = make(ctx, case, f16)
    conv, ad = layer(ctx, case, d, f16, extra)
    out = E.Tensor(ctx, n, h, w, co)
    ctx.set_precision(fast)
    try:
        conv.forward_adapted(E.Tensor.from_numpy(ctx, d["x"]), ad, E.DeviceArray.from_numpy(ctx, d["slot"]), out,
                             E.Tensor.from_numpy(ctx, d["res"]) if extra else None)
    finally:
        ctx.set_precision(False)
    y, base, low = reference(d["x"].reshape(-1, ci), d["w"], d["bias"] if extra else None,
                             d["res"].reshape(-1, co) if extra else None, d["a"], d["b"], d["scale"], d["slot"],
                             1 if pixel else h * w)
    err = np.abs(out.numpy().reshape(-1, co) - y)
    bound = (2.0 ** -10 if fast else 1e-5) * base + (ci + rank + 8) * U * low + U * np.abs(y)
    assert np.all(err <= bound), (err / bound).max()


@pytest.mark.parametrize("case", [CASES[1], CASES[3], CASES[5], CASES[12]])
def test_rows_without_adapter_are_the_projection(ctx, case):
    """Slots below 0 and at or above the number of adapters: the projection alone (few rows have a
    product of their own, so within its tolerance, not in bits)."""
    n, h, w, ci, co, _, slots, pixel = case
    d = make(ctx, case, True)
    conv, ad = layer(ctx, case, d, True)
    x, plain, out = E.Tensor.from_numpy(ctx, d["x"]), E.Tensor(ctx), E.Tensor(ctx)
    conv.forward(x, plain)
    slot = np.where(np.arange(d["slot"].size) % 2, d["slot"], np.where(np.arange(d["slot"].size) % 4, slots, -2**31)).astype(np.int32)
    conv.forward_adapted(x, ad, E.DeviceArray.from_numpy(ctx, slot), out)
    rows = np.repeat(slot, 1 if pixel else h * w).reshape(n, h, w)
    none = (rows < 0) | (rows >= slots)
    _, base, _ = reference(d["x"].reshape(-1, ci), d["w"], d["bias"], None, d["a"], d["b"], d["scale"],
                           np.full(d["slot"].size, -1), 1 if pixel else h * w)
    assert none.any()
    assert np.all((np.abs(out.numpy() - plain.numpy()) <= 1e-5 * base.reshape(n, h, w, co))[none])
    assert not np.array_equal(out.numpy(), plain.numpy())


@pytest.mark.parametrize("case", [(1, 1, 16, 64, 64, 8, 3, True), (1, 1, 100, 64, 64, 8, 3, True),
                                  (1, 1, 2100, 96, 1280, 8, 5, True)])
def test_values_that_are_not_finite_stay_with_their_request(ctx, case):
    """An adapter of NaN and infinity, and a row of NaN, among rows of other requests in the same tile."""
    d = make(ctx, case, False)
    rows, slots = case[2], case[6]
    d["slot"][:] = np.arange(rows) % slots
    conv, ad = layer(ctx, case, d, False)
    slot, good, out = E.DeviceArray.from_numpy(ctx, d["slot"]), E.Tensor(ctx), E.Tensor(ctx)
    conv.forward_adapted(E.Tensor.from_numpy(ctx, d["x"]), ad, slot, good)
    d["a"][1, 2], d["b"][1, :, 3] = np.nan, np.inf
    d["x"][0, 0, 5] = np.nan
    conv, ad = layer(ctx, case, d, False)
    conv.forward_adapted(E.Tensor.from_numpy(ctx, d["x"]), ad, slot, out)
    bad = (d["slot"] == 1) | (np.arange(rows) == 5)
    got = out.numpy()[0, 0]
    assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()
    # the projection repairs tiles with such sums on other instructions: equal but for its roundings
    assert np.abs(got - good.numpy()[0, 0])[~bad].max() < 1e-5


@pytest.mark.parametrize("f16", [False, True])
def test_f32_ranges(ctx, f16):
    """Rows, weights and adapters of sizes far from each other and from f16's range keep f32's errors,
    relative to the terms of their own sums."""
    case = (1, 1, 2100, 96, 1280, 8, 3, True)
    d = make(ctx, case, f16)
    d["x"] *= (10.0 ** (np.arange(2100) % 61 - 30)).astype(np.float32)[None, None, :, None]
    d["x"][..., :5] *= np.float32(2.0 ** -15)
    if not f16:
        d["w"] *= (10.0 ** (np.arange(1280) % 7 - 3)).astype(np.float32)[:, None]
        d["a"] *= np.array([1e-12, 1.0, 1e6], np.float32)[:, None, None]
        d["b"] *= np.array([1e5, 1e-5, 1.0], np.float32)[:, None, None]
    conv, ad = layer(ctx, case, d, f16, bias=False)
    out = E.Tensor(ctx)
    conv.forward_adapted(E.Tensor.from_numpy(ctx, d["x"]), ad, E.DeviceArray.from_numpy(ctx, d["slot"]), out)
    y, base, low = reference(d["x"].reshape(-1, 96), d["w"], None, None, d["a"], d["b"], d["scale"], d["slot"], 1)
    err = np.abs(out.numpy().reshape(-1, 1280) - y)
    bound = 1e-5 * base + (96 + 8 + 8) * U * low + U * np.abs(y) + 1e-45
    assert np.all(err <= bound), (err / bound).max()


def test_scratch_and_no_rows(ctx):
    case = (4, 1, 1, 640, 64, 16, 4, False)
    d = make(ctx, case, True)
    conv, ad = layer(ctx, case, d, True)
    x, slot, a, b = E.Tensor.from_numpy(ctx, d["x"]), E.DeviceArray.from_numpy(ctx, d["slot"]), E.Tensor(ctx), E.Tensor(ctx)
    size = ad.scratch(4, conv.weight)
    assert size > 0
    conv.forward_adapted(x, ad, slot, a)
    conv.forward_adapted(x, ad, slot, b, scratch=E.DeviceArray(ctx, (size,), np.uint8))
    assert np.array_equal(a.numpy(), b.numpy())
    with pytest.raises(MoebiusError, match="smaller"):
        conv.forward_adapted(x, ad, slot, b, scratch=E.DeviceArray(ctx, (size - 1,), np.uint8))
    conv.forward_adapted(E.Tensor(ctx, 0, 1, 1, 640), ad, E.DeviceArray(ctx, (0,), "i4"), b)
    assert b.shape == (0, 1, 1, 64)


def test_python_refusals(ctx):
    case = (2, 2, 2, 32, 16, 4, 2, False)
    d = make(ctx, case, False)
    conv, ad = layer(ctx, case, d, False)
    x, out = E.Tensor.from_numpy(ctx, d["x"]), E.Tensor(ctx)
    with pytest.raises(MoebiusError, match="slot is int32"):
        conv.forward_adapted(x, ad, E.DeviceArray(ctx, (3,), "i4"), out)
    with pytest.raises(MoebiusError, match="slot is int32"):
        conv.forward_adapted(x, ad, E.DeviceArray(ctx, (2,)), out)
    with pytest.raises(MoebiusError, match="input channels"):
        conv.forward_adapted(E.Tensor(ctx, 2, 2, 2, 31), ad, E.DeviceArray(ctx, (2,), "i4"), out)
    with pytest.raises(MoebiusError, match="adapter size"):
        Adapters(ctx, ad.a, ad.b, d["scale"], 32, 16, 5)
    with pytest.raises(MoebiusError, match="storage type"):
        Adapters(ctx, ad.a, E.Param(ctx, d["b"], f16=True), d["scale"], 32, 16, 4)
    with pytest.raises(MoebiusError, match="residual shape"):
        conv.forward_adapted(x, ad, E.DeviceArray(ctx, (2,), "i4"), out, E.Tensor(ctx, 1, 2, 2, 16))


@pytest.mark.parametrize("fast", [False, True])
@pytest.mark.parametrize("case", [(4, 1, 1, 640, 64, 16, 4, False), (2, 20, 20, 640, 640, 16, 4, False),
                                  (40, 5, 5, 96, 700, 8, 9, True)])
def test_captured_and_replayed(ctx, case, fast):
    """Two graphs of one projection with scratch of their own, replayed among eager calls in the
    context's workspace; without scratch a captured call is refused."""
    n, h, w, ci, co, rank, slots, pixel = case
    d = make(ctx, case, False)
    conv, ad = layer(ctx, case, d, False)
    slot = E.DeviceArray.from_numpy(ctx, d["slot"])
    xs = [E.Tensor.from_numpy(ctx, d["x"]), E.Tensor.from_numpy(ctx, d["x"][..., ::-1])]
    res = E.Tensor.from_numpy(ctx, d["res"])
    outs, eager = [E.Tensor(ctx, n, h, w, co) for _ in xs], E.Tensor(ctx)
    ctx.set_precision(fast)
    try:
        wants = []
        for x in xs:
            conv.forward_adapted(x, ad, slot, eager, res)
            wants.append(eager.numpy())
        scratch = [E.DeviceArray(ctx, (ad.scratch(n * h * w, conv.weight),), np.uint8) for _ in xs]
        with pytest.raises(MoebiusError, match="captured call needs scratch"):
            capture(ctx, lambda: conv.forward_adapted(xs[0], ad, slot, outs[0], res))
        graphs = [capture(ctx, lambda i=i: conv.forward_adapted(xs[i], ad, slot, outs[i], res, scratch[i])) for i in range(2)]
        for turn in range(4):
            for o in outs:
                o.upload(np.zeros((n, h, w, co), np.float32))
            for launch, _ in graphs:
                launch()
            conv.forward_adapted(xs[turn % 2], ad, slot, eager, res)
            ctx.synchronize()
            for o, want in zip(outs, wants):
                assert np.array_equal(o.numpy(), want)
            assert np.array_equal(eager.numpy(), wants[turn % 2])
        for _, destroy in graphs:
            destroy()
    finally:
        ctx.set_precision(False)


@pytest.mark.parametrize("case", [(3, 1, 5, 64, 64, 8, 3, True), (2, 25, 25, 64, 640, 8, 3, False)])
def test_residual_in_place(ctx, case):
    d = make(ctx, case, True)
    conv, ad = layer(ctx, case, d, True)
    x, slot = E.Tensor.from_numpy(ctx, d["x"]), E.DeviceArray.from_numpy(ctx, d["slot"])
    res, out = E.Tensor.from_numpy(ctx, d["res"]), E.Tensor(ctx)
    conv.forward_adapted(x, ad, slot, out, res)
    conv.forward_adapted(x, ad, slot, res, res)
    assert np.array_equal(res.numpy(), out.numpy())


@pytest.mark.parametrize("fast", [False, True])
@pytest.mark.parametrize("wf16", [False, True])
@pytest.mark.parametrize("af16", [False, True])
@pytest.mark.parametrize("case", [(1, 1, 20, 96, 80, 8, 3, True), (1, 1, 700, 1100, 320, 40, 3, True), (1, 1, 2100, 96, 1280, 8, 3, True),
                                  (1, 1, 5600, 70, 1030, 20, 3, True), (1, 1, 300, 1300, 650, 256, 2, True)])
def test_infinite_values(ctx, case, wf16, af16, fast):
    """Infinities in x, weight and adapters give the formula's infinities, and NaN where it has NaN, however many rows."""
    rows, ci, co, rank, slots = case[2:7]
    d = make(ctx, case, False)
    for name, half in (("w", wf16), ("a", af16), ("b", af16)):
        d[name] = d[name].astype(np.float16 if half else np.float32)
        d[name][np.abs(d[name].astype(np.float32)) < 2.0 ** -12] = 2.0 ** -12  # no product of infinity and zero
        d[name].reshape(-1)[::5] = np.sign(d[name].reshape(-1)[::5]) * 0.5  # low parts of zero
    d["x"] += np.where(d["x"] < 0, -2.0 ** -6, 2.0 ** -6).astype(np.float32)
    d["x"][0, 0, ::4] = np.sign(d["x"][0, 0, ::4])
    d["slot"][:] = np.arange(rows) % (slots + 1) - 1
    x = d["x"][0, 0]
    x[2, 7], x[9, 3], x[10, 3], x[10, 4], x[18, 5] = np.inf, -np.inf, np.inf, -np.inf, np.nan
    x[rows - 1, ci - 1] = np.inf
    d["w"][5, 1], d["w"][co - 1, ci - 1], d["w"][33, 2] = np.inf, -np.inf, np.nan
    d["a"][1, 3, 6], d["b"][1, 41, 2], d["b"][0, 2, rank - 1] = -np.inf, np.inf, np.inf
    conv = E.Conv1x1(ctx, ci, co, E.Param(ctx, d["w"], f16=wf16), d["bias"])
    ad = Adapters(ctx, E.Param(ctx, d["a"], f16=af16), E.Param(ctx, d["b"], f16=af16), d["scale"], ci, co, rank)
    out = E.Tensor(ctx)
    ctx.set_precision(fast)
    try:
        conv.forward_adapted(E.Tensor.from_numpy(ctx, d["x"]), ad, E.DeviceArray.from_numpy(ctx, d["slot"]), out)
    finally:
        ctx.set_precision(False)
    got = out.numpy()[0, 0]
    with np.errstate(invalid="ignore"):
        y, base, low = reference(x, d["w"], d["bias"], None, d["a"], d["b"], d["scale"], d["slot"], 1)
    assert 0 < np.isinf(y).sum() and 0 < np.isnan(y).sum() and 0.5 * y.size < np.isfinite(y).sum()
    assert np.array_equal(np.isnan(got), np.isnan(y))
    assert np.array_equal(np.isposinf(got), np.isposinf(y)) and np.array_equal(np.isneginf(got), np.isneginf(y))
    there = np.isfinite(y)
    bound = (2.0 ** -10 if fast else 1e-5) * base + (ci + rank + 8) * U * low + U * np.abs(y)
    assert np.all(np.abs(got[there] - y[there]) <= bound[there])


@pytest.mark.parametrize("fast", [False, True])
@pytest.mark.parametrize("wf16", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_weight_and_adapters_of_different_types(ctx, case, wf16, fast):
    n, h, w, ci, co, rank, slots, pixel = case
    d = make(ctx, case, wf16, seed=1)
    d["a"], d["b"] = (d[t].astype(np.float32 if wf16 else np.float16) for t in "ab")
    conv = E.Conv1x1(ctx, ci, co, E.Param(ctx, d["w"], f16=wf16), d["bias"])
    ad = Adapters(ctx, E.Param(ctx, d["a"], f16=not wf16), E.Param(ctx, d["b"], f16=not wf16), d["scale"], ci, co, rank)
    out = E.Tensor(ctx)
    ctx.set_precision(fast)
    try:
        conv.forward_adapted(E.Tensor.from_numpy(ctx, d["x"]), ad, E.DeviceArray.from_numpy(ctx, d["slot"]), out)
    finally:
        ctx.set_precision(False)
    y, base, low = reference(d["x"].reshape(-1, ci), d["w"], d["bias"], None, d["a"], d["b"], d["scale"], d["slot"], 1 if pixel else h * w)
    err = np.abs(out.numpy().reshape(-1, co) - y)
    bound = (2.0 ** -10 if fast else 1e-5) * base + (ci + rank + 8) * U * low + U * np.abs(y)
    assert np.all(err <= bound), (err / bound).max()


def test_refused_calls_leave_their_tensors(ctx):
    """A residual or an input that is also out, but of another shape, is refused before out is reshaped."""
    case = (2, 2, 2, 32, 16, 4, 2, False)
    d = make(ctx, case, False)
    conv, ad = layer(ctx, case, d, False)
    x, slot = E.Tensor.from_numpy(ctx, d["x"]), E.DeviceArray.from_numpy(ctx, d["slot"])
    small = np.ones((1, 2, 2, 16), np.float32)
    res = E.Tensor.from_numpy(ctx, small)
    with pytest.raises(MoebiusError, match="residual shape"):
        conv.forward_adapted(x, ad, slot, res, res)
    assert res.shape == small.shape and np.array_equal(res.numpy(), small)
    with pytest.raises(MoebiusError, match="overlap"):
        conv.forward_adapted(x, ad, slot, x)
    assert x.shape == d["x"].shape and np.array_equal(x.numpy(), d["x"])
