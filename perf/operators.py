"""Measured cases of the transformer operators: what a program that runs image
and video transformers on this framework has it do, through the package's
public entry points, with inputs already on the GPU.

    listed()             the named cases
    draw(rng)            one more case of the same ranges
    prepare(case, seed)  the state a program holds before the call
    run(state)           one pass and its outputs
    work(case)           the bytes and operations the path cannot do without
    exact(case, seed)    the outputs in 64 bits, from the definitions

With own = False run() computes the operators in their plain form, elementary
torch operations in 32 bits (64 for angles and for the block scores, whose
order decides); with own = True it calls the framework.

Five operators:

  rope     rotary positions with several axes (time, height, width)
  qknorm   RMS norm of every query and key head with the rotation in the same pass
  select   the key blocks each block of queries attends to, by the product of
           their mean query and the blocks' mean keys
  attend   attention over the selected blocks
  lora     a shared 1x1 projection with a low-rank adapter per request
"""
from __future__ import annotations

import math

import torch

own = False

THETA = 10000.0


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # The deepest map of a small image, one request: the call costs its launch.
        {"name": "rope_8x8_f32", "op": "rope", "n": 1, "t": 1, "h": 8, "w": 8, "heads": 8, "d": 40, "f16": False,
         "axes": 2, "halves": False, "inverse": False},
        # The queries of a video of 16 latent frames: bound by memory alone.
        {"name": "rope_video_f16", "op": "rope", "n": 1, "t": 16, "h": 32, "w": 32, "heads": 16, "d": 128,
         "f16": True, "axes": 3, "halves": True, "inverse": False},
        # One new token for each of 8 requests, queries and keys of a fused projection.
        {"name": "qknorm_token_f16", "op": "qknorm", "n": 8, "t": 1, "h": 1, "w": 1, "hq": 32, "hk": 8, "d": 128,
         "f16": True, "axes": 3, "halves": True},
        # Both guidance branches of a 64x64 latent, in the framework's f32 activations.
        {"name": "qknorm_image_f32", "op": "qknorm", "n": 2, "t": 1, "h": 64, "w": 64, "hq": 8, "hk": 8, "d": 160,
         "f16": False, "axes": 2, "halves": False},
        # The selection of the 64x64 latent: 64 blocks of 64 tokens.
        {"name": "select_image_f32", "op": "select", "n": 2, "q": 4096, "kv": 4096, "hq": 8, "hk": 8, "d": 80,
         "f16": False, "qb": 64, "kb": 64, "top": 16, "causal": False, "ragged": False},
        # The selection of a long video sequence.
        {"name": "select_video_f16", "op": "select", "n": 1, "q": 16384, "kv": 16384, "hq": 16, "hk": 8, "d": 128,
         "f16": True, "qb": 64, "kb": 64, "top": 32, "causal": False, "ragged": False},
        # One new token for each of 8 requests over caches of different lengths.
        {"name": "attend_token_f16", "op": "attend", "n": 8, "q": 1, "kv": 16384, "hq": 32, "hk": 8, "d": 128,
         "f16": True, "qb": 1, "kb": 64, "top": 32, "causal": True, "ragged": True},
        # Self-attention of both guidance branches of a 64x64 latent in f32.
        {"name": "attend_image_f32", "op": "attend", "n": 2, "q": 4096, "kv": 4096, "hq": 8, "hk": 8, "d": 80,
         "f16": False, "qb": 64, "kb": 64, "top": 16, "causal": False, "ragged": False},
        # Requests of different lengths continued over their caches, shared key heads.
        {"name": "attend_ragged_f16", "op": "attend", "n": 4, "q": 1000, "kv": 5003, "hq": 16, "hk": 4, "d": 64,
         "f16": True, "qb": 16, "kb": 32, "top": 24, "causal": True, "ragged": True},
        # Self-attention of the video sequence.
        {"name": "attend_video_f16", "op": "attend", "n": 1, "q": 16384, "kv": 16384, "hq": 16, "hk": 16, "d": 128,
         "f16": True, "qb": 128, "kb": 64, "top": 32, "causal": False, "ragged": False},
        # One row for each of 16 requests, each with an adapter of its own.
        {"name": "lora_token_f16w", "op": "lora", "n": 16, "rows": 1, "ci": 1280, "co": 1280, "rank": 16, "slots": 32,
         "f16w": True, "bias": True, "residual": False},
        # The projection of 8 images of 32x32 latents with their residual.
        {"name": "lora_images_f16w", "op": "lora", "n": 8, "rows": 1024, "ci": 1280, "co": 1280, "rank": 32,
         "slots": 16, "f16w": True, "bias": True, "residual": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "qknorm", "select", "attend", "attend", "lora"])
    if op in ("rope", "qknorm"):
        axes = rng.choice([1, 2, 3])
        c = {"op": op, "n": rng.randint(1, 4), "t": _log(rng, 1, 16) if axes == 3 else 1,
             "h": 1 if axes == 1 else _log(rng, 1, 128 if axes == 2 else 64),
             "w": _log(rng, 1, 8192) if axes == 1 else _log(rng, 1, 128 if axes == 2 else 64),
             "d": rng.choice([32, 40, 64, 72, 80, 96, 128, 160, 256]), "f16": rng.random() < 0.5, "axes": axes,
             "halves": rng.random() < 0.5}
        most = 33_000_000 // (c["n"] * c["t"] * c["h"] * c["w"] * c["d"])  # heads of the largest listed pass
        if op == "rope":
            c["heads"], c["inverse"] = max(1, min(most, rng.randint(1, 32))), rng.random() < 0.3
        else:
            c["hk"] = max(1, min(most // 4, rng.choice([1, 2, 4, 8, 16])))
            c["hq"] = c["hk"] * rng.choice([1, 1, 2, 4])
        return c
    if op in ("select", "attend"):
        c = {"op": op, "d": rng.choice([40, 64, 80, 96, 128, 160]), "f16": rng.random() < 0.6,
             "hk": rng.choice([1, 2, 4, 8]), "kb": rng.choice([16, 32, 64, 128]), "top": _log(rng, 4, 48)}
        c["hq"] = c["hk"] * rng.choice([1, 1, 2, 4])
        form = rng.choice(["token", "image", "ragged"])
        if form == "token":  # single tokens over caches
            kv = _log(rng, 100, 16384)
            n = max(1, min(_log(rng, 1, 32), 100_000_000 // (kv * c["hk"] * c["d"])))
            return dict(c, n=n, q=1, kv=kv, qb=1, causal=True, ragged=True)
        if form == "image":  # self-attention of a map or a video
            q, n, qb = _log(rng, 200, 8192), rng.randint(1, 2), rng.choice([32, 64, 128])
            c, kv = dict(c, causal=False, ragged=False), q
        else:
            q, n, qb = _log(rng, 8, 1500), rng.randint(1, 4), rng.choice([8, 16, 32])
            c, kv = dict(c, causal=True, ragged=True), q + _log(rng, 1, 4000)
        # keys per query such that the pass stays below the largest listed one
        keys = min(4e10 / (n * q * c["hq"] * c["d"]), 5e8 / (n * (q / qb + 1) * c["hk"] * c["d"]))
        return dict(c, n=n, q=q, kv=kv, qb=qb, top=max(5, min(c["top"], int(keys) // c["kb"])))
    n = _log(rng, 1, 16)
    return {"op": op, "n": n, "rows": _log(rng, 1, 8192 // n) if rng.random() < 0.6 else 1, "ci": _log(rng, 64, 1280),
            "co": _log(rng, 64, 1280), "rank": rng.choice([4, 8, 10, 16, 32, 64]), "slots": rng.randint(1, 32),
            "f16w": rng.random() < 0.6, "bias": rng.random() < 0.5, "residual": rng.random() < 0.5}


# ---------------------------------------------------------------- inputs

def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 64 + salt) & 0x7FFFFFFFFFFF)


def _normal(seed, salt, shape, std=1.0, mean=0.0):
    return torch.randn(tuple(shape), generator=_gen(seed, salt), device="cuda") * std + mean


def _ints(seed, salt, lo, hi, shape):
    return torch.randint(lo, hi, tuple(shape), generator=_gen(seed, salt), device="cuda")


def _store(c, x):
    return x.half() if c["f16"] else x


def _axis_dims(d, axes):
    """Even channel counts per axis that add up to d: a small first axis of three, equal halves of two."""
    if axes == 1:
        return [d]
    if axes == 2:
        a = 2 * ((d // 2 + 1) // 2)
        return [a, d - a]
    a = 2 * (3 * d // 16)
    return [d - 2 * a, a, a]


def _frequencies(dims):
    """theta^(-2i / dim) for every pair of every axis, in f64."""
    return torch.cat([THETA ** (-torch.arange(0, m, 2, dtype=torch.float64) / m) for m in dims]).cuda()


def _positions(c, seed):
    """The (time, height, width) of every token of one item, from a first position that a long run may have reached
    (single tokens: one of its own for every request)."""
    tokens = c["t"] * c["h"] * c["w"]
    if tokens == 1 and c["n"] > 1:
        return _ints(seed, 9, 0, 100_000, (c["n"], c["axes"])).int()
    i = torch.arange(tokens, device="cuda")
    p = torch.stack([i // (c["h"] * c["w"]), i // c["w"] % c["h"], i % c["w"]], 1)[:, 3 - c["axes"]:]
    first = _ints(seed, 9, 0, 20_000, (1, c["axes"]))
    first[:, 1:] = 0
    return (p + first).int()


def _lengths(c, seed):
    """Lengths of the items' caches and of their queries: the full ones, or ragged ones with at least a block of cache."""
    kv = torch.full((c["n"],), c["kv"], device="cuda", dtype=torch.int64)
    q = torch.full((c["n"],), c["q"], device="cuda", dtype=torch.int64)
    if c["ragged"]:
        q = torch.maximum(torch.ones_like(q), q - _ints(seed, 11, 0, max(1, c["q"] // 3), (c["n"],)))
        kv = torch.maximum(q, _ints(seed, 10, c["kv"] // 2, c["kv"] + 1, (c["n"],)))
        kv[0] = c["kv"]
    return q, kv


def _blocks_of(c, q_len, kv_len, score):
    """The `top` best blocks of `score` [n][query blocks][key heads][key blocks] that a block of queries may see, those
    of its own tokens first where causal; ascending, -1 behind the last. Ties go to the lower index."""
    nq, nk = score.shape[1], score.shape[3]
    i = torch.arange(nq, device="cuda")[None, :]
    b = torch.arange(nk, device="cuda")[None, None, :]
    live = (i * c["qb"] < q_len[:, None])[:, :, None]
    last = kv_len[:, None].expand(-1, nq) - 1
    forced = torch.zeros((c["n"], nq, nk), dtype=torch.bool, device="cuda")
    if c["causal"]:
        off = (kv_len - q_len)[:, None]
        lo, hi = off + i * c["qb"], off + torch.minimum((i + 1) * c["qb"], q_len[:, None]) - 1
        last = torch.minimum(last, hi)
        forced = (b >= (lo // c["kb"])[:, :, None]) & (b <= (hi // c["kb"])[:, :, None])
    seen = live & (b * c["kb"] <= last[:, :, None])
    inf = float("inf")
    s = torch.where((seen & forced)[:, :, None, :], inf, torch.where(seen[:, :, None, :], score, -inf))
    order = torch.sort(s, dim=-1, descending=True, stable=True).indices[..., :c["top"]]
    ok = torch.gather(seen[:, :, None, :].expand_as(s), 3, order)
    got = torch.sort(torch.where(ok, order, nk), dim=-1).values
    got = torch.where(got < nk, got, -1).int()
    pad = c["top"] - got.shape[-1]
    return torch.nn.functional.pad(got, (0, pad), value=-1) if pad > 0 else got


def _inputs(c, seed):
    """The tensors of one case, from the seed alone."""
    op = c["op"]
    if op == "rope":
        dims = _axis_dims(c["d"], c["axes"])
        p = _positions(c, seed)
        rows = c["n"] * c["t"] * c["h"] * c["w"]
        return {"x": _store(c, _normal(seed, 1, (rows, c["heads"], c["d"]))), "pos": p, "dims": dims,
                "freq": _frequencies(dims)}
    if op == "qknorm":
        dims = _axis_dims(c["d"], c["axes"])
        rows = c["n"] * c["t"] * c["h"] * c["w"]
        # queries, keys and values of one projection, next to each other in every row
        qkv = _store(c, _normal(seed, 1, (rows, c["hq"] + 2 * c["hk"], c["d"]), 1.7, 0.1))
        return {"qkv": qkv, "pos": _positions(c, seed), "dims": dims, "freq": _frequencies(dims),
                "gq": _normal(seed, 2, (c["d"],), 0.1, 1.0), "gk": _normal(seed, 3, (c["d"],), 0.1, 1.0), "eps": 1e-6}
    if op in ("select", "attend"):
        q_len, kv_len = _lengths(c, seed)
        nk, nq = -(-c["kv"] // c["kb"]), -(-c["q"] // c["qb"])
        # keys lie around a centre of their own block, queries near one of these
        centre = _normal(seed, 4, (c["n"], nk, c["hk"], c["d"]), 0.5)
        near = torch.arange(c["q"], device="cuda") * nk // c["q"]
        q = _normal(seed, 1, (c["n"], c["q"], c["hq"], c["d"]))
        q += centre[:, near].repeat_interleave(c["hq"] // c["hk"], 2)
        k = _normal(seed, 2, (c["n"], c["kv"], c["hk"], c["d"]))
        k += centre.repeat_interleave(c["kb"], 1)[:, :c["kv"]]
        st = {"q": _store(c, q), "k": _store(c, k), "q_len": q_len.int(), "kv_len": kv_len.int()}
        if op == "attend":
            st["v"] = _store(c, _normal(seed, 3, (c["n"], c["kv"], c["hk"], c["d"])))
            score = torch.rand((c["n"], nq, c["hk"], nk), generator=_gen(seed, 5), device="cuda")
            st["blocks"] = _blocks_of(c, q_len, kv_len, score)
            st["scale"] = 1.0 / math.sqrt(c["d"])
        return st
    rows = c["n"] * c["rows"]
    w = _normal(seed, 2, (c["co"], c["ci"]), math.sqrt(2.0 / c["ci"]))
    a = _normal(seed, 3, (c["slots"], c["rank"], c["ci"]), math.sqrt(1.0 / c["ci"]))
    b = _normal(seed, 4, (c["slots"], c["co"], c["rank"]), 0.1)
    if c["f16w"]:
        w, a, b = w.half(), a.half(), b.half()
    return {"x": _normal(seed, 1, (rows, c["ci"])), "w": w, "a": a, "b": b,
            "scale": _normal(seed, 5, (c["slots"],), 0.2, 1.0),
            # the adapter of each request; one in eight has none
            "slot": torch.where(_ints(seed, 7, 0, 8, (c["n"],)) == 0, -1, _ints(seed, 6, 0, c["slots"], (c["n"],))).int(),
            "bias": _normal(seed, 8, (c["co"],), 0.02) if c["bias"] else None,
            "residual": _normal(seed, 9, (rows, c["co"])) if c["residual"] else None}


# ---------------------------------------------------------------- the calls

_kept: dict = {}


class _View:
    """A device buffer of the framework as torch sees it (no copy)."""

    def __init__(self, d):
        self.keep = d
        self.__cuda_array_interface__ = {"shape": tuple(d.shape), "typestr": d.dtype.str, "data": (d.ptr, False),
                                         "version": 2}


def _torch(d):
    return torch.as_tensor(_View(d), device="cuda")


def _own_state(c, d):
    """The framework's arrays of a case's tensors, its outputs and the objects that a program keeps."""
    from moebius_cpu_amd import attention as A
    from moebius_cpu_amd import engine as E

    if "ctx" not in _kept:
        _kept["ctx"] = E.Context(0)
    ctx = _kept["ctx"]

    def array(t):
        if t is None:
            return None
        dev = E.DeviceArray(ctx, t.shape, {torch.float32: "f4", torch.float16: "f2", torch.int32: "i4"}[t.dtype])
        _torch(dev).copy_(t)
        return dev

    def outputs(**named):
        """Zeroed outputs, and torch's view of them."""
        return named, {k: _torch(v).zero_() for k, v in named.items()}

    st = {"op": c["op"], "case": c}
    if c["op"] in ("rope", "qknorm"):
        st["rope"] = A.RopeAxes(ctx, d["dims"], theta=THETA, pairing="halves" if c["halves"] else "interleaved")
        st["pos"] = array(d["pos"])
    if c["op"] == "rope":
        rows, heads, dim = d["x"].shape
        x = array(d["x"])
        out, st["view"] = outputs(out=E.DeviceArray(ctx, d["x"].shape, x.dtype))
        st.update(x=A.Heads(x, 1, rows, heads, dim), out=A.Heads(out["out"], 1, rows, heads, dim))
    elif c["op"] == "qknorm":
        rows, hq, hk, dim = d["qkv"].shape[0], c["hq"], c["hk"], c["d"]
        qkv, ld = array(d["qkv"]), (c["hq"] + 2 * c["hk"]) * c["d"]
        out, st["view"] = outputs(q=E.DeviceArray(ctx, (rows, hq, dim), qkv.dtype),
                                  k=E.DeviceArray(ctx, (rows, hk, dim), qkv.dtype))
        st.update(q=A.Heads(qkv, 1, rows, hq, dim, ld=ld), k=A.Heads(qkv, 1, rows, hk, dim, ld=ld, offset=hq * dim),
                  gq=array(d["gq"]), gk=array(d["gk"]), eps=d["eps"], q_out=A.Heads(out["q"], 1, rows, hq, dim),
                  k_out=A.Heads(out["k"], 1, rows, hk, dim))
    elif c["op"] in ("select", "attend"):
        n, nq, nk = c["n"], -(-c["q"] // c["qb"]), -(-c["kv"] // c["kb"])
        st.update(q=A.Heads(array(d["q"]), n, c["q"], c["hq"], c["d"]), k=A.Heads(array(d["k"]), n, c["kv"], c["hk"], c["d"]),
                  q_len=array(d["q_len"]), kv_len=array(d["kv_len"]))
        if c["op"] == "select":
            out, st["view"] = outputs(means=E.DeviceArray(ctx, (n, nk, c["hk"], c["d"])),
                                      blocks=E.DeviceArray(ctx, (n, nq, c["hk"], c["top"]), "i4"))
            st.update(out)
        else:
            out, st["view"] = outputs(out=E.DeviceArray(ctx, d["q"].shape, st["q"].dtype))
            st.update(v=A.Heads(array(d["v"]), n, c["kv"], c["hk"], c["d"]), blocks=array(d["blocks"]),
                      out=A.Heads(out["out"], n, c["q"], c["hq"], c["d"]), scale=d["scale"])
    else:
        from moebius_cpu_amd.adapters import Adapters

        w = E.Param(ctx, d["w"].cpu().numpy(), f16=c["f16w"])
        st["adapters"] = Adapters(ctx, E.Param(ctx, d["a"].cpu().numpy(), f16=c["f16w"]),
                                  E.Param(ctx, d["b"].cpu().numpy(), f16=c["f16w"]), d["scale"].cpu().numpy(),
                                  c["ci"], c["co"], c["rank"])
        st["conv"] = E.Conv1x1(ctx, c["ci"], c["co"], w, None if d["bias"] is None else d["bias"].cpu().numpy())

        def tensor(t):
            if t is None:
                return None
            dev = E.Tensor(ctx, c["n"], 1, c["rows"], t.shape[1])
            _torch(dev).copy_(t.view(dev.shape))
            return dev

        out, view = outputs(out=E.Tensor(ctx, c["n"], 1, c["rows"], c["co"]))
        st["view"] = {"out": view["out"].view(c["n"] * c["rows"], c["co"])}
        st.update(out, x=tensor(d["x"]), residual=tensor(d["residual"]), slot=array(d["slot"]))
    torch.cuda.synchronize()
    return st


def prepare(case, seed):
    d = _inputs(case, seed)
    if own:
        return _own_state(case, d)
    return dict(d, op=case["op"], case=case)


def _run_own(st):
    c = st["case"]
    if st["op"] == "rope":
        from moebius_cpu_amd.attention import rope_axes

        rope_axes(st["x"], st["pos"], st["rope"], st["out"], inverse=c["inverse"])
    elif st["op"] == "qknorm":
        from moebius_cpu_amd.attention import qk_norm_rope

        qk_norm_rope(st["q"], st["k"], st["gq"], st["gk"], st["eps"], st["pos"], st["rope"], st["q_out"], st["k_out"])
    elif st["op"] == "select":
        from moebius_cpu_amd.attention import block_means, block_select

        block_means(st["k"], c["kb"], st["means"], length=st["kv_len"])
        block_select(st["q"], st["means"], c["kv"], st["blocks"], q_block=c["qb"], kv_block=c["kb"],
                     causal=c["causal"], q_len=st["q_len"], kv_len=st["kv_len"])
    elif st["op"] == "attend":
        from moebius_cpu_amd.attention import block_attention

        block_attention(st["q"], st["k"], st["v"], st["blocks"], st["out"], scale=st["scale"], q_block=c["qb"],
                        kv_block=c["kb"], causal=c["causal"], q_len=st["q_len"], kv_len=st["kv_len"])
    else:
        st["conv"].forward_adapted(st["x"], st["adapters"], st["slot"], st["out"], st["residual"])
    return st["view"]


def run(st):
    if own:
        return _run_own(st)
    return {"rope": _plain_rope, "qknorm": _plain_qknorm, "select": _plain_select, "attend": _plain_attend,
            "lora": _plain_lora}[st["op"]](st, st["case"])


# ---------------------------------------------------------------- the plain forms

def _plain_angles(st, rows):
    """cos and sin of every row and pair [rows][1][pairs]: the angles in f64, item after item over the same positions."""
    axis = torch.repeat_interleave(torch.arange(len(st["dims"])), torch.tensor(st["dims"]) // 2).cuda()
    a = st["pos"].double()[:, axis] * st["freq"]
    a = a.repeat(rows // a.shape[0], 1)[:, None]
    return torch.cos(a).float(), torch.sin(a).float()


def _plain_turn(x, cos, sin, halves):
    """x [rows][heads][d] in f32, turned pair by pair."""
    if halves:
        a, b = x.chunk(2, -1)
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)


def _plain_rope(st, c):
    cos, sin = _plain_angles(st, st["x"].shape[0])
    return {"out": _plain_turn(st["x"].float(), cos, -sin if c["inverse"] else sin, c["halves"]).to(st["x"].dtype)}


def _plain_qknorm(st, c):
    q, k = st["qkv"][:, :c["hq"]].float(), st["qkv"][:, c["hq"]:c["hq"] + c["hk"]].float()
    cos, sin = _plain_angles(st, q.shape[0])
    q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + st["eps"]) * st["gq"]
    k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + st["eps"]) * st["gk"]
    t = st["qkv"].dtype
    return {"q": _plain_turn(q, cos, sin, c["halves"]).to(t), "k": _plain_turn(k, cos, sin, c["halves"]).to(t)}


def _plain_means(x, length, block):
    """Mean over every block of tokens [n][blocks][heads][d], f64 sums rounded once to f32; zeros where a block is empty."""
    n, tokens, heads, d = x.shape
    nb = -(-tokens // block)
    i = torch.arange(nb * block, device="cuda")
    x = torch.nn.functional.pad(x.double(), (0, 0, 0, 0, 0, nb * block - tokens))
    x = torch.where((i < length[:, None])[:, :, None, None], x, 0.0)
    count = (length[:, None] - torch.arange(nb, device="cuda") * block).clamp(0, block)
    return (x.view(n, nb, block, heads, d).sum(2) / count.clamp(min=1)[:, :, None, None]).float()


def _plain_select(st, c):
    q_len, kv_len, g = st["q_len"].long(), st["kv_len"].long(), c["hq"] // c["hk"]
    km = _plain_means(st["k"], kv_len, c["kb"])
    n, q = c["n"], st["q"].view(c["n"], c["q"], c["hk"], g, c["d"])
    # the mean query of a block and of the heads that share a key head: a mean over blocks of qb * g rows
    qm = _plain_means(q.transpose(2, 3).reshape(n, c["q"] * g, c["hk"], c["d"]), q_len * g, c["qb"] * g)
    score = torch.matmul(qm.double().transpose(1, 2), km.double().permute(0, 2, 3, 1).contiguous())
    return {"means": km, "blocks": _blocks_of(c, q_len, kv_len, score.transpose(1, 2))}


def _plain_attend(st, c):
    n, qb, kb, hk, d, g = c["n"], c["qb"], c["kb"], c["hk"], c["d"], c["hq"] // c["hk"]
    nq, nk, top = st["blocks"].shape[1], -(-c["kv"] // kb), st["blocks"].shape[3]
    q_len, kv_len = st["q_len"].long()[:, None, None], st["kv_len"].long()[:, None, None]
    # the tokens of the selected blocks [n][nq][hk][top * kb], and which of them there are
    blocks = st["blocks"].long()
    token = blocks[..., None] * kb + torch.arange(kb, device="cuda")
    token = torch.where(blocks[..., None] >= 0, token, nk * kb).flatten(3)
    there = token < kv_len[..., None]
    at = token.clamp(max=c["kv"] - 1)
    item = torch.arange(n, device="cuda")[:, None, None, None]
    head = torch.arange(hk, device="cuda")[None, None, :, None]
    k, v = st["k"][item, at, head].float(), st["v"][item, at, head].float()  # [n][nq][hk][keys][d]
    v = torch.where(there[..., None], v, 0.0)
    q = torch.nn.functional.pad(st["q"].float(), (0, 0, 0, 0, 0, nq * qb - c["q"]))
    q = q.view(n, nq, qb, hk, g, d).permute(0, 1, 3, 2, 4, 5).reshape(n, nq, hk, qb * g, d)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * st["scale"]
    seen = there[:, :, :, None, :]
    if c["causal"]:
        i = torch.arange(nq * qb, device="cuda").view(nq, qb).repeat_interleave(g, 1)
        seen = seen & (token[:, :, :, None, :] <= (i + kv_len - q_len)[:, :, None, :, None])
    s = torch.where(seen, s, float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = o.view(n, nq, hk, qb, g, d).permute(0, 1, 3, 2, 4, 5).reshape(n, nq * qb, c["hq"], d)[:, :c["q"]]
    live = torch.arange(c["q"], device="cuda")[None, :] < q_len[:, :, 0]
    return {"out": torch.where(live[:, :, None, None], o, 0.0).to(st["q"].dtype)}


def _plain_lora(st, c):
    x = st["x"]
    y = torch.matmul(x, st["w"].float().t())
    if st["bias"] is not None:
        y = y + st["bias"]
    if st["residual"] is not None:
        y = y + st["residual"]
    slot = st["slot"].long()
    a, b = st["a"].float()[slot.clamp(min=0)], st["b"].float()[slot.clamp(min=0)]
    scale = torch.where(slot >= 0, st["scale"][slot.clamp(min=0)], 0.0)[:, None, None]
    t = torch.matmul(x.view(c["n"], c["rows"], c["ci"]), a.transpose(1, 2).contiguous()) * scale
    return {"out": y + torch.matmul(t, b.transpose(1, 2).contiguous()).view(y.shape)}


# ---------------------------------------------------------------- bytes and operations

def work(case):
    c, op = case, case["op"]
    if op == "rope":
        e = c["n"] * c["t"] * c["h"] * c["w"] * c["heads"] * c["d"]
        return {"bytes": 2.0 * e * (2 if c["f16"] else 4), "flops": 3.0 * e}
    if op == "qknorm":
        e = c["n"] * c["t"] * c["h"] * c["w"] * (c["hq"] + c["hk"]) * c["d"]
        return {"bytes": 2.0 * e * (2 if c["f16"] else 4), "flops": 8.0 * e}
    if op in ("select", "attend"):
        size, g = 2 if c["f16"] else 4, c["hq"] // c["hk"]
        nq, nk = -(-c["q"] // c["qb"]), -(-c["kv"] // c["kb"])
        queries = float(c["n"] * c["q"] * c["hq"] * c["d"])
        if op == "select":
            keys = float(c["n"] * c["kv"] * c["hk"] * c["d"])
            means, scores = keys / c["kb"], float(c["n"] * nq * c["hk"]) * nk
            return {"bytes": size * (queries + keys) + 4.0 * means + 4.0 * c["n"] * nq * c["hk"] * c["top"],
                    "flops": queries + keys + 2.0 * scores * c["d"]}
        picked = min(c["top"] * c["kb"], c["kv"])
        read = float(c["n"] * c["hk"] * c["d"]) * min(c["kv"], nq * picked)  # every selected key and value once
        return {"bytes": size * (2.0 * queries + 2.0 * read), "flops": 4.0 * queries * picked}
    rows, wb = c["n"] * c["rows"], 2 if c["f16w"] else 4
    used = min(c["n"], c["slots"])
    return {"bytes": 4.0 * rows * (c["ci"] + c["co"] * (2 if c["residual"] else 1)) + wb * c["ci"] * c["co"]
            + wb * used * c["rank"] * (c["ci"] + c["co"]),
            "flops": 2.0 * rows * (c["ci"] * c["co"] + c["rank"] * (c["ci"] + c["co"]))}


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_turn(x, st, rows, halves, inverse=False):
    """Each pair as a complex number times e^(i angle)."""
    first = 0
    angle = torch.empty((st["pos"].shape[0], sum(st["dims"]) // 2), dtype=torch.float64, device="cuda")
    for axis, m in enumerate(st["dims"]):
        f = torch.pow(torch.tensor(THETA, dtype=torch.float64), torch.arange(m // 2, dtype=torch.float64) * (-2.0 / m))
        angle[:, first:first + m // 2] = torch.outer(st["pos"][:, axis].double(), f.cuda())
        first += m // 2
    turn = torch.polar(torch.ones_like(angle), -angle if inverse else angle)
    turn = turn[torch.arange(rows, device="cuda") % turn.shape[0]][:, None, :]
    if halves:
        h = x.shape[-1] // 2
        z = torch.complex(x[..., :h], x[..., h:]) * turn
        return torch.cat([z.real, z.imag], -1)
    z = torch.view_as_complex(x.reshape(*x.shape[:-1], -1, 2).contiguous()) * turn
    return torch.view_as_real(z).reshape(x.shape)


def exact(case, seed):
    c = case
    st = _inputs(c, seed)
    if c["op"] == "rope":
        return {"out": _exact_turn(st["x"].double(), st, st["x"].shape[0], c["halves"], c["inverse"])}
    if c["op"] == "qknorm":
        out = {}
        for name, lo, hi, gamma in (("q", 0, c["hq"], st["gq"]), ("k", c["hq"], c["hq"] + c["hk"], st["gk"])):
            x = st["qkv"][:, lo:hi].double()
            x = x / torch.sqrt(torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / c["d"] + st["eps"])
            out[name] = _exact_turn(x * gamma.double(), st, x.shape[0], c["halves"])
        return out
    if c["op"] == "select":
        means = torch.zeros((c["n"], -(-c["kv"] // c["kb"]), c["hk"], c["d"]), dtype=torch.float64, device="cuda")
        for i in range(c["n"]):
            for b, lo in enumerate(range(0, int(st["kv_len"][i]), c["kb"])):
                means[i, b] = st["k"][i, lo:min(lo + c["kb"], int(st["kv_len"][i]))].double().mean(0)
        return {"means": means, "blocks": None}
    if c["op"] == "attend":
        g, n, nq = c["hq"] // c["hk"], c["n"], st["blocks"].shape[1]
        out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
        lens = list(zip(st["q_len"].tolist(), st["kv_len"].tolist()))
        if n * nq * c["hk"] > 20_000:
            return None
        blocks = st["blocks"].cpu()
        for i, (ql, kl) in enumerate(lens):
            for b in range(-(-ql // c["qb"])):
                rows = torch.arange(b * c["qb"], min((b + 1) * c["qb"], ql), device="cuda")
                for h in range(c["hk"]):
                    token = torch.cat([torch.arange(j * c["kb"], min((j + 1) * c["kb"], kl))
                                       for j in blocks[i, b, h].tolist() if j >= 0] or [torch.arange(0)]).cuda()
                    k, v = st["k"][i, token, h].double(), st["v"][i, token, h].double()
                    for e in range(h * g, (h + 1) * g):
                        s = torch.matmul(st["q"][i, rows, e].double(), k.t()) * st["scale"]
                        if c["causal"]:
                            s = s.masked_fill(token[None, :] > (rows + kl - ql)[:, None], -math.inf)
                        out[i, rows, e] = torch.matmul(torch.softmax(s, -1), v)
        return {"out": out}
    x, y = st["x"].double(), []
    for i in range(c["n"]):
        part = x[i * c["rows"]:(i + 1) * c["rows"]]
        j = int(st["slot"][i])
        w = st["w"].double()
        if j >= 0:  # the adapter folded into the weight
            w = w + st["scale"][j].double() * torch.matmul(st["b"][j].double(), st["a"][j].double())
        y.append(torch.matmul(part, w.t()))
    y = torch.cat(y)
    if st["bias"] is not None:
        y = y + st["bias"].double()
    return {"out": y if st["residual"] is None else y + st["residual"].double()}
