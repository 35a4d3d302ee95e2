"""Measured cases of the operators around a streaming transformer block: what a
program that generates images and videos token after token, or frame after frame,
has this framework do, through the package's public entry points, with inputs
already on the GPU.

    listed()             the named cases
    draw(rng)            one more case of the same ranges
    prepare(case, seed)  the state a program holds before the call
    run(state)           one pass and its outputs
    work(case)           the bytes and operations the path cannot do without
    exact(case, seed)    the outputs in 64 bits, from the definitions

With own = False run() computes the operators in their plain form, elementary
torch operations in 32 bits (64 for quotients next to a border of two codes);
with own = True it calls the framework.

Three operators:

  cache   keys and values quantised to 8 bits as they are written into the pages of a
          cache, with a scale for each block of tokens and head, and the blocks that
          were written read back
  attend  attention over such a cache: causal or not, with a sliding window and a few
          first tokens that stay visible
  norm    the gated residual of a branch (normed or not) and the modulated norm of the sum
"""
from __future__ import annotations

import math

import torch

own = False


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # One new token for each of 16 requests, into blocks that are partly filled.
        {"name": "cache_token_f16", "op": "cache", "n": 16, "tokens": 1, "hist": 500, "hk": 8, "d": 128, "block": 64,
         "f16": True},
        # Both guidance branches of a 64x64 latent, in the framework's f32 activations.
        {"name": "cache_image_f32", "op": "cache", "n": 2, "tokens": 4096, "hist": 0, "hk": 8, "d": 80, "block": 64,
         "f16": False},
        # A video sequence of 16 latent frames behind a text of odd length.
        {"name": "cache_video_f16", "op": "cache", "n": 1, "tokens": 16384, "hist": 77, "hk": 16, "d": 128, "block": 64,
         "f16": True},
        # One new token of a single request over a short cache in f32: the call costs its latency.
        {"name": "attend_short_f32", "op": "attend", "n": 1, "q": 1, "kv": 300, "hq": 8, "hk": 8, "d": 80, "block": 32,
         "f16": False, "causal": True, "window": 0, "sinks": 0, "ragged": False},
        # One new token for each of 8 requests over caches of different lengths.
        {"name": "attend_token_f16", "op": "attend", "n": 8, "q": 1, "kv": 16384, "hq": 32, "hk": 8, "d": 128, "block": 64,
         "f16": True, "causal": True, "window": 0, "sinks": 0, "ragged": True},
        # Requests of different lengths continued by a window over their caches, the first tokens kept.
        {"name": "attend_window_f16", "op": "attend", "n": 4, "q": 1000, "kv": 5003, "hq": 16, "hk": 4, "d": 64, "block": 32,
         "f16": True, "causal": True, "window": 1500, "sinks": 100, "ragged": True},
        # Self-attention of both guidance branches of a 64x64 latent in f32.
        {"name": "attend_image_f32", "op": "attend", "n": 2, "q": 4096, "kv": 4096, "hq": 8, "hk": 8, "d": 80, "block": 64,
         "f16": False, "causal": False, "window": 0, "sinks": 0, "ragged": False},
        # Four new frames of a video over the first frame and those of the window before them.
        {"name": "attend_frames_f16", "op": "attend", "n": 1, "q": 4096, "kv": 32768, "hq": 16, "hk": 16, "d": 128,
         "block": 128, "f16": True, "causal": False, "window": 12288, "sinks": 1024, "ragged": False},
        # The last quarter of a long prompt.
        {"name": "attend_prompt_f16", "op": "attend", "n": 1, "q": 4096, "kv": 16384, "hq": 32, "hk": 8, "d": 128,
         "block": 64, "f16": True, "causal": True, "window": 0, "sinks": 0, "ragged": False},
        # One row for each of 16 requests, each with its own modulation.
        {"name": "norm_token_f32", "op": "norm", "n": 16, "rows": 1, "c": 1280, "x16": False, "h16": False, "post": "none",
         "pre": "layer", "affine": False, "branch": True, "mod": True},
        # Both guidance branches of a 64x64 latent.
        {"name": "norm_image_f32", "op": "norm", "n": 2, "rows": 4096, "c": 1280, "x16": False, "h16": False, "post": "none",
         "pre": "layer", "affine": False, "branch": True, "mod": True},
        # A video sequence in f16 branches with norms before and after the block.
        {"name": "norm_video_f16", "op": "norm", "n": 1, "rows": 16384, "c": 2048, "x16": False, "h16": True, "post": "rms",
         "pre": "rms", "affine": True, "branch": True, "mod": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["cache", "attend", "attend", "attend", "norm"])
    if op == "cache":
        c = {"op": op, "hk": rng.choice([1, 2, 4, 8, 16]), "d": rng.choice([32, 40, 64, 72, 80, 96, 128, 160]),
             "block": rng.choice([16, 32, 64, 128]), "f16": rng.random() < 0.6}
        tokens = 1 if rng.random() < 0.4 else _log(rng, 2, 16384)
        most = 33_000_000 // (c["hk"] * c["d"] * (tokens + c["block"]))
        return dict(c, n=max(1, min(most, _log(rng, 1, 32))), tokens=tokens, hist=rng.choice([0, rng.randint(1, 600)]))
    if op == "attend":
        c = {"op": op, "d": rng.choice([40, 64, 80, 96, 128, 160]), "hk": rng.choice([1, 2, 4, 8, 16]),
             "block": rng.choice([16, 32, 64, 128]), "f16": rng.random() < 0.6}
        c["hq"] = c["hk"] * rng.choice([1, 1, 2, 4])
        form = rng.choice(["token", "few", "prompt", "frames"])
        kv = _log(rng, 20, 16384)
        q = 1 if form == "token" else min(kv, _log(rng, 2, 64) if form == "few" else _log(rng, 64, 4096))
        n = max(1, min(_log(rng, 1, 32 if form == "token" else 4), 60_000_000 // (kv * c["hk"] * c["d"]),
                       int(1.2e9 / (float(q) * kv * c["hq"])), int(1.0e11 / (float(q) * kv * c["hq"] * c["d"]))))
        while c["hq"] > c["hk"] and float(q) * kv * c["hq"] * c["d"] > 1.0e11:
            c["hq"] //= 2
        window = rng.choice([0, _log(rng, 8, kv)])
        return dict(c, n=n, q=q, kv=kv, causal=form != "frames", window=window,
                    sinks=rng.choice([0, rng.randint(1, 300)]) if window else 0, ragged=rng.random() < 0.6)
    c = {"op": op, "c": _log(rng, 32, 8192), "x16": rng.random() < 0.3, "h16": rng.random() < 0.5,
         "post": rng.choice(["none", "rms", "layer"]), "pre": rng.choice(["none", "rms", "layer", "layer"]),
         "affine": rng.random() < 0.5, "branch": rng.random() < 0.8, "mod": rng.random() < 0.8}
    if c["c"] % 8 and rng.random() < 0.7:
        c["c"] += 8 - c["c"] % 8
    n = _log(rng, 1, 32)
    return dict(c, n=n, rows=1 if rng.random() < 0.3 else _log(rng, 1, max(1, min(16384, 33_000_000 // (n * c["c"])))))


# ---------------------------------------------------------------- inputs

def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 64 + salt) & 0x7FFFFFFFFFFF)


def _normal(seed, salt, shape, std=1.0, mean=0.0):
    return torch.randn(tuple(shape), generator=_gen(seed, salt), device="cuda") * std + mean


def _ints(seed, salt, lo, hi, shape):
    return torch.randint(lo, hi, tuple(shape), generator=_gen(seed, salt), device="cuda")


def _store(f16, x):
    return x.half() if f16 else x


def _keys_values(c, seed, tokens, salt):
    """Keys with channels of different size, as norms with a learned scale leave them, and values."""
    size = 0.5 + torch.rand((c["hk"], c["d"]), generator=_gen(seed, salt), device="cuda")
    k = _normal(seed, salt + 1, (c["n"], tokens, c["hk"], c["d"])) * size
    return _store(c["f16"], k), _store(c["f16"], _normal(seed, salt + 2, (c["n"], tokens, c["hk"], c["d"])))


def _pages(c, seed, blocks):
    """The pages of every item, in the order in which a busy cache hands them out."""
    return torch.randperm(c["n"] * blocks, generator=_gen(seed, 9), device="cuda").view(c["n"], blocks).int()


def _inputs(c, seed):
    """The tensors of one case, from the seed alone."""
    op = c["op"]
    if op == "cache":
        k, v = _keys_values(c, seed, c["tokens"], 1)
        st = {"k": k, "v": v, "table": _pages(c, seed, -(-(c["hist"] + c["tokens"]) // c["block"])),
              "first": torch.zeros(c["n"], dtype=torch.int32, device="cuda")}
        if c["hist"]:  # items of different lengths
            st["first"] = _ints(seed, 10, (c["hist"] + 1) // 2, c["hist"] + 1, (c["n"],)).int()
            st["k0"], st["v0"] = _keys_values(c, seed, c["hist"], 4)
        return st
    if op == "attend":
        kv = torch.full((c["n"],), c["kv"], device="cuda", dtype=torch.int64)
        q = torch.full((c["n"],), c["q"], device="cuda", dtype=torch.int64)
        if c["ragged"]:
            q = torch.maximum(torch.ones_like(q), q - _ints(seed, 11, 0, max(1, c["q"] // 3), (c["n"],)))
            kv = torch.maximum(q, _ints(seed, 10, c["kv"] // 2, c["kv"] + 1, (c["n"],)))
            kv[0] = c["kv"]
        k, v = _keys_values(c, seed, c["kv"], 1)
        return {"q": _store(c["f16"], _normal(seed, 7, (c["n"], c["q"], c["hq"], c["d"]), 1.5)), "k": k, "v": v,
                "q_len": q.int(), "kv_len": kv.int(), "table": _pages(c, seed, -(-c["kv"] // c["block"])),
                "scale": 1.0 / math.sqrt(c["d"])}
    shape = (c["n"], c["rows"], c["c"])
    st = {"x": _store(c["x16"], _normal(seed, 1, shape, 1.5, 0.2)), "h": None, "gate": None, "scale": None, "shift": None,
          "g_post": None, "g_pre": None, "b_pre": None, "eps": 1e-6, "keep": 1.0}
    if c["branch"]:
        st["h"] = _store(c["h16"], _normal(seed, 2, shape, 0.8, -0.1))
        st["keep"] = 0.9
    if c["mod"]:  # shift, scale and gate of one projection, next to each other in every row
        st["mod"] = _normal(seed, 3, (c["n"], 3 * c["c"]), 0.3)
        st["shift"], st["scale"], st["gate"] = st["mod"].view(c["n"], 3, 1, c["c"]).unbind(1)
    if c["affine"]:
        st["g_post"], st["g_pre"] = _normal(seed, 4, (c["c"],), 0.1, 1.0), _normal(seed, 5, (c["c"],), 0.1, 1.0)
        st["b_pre"] = _normal(seed, 6, (c["c"],), 0.1) if c["pre"] == "layer" else None
    return st


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
    from moebius_cpu_amd import cache as K
    from moebius_cpu_amd import engine as E
    from moebius_cpu_amd import gated_norm as G
    from moebius_cpu_amd.attention import Heads

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

    def heads(t):
        return Heads(array(t), t.shape[0], t.shape[1], t.shape[2], t.shape[3])

    st = {"op": c["op"], "case": c}
    def write(k, v, length):
        k, v, length = heads(k), heads(v), array(length)
        torch.cuda.synchronize()  # the copies run on torch's stream
        K.cache_write(st["cache"], st["table"], k, v, length=length)
        ctx.synchronize()

    if c["op"] in ("cache", "attend"):
        st["cache"] = K.Cache8(ctx, d["table"].numel(), c["hk"], c["d"], c["block"])
        st["table"] = array(d["table"])
    if c["op"] == "cache":
        n, rows = c["n"], _rows_back(c)
        if c["hist"]:
            write(d["k0"], d["v0"], d["first"])
        start = d["first"] // c["block"] * c["block"]
        out, st["view"] = outputs(k=E.DeviceArray(ctx, (n, rows, c["hk"], c["d"]), "f2" if c["f16"] else "f4"),
                                  v=E.DeviceArray(ctx, (n, rows, c["hk"], c["d"]), "f2" if c["f16"] else "f4"))
        st.update(k=heads(d["k"]), v=heads(d["v"]), first=array(d["first"]), start=array(start),
                  back=array(d["first"] - start + c["tokens"]), k_out=Heads(out["k"], n, rows, c["hk"], c["d"]),
                  v_out=Heads(out["v"], n, rows, c["hk"], c["d"]))
    elif c["op"] == "attend":
        write(d["k"], d["v"], d["kv_len"])
        out, st["view"] = outputs(out=E.DeviceArray(ctx, d["q"].shape, "f2" if c["f16"] else "f4"))
        st.update(q=heads(d["q"]), q_len=array(d["q_len"]), kv_len=array(d["kv_len"]), scale=d["scale"],
                  out=Heads(out["out"], c["n"], c["q"], c["hq"], c["d"]))
    else:
        n, rows, ch = d["x"].shape
        out, st["view"] = outputs(**({"x": E.DeviceArray(ctx, d["x"].shape, "f2" if c["x16"] else "f4")} if c["branch"] else {}),
                                  y=E.DeviceArray(ctx, d["x"].shape, "f2" if c["h16"] else "f4"))
        st.update(x=heads(d["x"][:, :, None]), y=Heads(out["y"], n, rows, 1, ch), x_out=None, branch=None, keep=d["keep"],
                  post=None, pre=None, gate=None, scale=None, shift=None)
        if c["pre"] != "none":
            st["pre"] = G.Norm(c["pre"], array(d["g_pre"]), array(d["b_pre"]), d["eps"])
        if c["branch"]:
            st.update(branch=heads(d["h"][:, :, None]), x_out=Heads(out["x"], n, rows, 1, ch))
            if c["post"] != "none":
                st["post"] = G.Norm(c["post"], array(d["g_post"]), None, d["eps"])
        if c["mod"]:
            mod = array(d["mod"])
            st.update({k: Heads(mod, n, 1, 1, ch, ld=3 * ch, offset=i * ch)
                       for i, k in enumerate(("shift", "scale", "gate")) if k != "gate" or c["branch"]})
    _kept["ctx"].synchronize()
    torch.cuda.synchronize()
    return st


def prepare(case, seed):
    d = _inputs(case, seed)
    if own:
        return _own_state(case, d)
    st = dict(d, op=case["op"], case=case)
    if case["op"] == "attend":  # what the cache holds
        for name in ("k", "v"):
            st[name] = _plain_quantise(d[name], d["kv_len"], case["block"])
    if case["op"] == "cache" and case["hist"]:
        for name in ("k0", "v0"):
            st[name] = _plain_quantise(d[name], d["first"], case["block"])
    return st


def _run_own(st):
    c = st["case"]
    if st["op"] == "cache":
        from moebius_cpu_amd.cache import cache_read, cache_write

        cache_write(st["cache"], st["table"], st["k"], st["v"], first=st["first"])
        cache_read(st["cache"], st["table"], st["k_out"], st["v_out"], first=st["start"], length=st["back"])
    elif st["op"] == "attend":
        from moebius_cpu_amd.cache import cache_attention

        cache_attention(st["q"], st["cache"], st["table"], st["out"], scale=st["scale"], causal=c["causal"],
                        window=c["window"], sinks=c["sinks"], q_len=st["q_len"], kv_len=st["kv_len"])
    else:
        from moebius_cpu_amd.gated_norm import gated_norm

        gated_norm(st["x"], branch=st["branch"], post=st["post"], gate=st["gate"], keep=st["keep"], x_out=st["x_out"],
                   pre=st["pre"], scale=st["scale"], shift=st["shift"], y=st["y"])
    return st["view"]


def run(st):
    if own:
        return _run_own(st)
    return {"cache": _plain_cache, "attend": _plain_attend, "norm": _plain_norm}[st["op"]](st, st["case"])


# ---------------------------------------------------------------- the plain forms

def _rows_back(c):
    """Rows that hold the written blocks read back: from the first token of the block that the writing begins in."""
    return c["tokens"] + (min(c["block"] - 1, c["hist"]) if c["hist"] else 0)


def _plain_quantise(x, length, block, codes=None, scale=None, off=None):
    """The codes [n][blocks][block][heads][d] and the scales [n][blocks][heads] of the tokens x [n][tokens][heads][d] below
    length [n], from place off [n] of the first block on, behind the codes [n][block][heads][d] that it holds at its scale."""
    n, tokens, heads, d = x.shape
    off = torch.zeros(n, dtype=torch.int64, device="cuda") if off is None else off.long()
    nb = -(-(tokens + (block - 1 if codes is not None else 0)) // block)
    at = torch.arange(nb * block, device="cuda")[None, :] - off[:, None]  # the token at every place
    new = (at >= 0) & (at < length.long()[:, None])
    x = torch.gather(x, 1, at.clamp(0, tokens - 1)[:, :, None, None].expand(-1, -1, heads, d))
    x = torch.where(new[:, :, None, None], x.float(), 0.0).view(n, nb, block, heads, d)
    s = x.abs().amax((2, 4)) / 127.0
    if codes is not None:
        s[:, 0] = torch.where((off > 0)[:, None], torch.maximum(s[:, 0], scale), s[:, 0])
    by = torch.where(s > 0, s, 1.0).double()[:, :, None, :, None]
    got = torch.round(x.double() / by).clamp(-127, 127).float()
    if codes is not None:
        old = torch.round(codes.double() * scale.double()[:, None, :, None] / by[:, 0])
        got[:, 0] = torch.where((torch.arange(block, device="cuda") < off[:, None])[:, :, None, None], old.float(), got[:, 0])
    return got, s


def _plain_cache(st, c):
    n, b, out = c["n"], c["block"], {}
    length = torch.full((n,), c["tokens"], device="cuda")
    off = st["first"].long() % b
    back = torch.arange(_rows_back(c), device="cuda")[None, :] < (off + c["tokens"])[:, None]
    for name in ("k", "v"):
        codes = scale = None
        if c["hist"]:
            at = (st["first"].long() // b).clamp(max=st[name + "0"][0].shape[1] - 1)
            codes, scale = (t[torch.arange(n, device="cuda"), at] for t in st[name + "0"])
        codes, scale = _plain_quantise(st[name], length, b, codes, scale, off)
        x = (codes * scale[:, :, None, :, None]).flatten(1, 2)
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, max(0, _rows_back(c) - x.shape[1])))[:, :_rows_back(c)]
        out[name] = torch.where(back[:, :, None, None], x, 0.0).to(st[name].dtype)
    return out


def _visible(c, q_len, kv_len):
    """Which keys each query sees [n][q][kv]."""
    i, j = torch.arange(c["q"], device="cuda")[None, :, None], torch.arange(c["kv"], device="cuda")[None, None, :]
    q_len, kv_len = q_len.long()[:, None, None], kv_len.long()[:, None, None]
    at = i + kv_len - q_len
    seen = (j < kv_len) & (i < q_len)
    if c["causal"]:
        seen = seen & (j <= at)
    if c["window"]:
        seen = seen & ((j > at - c["window"]) | (j < c["sinks"]))
    return seen


def _plain_attend(st, c):
    n, hk, d, g = c["n"], c["hk"], c["d"], c["hq"] // c["hk"]
    k, v = ((codes * scale[:, :, None, :, None]).flatten(1, 2)[:, :c["kv"]].transpose(1, 2) for codes, scale in (st["k"], st["v"]))
    q = st["q"].float().view(n, c["q"], hk, g, d).permute(0, 2, 3, 1, 4).reshape(n, hk, g * c["q"], d)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(st["scale"]).view(n, hk, g, c["q"], c["kv"])
    seen = _visible(c, st["q_len"], st["kv_len"])[:, None, None]
    s = torch.where(seen, s, float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    o = torch.matmul(p.view(n, hk, g * c["q"], c["kv"]), v.contiguous()).view(n, hk, g, c["q"], d)
    o = o / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return {"out": o.permute(0, 3, 1, 2, 4).reshape(n, c["q"], c["hq"], d).to(st["q"].dtype)}


def _plain_normed(x, kind, gamma, beta, eps):
    if kind == "none":
        return x
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    if gamma is not None:
        x = x * gamma
    return x if beta is None else x + beta


def _plain_norm(st, c):
    s, out = st["x"].float(), {}
    if c["branch"]:
        h = _plain_normed(st["h"].float(), c["post"], st["g_post"], None, st["eps"])
        s = st["keep"] * s + (h if st["gate"] is None else st["gate"] * h)
        out["x"] = s.to(st["x"].dtype)
    y = _plain_normed(s, c["pre"], st["g_pre"], st["b_pre"], st["eps"])
    if c["mod"]:
        y = y * (1.0 + st["scale"]) + st["shift"]
    return dict(out, y=y.half() if c["h16"] else y)


# ---------------------------------------------------------------- bytes and operations

def _pairs(c):
    """Pairs of a query and a key that it sees, of one head, were all items full; and the keys that any query sees."""
    q, kv = c["q"], c["kv"]
    pairs = 0.0
    window, sinks = c["window"] or kv, c["sinks"]
    for i in (range(q) if q <= 64 else [(q - 1) * f / 63.0 for f in range(64)]):  # linear between: a mean of 64 rows
        at = i + kv - q
        hi = at + 1 if c["causal"] else kv
        lo = max(0, at - window + 1)
        pairs += (hi - lo) + min(lo, sinks)
    first = max(0, kv - q - window + 1)
    return pairs * max(1.0, q / 64.0), kv - first + min(first, sinks)


def work(case):
    c, op = case, case["op"]
    if op == "cache":
        e = 2.0 * c["n"] * c["tokens"] * c["hk"] * c["d"]
        return {"bytes": e * (2 * (2 if c["f16"] else 4) + 2), "flops": 4.0 * e}
    if op == "attend":
        pairs, keys = _pairs(c)
        return {"bytes": 2.0 * c["n"] * keys * c["hk"] * c["d"] + 2.0 * c["n"] * c["q"] * c["hq"] * c["d"] * (2 if c["f16"] else 4),
                "flops": 4.0 * c["n"] * pairs * c["hq"] * c["d"]}
    e = float(c["n"] * c["rows"] * c["c"])
    x, h = 2 if c["x16"] else 4, 2 if c["h16"] else 4
    return {"bytes": e * (x + h + (x + h if c["branch"] else 0)) + (4.0 * c["n"] * c["c"] * 3 if c["mod"] else 0),
            "flops": 12.0 * e}


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_codes(x, held=None, scale=None):
    """Codes of the tokens x [tokens][heads][d] of one block, and of those held before, as [tokens][heads][d], and the
    scales [heads]: the f32 value next to the largest magnitude over 127, or the scale before if that is larger."""
    s = (x.double().abs().amax(0).amax(-1) / 127.0).float().double()
    if held is not None:
        s = torch.maximum(s, scale)
    by = torch.where(s > 0, s, 1.0)[:, None]
    codes = torch.round(x.double() / by)
    if held is not None:
        codes = torch.cat([torch.round(held * scale[:, None] / by), codes])
    return codes, s


def _exact_values(x, block):
    """What a cache holds of the tokens x [tokens][heads][d], in 64 bits."""
    return torch.cat([codes * s[:, None] for codes, s in (_exact_codes(x[lo:lo + block]) for lo in range(0, x.shape[0], block))])


def exact(case, seed):
    c = case
    st = _inputs(c, seed)
    if c["op"] == "cache":
        out, b = {}, c["block"]
        if c["n"] * c["tokens"] > 200_000:
            return None
        for name in ("k", "v"):
            got = torch.zeros((c["n"], _rows_back(c), c["hk"], c["d"]), dtype=torch.float64, device="cuda")
            for i, first in enumerate(st["first"].tolist()):
                off, x, parts = first % b, st[name][i], []
                held = _exact_codes(st[name + "0"][i, first - off:first]) if off else (None, None)
                at = 0
                while at < c["tokens"]:
                    step = min(c["tokens"] - at, b - (off if at == 0 else 0))
                    codes, s = _exact_codes(x[at:at + step], *(held if at == 0 else (None, None)))
                    parts.append(codes * s[:, None])
                    at += step
                got[i, :off + c["tokens"]] = torch.cat(parts)
            out[name] = got
        return out
    if c["op"] == "attend":
        g = c["hq"] // c["hk"]
        out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
        for i, (ql, kl) in enumerate(zip(st["q_len"].tolist(), st["kv_len"].tolist())):
            k, v = _exact_values(st["k"][i, :kl], c["block"]), _exact_values(st["v"][i, :kl], c["block"])
            at = torch.arange(kl - ql, kl, device="cuda")[:, None]
            j = torch.arange(kl, device="cuda")[None, :]
            hidden = j > (at if c["causal"] else kl)
            if c["window"]:
                hidden = hidden | ((at - j >= c["window"]) & (j >= c["sinks"]))
            for h in range(c["hq"]):
                s = torch.matmul(st["q"][i, :ql, h].double(), k[:, h // g].t().contiguous()) * st["scale"]
                out[i, :ql, h] = torch.matmul(torch.softmax(s.masked_fill_(hidden, -math.inf), -1), v[:, h // g].contiguous())
        return {"out": out}

    def normed(x, kind, gamma, beta):
        if kind == "none":
            return x
        if kind == "layer":
            x = (x - x.mean(-1, keepdim=True)) / torch.sqrt(x.var(-1, unbiased=False, keepdim=True) + st["eps"])
        else:
            x = x / torch.sqrt(torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / c["c"] + st["eps"])
        x = x if gamma is None else x * gamma.double()
        return x if beta is None else x + beta.double()

    out, s = {}, st["x"].double()
    if c["branch"]:
        h = normed(st["h"].double(), c["post"], st["g_post"], None)
        out["x"] = s = s * st["keep"] + (h * st["gate"].double() if c["mod"] else h)
    y = normed(s, c["pre"], st["g_pre"], st["b_pre"])
    out["y"] = y + y * st["scale"].double() + st["shift"].double() if c["mod"] else y
    return out
