"""The gated residual of a branch and the modulated norm of the sum, in one pass
(include/moebius_hip.h mh_gated_norm); the reference has no counterpart.

    pre = Norm("layer", eps=1e-6)
    gated_norm(x, pre=pre, scale=scale_1, shift=shift_1, y=y)                          # before a block
    gated_norm(x, branch=h, gate=gate_1, x_out=x, pre=pre, scale=scale_2, shift=shift_2, y=y)  # between two
    gated_norm(x, branch=h, gate=gate_2, x_out=x)                                      # behind the last
"""
from __future__ import annotations

import struct

import numpy as np

from . import _lib
from ._lib import MoebiusError, check, lib
from .attention import Heads
from .engine import DeviceArray

_F32 = np.dtype(np.float32)
# _lib.GatedNorm, packed: a call of few rows takes no longer on the device than here.
_PACK = struct.Struct("=4Q4Q2I2QIfIf2QIf2Q3Q3Q").pack


class Norm:
    """"none", "rms" or "layer" over the channels of a row, with gamma and beta [c] f32 (None: 1 and 0)."""

    def __init__(self, kind: str = "none", gamma: DeviceArray | None = None, beta: DeviceArray | None = None,
                 eps: float = 1e-6):
        if kind not in _lib.NORM:
            raise MoebiusError(1, f"unknown norm {kind!r}")
        for a in (gamma, beta):
            if a is not None and a.dtype != _F32:
                raise MoebiusError(1, "gamma and beta are f32 of the row's channels")
        self.gamma, self.beta = gamma, beta
        self._c = None if gamma is None and beta is None else (gamma if beta is None else beta).nbytes // 4
        if gamma is not None and beta is not None and gamma.nbytes != beta.nbytes:
            raise MoebiusError(1, "gamma and beta are f32 of the row's channels")
        self._args = (_lib.NORM[kind], float(eps), 0 if gamma is None else gamma.ptr, 0 if beta is None else beta.ptr)


_NONE = Norm()


def gated_norm(x: Heads, branch: Heads | None = None, post: Norm | None = None, gate: Heads | None = None,
               keep: float = 1.0, x_out: Heads | None = None, pre: Norm | None = None, scale: Heads | None = None,
               shift: Heads | None = None, y: Heads | None = None):
    """s = keep x + gate post(branch) (no branch: s = x), x_out = s, y = pre(s) (1 + scale) + shift, over rows
    of all heads * d channels of x. gate, scale and shift: f32 views of one row [1, c] per item. x_out has
    x's type, y the branch's; an output may be an input of its type."""
    ctx, n, tokens, c = x.ctx, x.n, x.tokens, x.heads * x.d
    bp = bl = op = ol = yp = yl = gp = gl = sp = sl = hp = hl = 0
    code = x.code
    if y is not None:
        yp, yl, code = y.buf.ptr + y._offset, y.ld, y.code
        if y.n != n or y.tokens != tokens or y.heads * y.d != c:
            raise MoebiusError(1, "x, branch, x_out and y differ in shape")
        if y.ctx is not ctx:
            raise MoebiusError(1, "rows of different contexts")
    if branch is not None:
        bp, bl = branch.buf.ptr + branch._offset, branch.ld
        if branch.n != n or branch.tokens != tokens or branch.heads * branch.d != c:
            raise MoebiusError(1, "x, branch, x_out and y differ in shape")
        if branch.ctx is not ctx:
            raise MoebiusError(1, "rows of different contexts")
        if y is not None and branch.code != code:
            raise MoebiusError(1, "branch and y differ in type")
        code = branch.code
    if x_out is not None:
        op, ol = x_out.buf.ptr + x_out._offset, x_out.ld
        if x_out.n != n or x_out.tokens != tokens or x_out.heads * x_out.d != c:
            raise MoebiusError(1, "x, branch, x_out and y differ in shape")
        if x_out.ctx is not ctx:
            raise MoebiusError(1, "rows of different contexts")
        if x_out.code != x.code:
            raise MoebiusError(1, "x and x_out differ in type")
    if gate is not None:
        gp, gl = _vector(gate, n, c, ctx)
    if scale is not None:
        sp, sl = _vector(scale, n, c, ctx)
    if shift is not None:
        hp, hl = _vector(shift, n, c, ctx)
    post = _NONE if post is None else post
    pre = _NONE if pre is None else pre
    if (post._c is not None and post._c != c) or (pre._c is not None and pre._c != c):
        raise MoebiusError(1, "gamma and beta are f32 of the row's channels")
    st = lib().mh_gated_norm(ctx.h, _PACK(x.buf.ptr + x._offset, bp, op, yp, x.ld, bl, ol, yl, x.code, code, n * tokens,
                                          tokens or 1, c, keep, *post._args, *pre._args, gp, sp, hp, gl, sl, hl))
    if st:
        check(st)


def _vector(a, n, c, ctx):
    if a.n != n or a.tokens != 1 or a.heads * a.d != c or a.code != _lib.DTYPE_F32:
        raise MoebiusError(1, "gate, scale and shift are f32 [n, 1, c]")
    if a.ctx is not ctx:
        raise MoebiusError(1, "rows of different contexts")
    return a.buf.ptr + a._offset, a.ld
