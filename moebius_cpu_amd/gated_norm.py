"""The gated residual of a branch and the modulated norm of the sum, in one pass
(include/moebius_hip.h mh_gated_norm); the reference has no counterpart.

    pre = Norm("layer", eps=1e-6)
    gated_norm(x, pre=pre, scale=scale_1, shift=shift_1, y=y)                          # before a block
    gated_norm(x, branch=h, gate=gate_1, x_out=x, pre=pre, scale=scale_2, shift=shift_2, y=y)  # between two
    gated_norm(x, branch=h, gate=gate_2, x_out=x)                                      # behind the last
"""
from __future__ import annotations

import ctypes

import numpy as np

from . import _lib
from ._lib import MoebiusError, check, lib
from .attention import Heads
from .engine import DeviceArray, _ptr

_F32 = np.dtype(np.float32)


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
        self.c = _lib.Norm(_lib.NORM[kind], float(eps), _ptr(gamma), _ptr(beta))

    def _of(self, c):
        for a in (self.gamma, self.beta):
            if a is not None and a.nbytes != 4 * c:
                raise MoebiusError(1, "gamma and beta are f32 of the row's channels")
        return self.c


_NONE = Norm()


def gated_norm(x: Heads, branch: Heads | None = None, post: Norm | None = None, gate: Heads | None = None,
               keep: float = 1.0, x_out: Heads | None = None, pre: Norm | None = None, scale: Heads | None = None,
               shift: Heads | None = None, y: Heads | None = None):
    """s = keep x + gate post(branch) (no branch: s = x), x_out = s, y = pre(s) (1 + scale) + shift, over rows
    of all heads * d channels of x. gate, scale and shift: f32 views of one row [1, c] per item. x_out has
    x's type, y the branch's; an output may be an input of its type."""
    n, rows, c = x.n, x.rows, x.heads * x.d
    for a in (branch, x_out, y):
        if a is None:
            continue
        if (a.n, a.tokens, a.heads * a.d) != (n, x.tokens, c):
            raise MoebiusError(1, "x, branch, x_out and y differ in shape")
        if a.ctx is not x.ctx:
            raise MoebiusError(1, "rows of different contexts")
    if x_out is not None and x_out.code != x.code:
        raise MoebiusError(1, "x and x_out differ in type")
    if branch is not None and y is not None and branch.code != y.code:
        raise MoebiusError(1, "branch and y differ in type")
    for a in (gate, scale, shift):
        if a is not None and ((a.n, a.tokens, a.heads * a.d) != (n, 1, c) or a.code != _lib.DTYPE_F32):
            raise MoebiusError(1, "gate, scale and shift are f32 [n, 1, c]")
    other = branch if branch is not None else y

    def at(a):
        return (None, 0) if a is None else (a.ptr, a.ld)

    (bp, bl), (xp, xl), (yp, yl) = at(branch), at(x_out), at(y)
    (gp, gl), (sp, sl), (hp, hl) = at(gate), at(scale), at(shift)
    st = lib().mh_gated_norm(x.ctx.h, ctypes.byref(_lib.GatedNorm(
        x.ptr, bp, xp, yp, x.ld, bl, xl, yl, x.code, x.code if other is None else other.code, rows, max(x.tokens, 1), c,
        float(keep), (post or _NONE)._of(c), (pre or _NONE)._of(c), gp, sp, hp, gl, sl, hl)))
    if st:
        check(st)
