"""Low-rank adapters of many requests beside a shared 1x1 projection
(include/moebius_hip.h mh_conv1x1_lora; Conv1x1.forward_adapted)."""
from __future__ import annotations

import ctypes

from . import _lib
from ._lib import MoebiusError, check, lib
from .engine import Context, Param, _vec


class Adapters:
    """a [slots, rank, c_in], b [slots, c_out, rank] (Params of one storage type) and scale [slots]
    of a projection [c_out, c_in]; an adapter of lower rank fills the rest with zeros."""

    def __init__(self, ctx: Context, a: Param, b: Param, scale, c_in: int, c_out: int, rank: int):
        self.ctx, self.a, self.b, self.scale = ctx, a, b, _vec(ctx, scale)
        self.c_in, self.c_out, self.rank, self.slots = c_in, c_out, rank, self.scale.nbytes // 4
        if a.dtype != b.dtype:
            raise MoebiusError(1, "adapters differ in storage type")
        if len(a) != self.slots * rank * c_in or len(b) != self.slots * c_out * rank:
            raise MoebiusError(1, "adapter size")
        self.c = _lib.AdapterSet(a.ptr, b.ptr, self.scale.ptr, a.dtype, self.slots, rank, 0)

    def scratch(self, rows: int, weight: Param) -> int:
        """Bytes of scratch that a call over `rows` rows of a projection by `weight` needs, for calls
        that are captured into a graph."""
        n = ctypes.c_uint64()
        check(lib().mh_conv1x1_lora_scratch(self.ctx.h, rows, self.c_in, self.c_out, weight.dtype, self.rank,
                                            ctypes.byref(n)))
        return int(n.value)
