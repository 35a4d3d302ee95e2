"""Calls on a context's stream captured into a graph."""
from __future__ import annotations

import ctypes

from moebius_cpu_amd import _lib


def capture(ctx, calls):
    """(launch, destroy) of the calls captured from the context's stream; where one of them raises,
    what was captured before it is dropped and the error goes on."""
    hip = ctypes.CDLL("libamdhip64.so")
    stream = ctypes.c_void_p(_lib.lib().mh_context_stream(ctx.h))
    graph, run = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 2) == 0  # relaxed
    try:
        calls()
    except BaseException:
        hip.hipStreamEndCapture(stream, ctypes.byref(graph))
        if graph:
            hip.hipGraphDestroy(graph)
        raise
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, 0) == 0

    def launch():
        assert hip.hipGraphLaunch(run, stream) == 0

    return launch, lambda: (hip.hipGraphExecDestroy(run), hip.hipGraphDestroy(graph))
