"""Captured calls of a plan whose tables went up on the captured stream itself,
behind work there, with the graph launched on another stream: the graph holds no
copy of the tables, so they must be there when the capture ends."""
import ctypes

import numpy as np
import pytest

from test_gpu_paged import Q8, TYPES, Cache, Rows, queries, refused
from test_zz_no_alloc import _hip

pytestmark = pytest.mark.gpu


@TYPES
@pytest.mark.parametrize("mode", [0, 1, 2], ids=["global", "thread", "relaxed"])
def test_set_and_captured_on_one_stream_launched_on_another(gctx, kvt, mode):
    hip = _hip()
    rng = np.random.default_rng(33)
    busy = Cache(gctx, rng, Q8, 128, 2, 8, [(3000, 500)])
    busy.write_new()
    bq, bo = Rows(gctx, queries(rng, busy)), Rows(gctx, np.zeros((busy.new, busy.heads * busy.hd), np.float32))
    c = Cache(gctx, rng, kvt, 128, 2, 8, [(900, 3), (200, 40)])
    c.write_new()
    q = queries(rng, c)
    want = c.check(q)
    qd, out = Rows(gctx, q), Rows(gctx, np.zeros_like(q))
    a, b = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamCreate(ctypes.byref(a)) == 0 and hip.hipStreamCreate(ctypes.byref(b)) == 0
    held = []
    try:
        for _ in range(3):
            graph, exe = ctypes.c_void_p(), ctypes.c_void_p()
            out.buf.write(out.host)
            # other sequences first: a stale table would show
            plan = c.pool.plan([(t[::-1], n, m, None) for t, n, m, _ in c.seqs], 8)
            gctx.sync()
            gctx.set_stream(a.value)
            for _ in range(60):
                busy.plan.attend(0, bq.ptr, bo.ptr)
            plan.set(c.seqs, 8)
            assert hip.hipStreamBeginCapture(a, mode) == 0
            plan.attend(0, qd.ptr, out.ptr)
            plan.attend(0, qd.ptr, out.ptr)
            assert hip.hipStreamEndCapture(a, ctypes.byref(graph)) == 0
            gctx.set_stream(None)
            held.append((plan, graph, exe))
            assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0) == 0
            for _ in range(2):
                assert hip.hipGraphLaunch(exe, b) == 0
            assert hip.hipStreamSynchronize(b) == 0
            np.testing.assert_array_equal(out.get().reshape(want.shape), want)
            assert hip.hipStreamSynchronize(a) == 0
    finally:
        gctx.set_stream(None)
        for st in (a, b):
            hip.hipStreamSynchronize(st)
        for plan, graph, exe in held:
            if exe:
                hip.hipGraphExecDestroy(exe)
            hip.hipGraphDestroy(graph)
            plan.free()
        for st in (a, b):
            hip.hipStreamDestroy(st)
    for x in (bq, bo, qd, out):
        x.buf.free()
    c.free()
    busy.free()


def test_refused_calls_of_a_capture_leave_the_plan_free(gctx):
    """A plan none of whose calls was recorded can be set again."""
    hip = _hip()
    c = Cache(gctx, np.random.default_rng(34), Q8, 64, 1, 2, [(70, 5)])
    c.write_new()
    far = c.pool.plan([([-1, c.tables[0][1]], 70, 5)], 2, 3)
    m = Rows(gctx, np.zeros((5, 4 * 128)))
    st, graph = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamCreate(ctypes.byref(st)) == 0
    gctx.set_stream(st.value)
    try:
        assert hip.hipStreamBeginCapture(st, 2) == 0
        refused(-1, c.plan.attend, 0, m.ptr, m.ptr)
        refused(-1, c.plan.read, 0, m.ptr, m.ptr)
        refused(-5, far.read, 0, m.ptr, m.ptr + 4 * 256, True, 512, 512)
        assert hip.hipStreamEndCapture(st, ctypes.byref(graph)) == 0
    finally:
        gctx.set_stream(None)
        if graph.value:
            hip.hipGraphDestroy(graph)
        hip.hipStreamDestroy(st)
    c.plan.set(c.seqs, 2)
    far.set(c.seqs, 2)
    c.check(queries(np.random.default_rng(35), c))
    m.buf.free()
    far.free()
    c.free()
