"""Plans built on the GPU: calls that test_gpu_paged_build.py does not make."""
import contextlib
import ctypes

import numpy as np
import pytest

from test_gpu_paged import Q8, Cache, Rows, queries, refused
from test_gpu_paged_build import I32, Built, Lists, every_type  # noqa: F401
from test_gpu_paged_q4 import Q4
from test_zz_no_alloc import _hip

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("spread", [0, 1], ids=["one", "many"])
def test_pages_of_sequences_without_new_tokens_under_a_window(gctx, spread):
    """No new token sees them: they may be absent, as they may in plans set from the host.  By the
    kernel of one workgroup, and (among many sequences of nothing) by those of several."""
    n = 3 + 3000 * spread
    pool = gctx.pool(1, 1, 64, 16, Q8)
    pool.take(16)
    tables = np.full((n, 6), -1, I32)
    tables[1, 3:5] = 3, 4
    for window, sinks, M, code in ((70, 0, 2, 0), (70, 65, 0, 0), (1 << 20, 0, 0, 0), (0, 0, 0, -1)):
        plan = pool.device_plan(n, 4, 4, 6, 2, window=window, sinks=sinks)
        ls = Lists(gctx, [300] * 3 + [0] * (n - 3), [0, M, 0] + [0] * (n - 3), tables, [9], 0, 4)
        ls.build(plan)
        if code:
            ls.refused(code)
        else:
            ls.check()
        ls.free(), plan.free()
    host = pool.plan([([-1] * 5, 300, 0), ([-1, -1, -1, 3, 4], 300, 2)], 2, 70)
    host.free()
    pool.free()


@contextlib.contextmanager
def streams(ctx, n):
    """n streams; in the end the context is on its own again."""
    hip, st = _hip(), [ctypes.c_void_p() for _ in range(n)]
    for x in st:
        assert hip.hipStreamCreate(ctypes.byref(x)) == 0
    try:
        yield hip, st
    finally:
        ctx.set_stream(None)
        for x in st:
            hip.hipStreamSynchronize(x)
            hip.hipStreamDestroy(x)


@contextlib.contextmanager
def captured(hip, st, mode):
    """A capture of a stream that has to end as one that nothing broke."""
    graph = ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(st, mode) == 0
    try:
        yield
    finally:
        rc = hip.hipStreamEndCapture(st, ctypes.byref(graph))
        if graph:
            hip.hipGraphDestroy(graph)
    assert rc == 0


def test_another_stream_while_one_is_captured(gctx):
    """A build and calls go from stream to stream while a stream that has nothing to do with them
    is being captured in the global mode: they are not refused and the capture stays whole."""
    rng = np.random.default_rng(51)
    c = Built(gctx, rng, Q4, 128, 2, 8, [(900, 3)])
    c.write_new()
    q = queries(rng, c)
    want = c.check(q)
    none = Lists(gctx, [0], [0], c.lists.host["tables"], [], 0, c.room)
    qd, out = Rows(gctx, c.pad(q, np.nan)), Rows(gctx, np.full((c.room, c.heads * c.hd), 9.0))
    with streams(gctx, 2) as (hip, (other, taken)):
        for rep in range(3):
            out.buf.write(out.host)
            none.build(c.plan)
            gctx.sync()
            with captured(hip, taken, 0):
                c.lists.build(c.plan)
                gctx.set_stream(other.value)
                c.plan.attend(0, qd.ptr, out.ptr)
                gctx.set_stream(None)
                none.build(c.plan)
                gctx.set_stream(other.value)
                none.build(c.plan)
                gctx.set_stream(None)
            assert hip.hipStreamSynchronize(other) == 0
            gctx.sync()
            np.testing.assert_array_equal(out.get()[:c.new].reshape(want.shape), want)
    for x in (qd, out):
        x.buf.free()
    none.free(), c.free()


def test_the_stream_of_the_last_call_is_captured(gctx):
    """Left before its capture: another stream waits for what was on it.  Left within it: a call on
    another stream is refused until the capture has ended, and the capture stays whole."""
    rng = np.random.default_rng(52)
    busy = Cache(gctx, rng, Q8, 128, 2, 8, [(3000, 500)])
    busy.write_new()
    bq, bo = Rows(gctx, queries(rng, busy)), Rows(gctx, np.zeros((busy.new, busy.heads * busy.hd), np.float32))
    c = Built(gctx, rng, Q4, 64, 2, 8, [(500, 2), (70, 1)])
    c.write_new()
    q = queries(rng, c)
    want = c.check(q)
    none = Lists(gctx, [0, 0], [0, 0], c.lists.host["tables"], [], 0, c.room)
    qd, out = Rows(gctx, c.pad(q, np.nan)), Rows(gctx, np.full((c.room, c.heads * c.hd), 9.0))

    def work():
        none.build(c.plan)
        for _ in range(20):
            busy.plan.attend(0, bq.ptr, bo.ptr)
        c.lists.build(c.plan)

    def held(st):
        assert hip.hipStreamSynchronize(st) == 0
        np.testing.assert_array_equal(out.get()[:c.new].reshape(want.shape), want)
        out.buf.write(out.host)

    with streams(gctx, 2) as (hip, (st, other)):
        gctx.set_stream(st.value)
        work()
        gctx.set_stream(other.value)
        with captured(hip, st, 2):
            c.plan.attend(0, qd.ptr, out.ptr)
        held(other)
        gctx.set_stream(st.value)
        work()
        with captured(hip, st, 2):
            refused(-1, c.plan.attend, 0, qd.ptr, out.ptr)
            gctx.set_stream(other.value)
            refused(-1, c.plan.attend, 0, qd.ptr, out.ptr)
            refused(-1, none.build, c.plan)
            gctx.set_stream(None)
        gctx.set_stream(other.value)
        c.plan.attend(0, qd.ptr, out.ptr)
        held(other)
    for x in (bq, bo, qd, out):
        x.buf.free()
    none.free(), c.free(), busy.free()
