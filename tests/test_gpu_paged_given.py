"""A paged cache shows the rows that it was given, never what its pages held for
another: reads past the last new tokens are zeros, and a length or a path that
reaches past them is refused."""
import numpy as np
import pytest

from test_gpu_paged import F16, Q8, refused
from test_gpu_paged_steps import CFG64, Setup
from test_gpu_paged_steps import Q8 as Q8_0

pytestmark = pytest.mark.gpu


@pytest.fixture
def setup(gctx, orc, request):
    t = Setup(gctx, orc, CFG64, Q8_0, kvt=request.param, pages=4)
    # both pages of the pool's first take, full of another cache's rows
    other = t.gm.kv_paged(t.pool, 256)
    other.write(*np.full((2,) + other.shape, 5.0, np.float32))
    other.free()
    yield t
    t.free()


KINDS = pytest.mark.parametrize("setup", [F16, Q8], ids=["f16", "q8"], indirect=True)


@KINDS
@pytest.mark.parametrize("M", [1, 9, 64, 70])
def test_rows_past_the_new_tokens_read_zero(setup, M):
    kv = setup.gm.kv_paged(setup.pool, 200)
    setup.kvs.append(kv)
    toks = list(range(M))
    setup.step([(kv, toks, None, True)])
    for x in kv.read():
        assert x[:, :M].any((0, 2)).all() and not x[:, M:].any()
    # tokens that were not committed are the cache's own
    setup.step([(kv, [7, 8, 9], None, False)])
    for x in kv.read():
        assert x[:, :M + 3].any((0, 2)).all() and not x[:, M + 3:].any()


@KINDS
def test_lengths_and_paths_past_the_new_tokens_are_refused(setup):
    kv = setup.gm.kv_paged(setup.pool, 200)
    setup.kvs.append(kv)
    refused(-5, kv.truncate, 1)
    setup.step([(kv, [1, 2, 3, 4], [-1, 0, 0, 1], False)])
    refused(-5, kv.truncate, 5)
    refused(-5, kv.commit, [0, 4])
    kv.commit([0, 2])
    assert kv.pointers()[2] == 2
    refused(-5, kv.truncate, 5)
    kv.truncate(4)
    kv.truncate(0)
    assert setup.pool.available == 4
    # pages taken anew hold nothing of it
    setup.step([(kv, [1], None, False)])
    refused(-5, kv.truncate, 2)
    for x in kv.read():
        assert x[:, :1].any() and not x[:, 1:].any()


@KINDS
def test_a_refused_step_gives_nothing(setup):
    kv, hog = (setup.gm.kv_paged(setup.pool, 256) for _ in range(2))
    setup.kvs += [kv, hog]
    setup.step([(kv, [1, 2], None, True)])
    refused(-4, setup.step, [(kv, [5] * 70, None, False), (hog, [6] * 180, None, False)])
    refused(-5, kv.truncate, 3)
    for x in kv.read():
        assert x[:, :2].any((0, 2)).all() and not x[:, 2:].any()


@KINDS
def test_a_written_cache_is_given_all_of_its_rows(setup):
    kv = setup.gm.kv_paged(setup.pool, 100)
    setup.kvs.append(kv)
    k, v = np.random.default_rng(1).standard_normal((2,) + kv.shape).astype(np.float32)
    kv.write(k, v)
    assert all(x.any((0, 2)).all() for x in kv.read())
    kv.truncate(99)
    setup.step([(kv, [3], None, True)])
    refused(-5, kv.truncate, 101)
    kv.truncate(10)
    # the rest of the page that length ends in is still its own
    kv.truncate(64)
    refused(-5, kv.truncate, 65)
    for x in kv.read():
        assert x[:, :64].any((0, 2)).all() and not x[:, 64:].any()


def test_pools_past_64_bits_are_refused(gctx):
    """Sizes whose product of bytes comes round to some 6 MB in 64 bits."""
    for layers, kv, pages in ((36359, 900, 8535041), (45133, 709, 8728098)):
        assert (layers * kv * pages * (4 * 64 * 256 + 8 * 64)) % 2 ** 64 < 10 ** 7
        refused(-4, gctx.pool, layers, kv, 256, pages, F16)
    refused(-4, gctx.pool, 65535, 1024, 256, 1 << 24, F16)
    gctx.pool(3, 2, 256, 5, F16).free()


@KINDS
@pytest.mark.parametrize("window", [0, 70])
def test_a_refused_write_leaves_the_cache_as_it_was(gctx, setup, window):
    """A write that its plan refuses (the stream is being captured): the cache's
    rows, length and pages, and the pool's, are those before."""
    import ctypes

    from test_zz_no_alloc import _hip

    hip = _hip()
    kv = setup.gm.kv_paged(setup.pool, 250, window=window)
    setup.kvs.append(kv)
    for n in (100, 60):
        setup.step([(kv, [(7 * i) % 300 for i in range(n)], None, True)])
    before, free = kv.read(), setup.pool.available
    rows = np.full((2,) + kv.shape, 3.0, np.float32)
    st, graph = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamCreate(ctypes.byref(st)) == 0
    gctx.set_stream(st.value)
    try:
        assert hip.hipStreamBeginCapture(st, 2) == 0
        refused(-1, kv.write, *rows)
        assert hip.hipStreamEndCapture(st, ctypes.byref(graph)) == 0
    finally:
        gctx.set_stream(None)
        if graph.value:
            hip.hipGraphDestroy(graph)
        hip.hipStreamDestroy(st)
    assert setup.pool.available == free and kv.pointers()[2] == 160
    for x, y in zip(kv.read(), before):
        np.testing.assert_array_equal(x, y)
    setup.step([(kv, [5], None, False)])
    kv.write(*rows)
    assert setup.pool.available == 0 and all((x != 0).all() for x in kv.read())


@KINDS
@pytest.mark.parametrize("M", [1, 30])
def test_a_step_that_its_plan_refuses_takes_no_pages(gctx, setup, M):
    import ctypes

    from test_zz_no_alloc import _hip

    hip = _hip()
    kv = setup.gm.kv_paged(setup.pool, 200)
    setup.kvs.append(kv)
    setup.step([(kv, [1] * 64, None, True)])
    before = kv.read()
    buf = gctx.buffer(M * CFG64["vocab"] * 4)
    st, graph = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamCreate(ctypes.byref(st)) == 0
    gctx.set_stream(st.value)
    try:
        assert hip.hipStreamBeginCapture(st, 2) == 0
        refused(-1, setup.gm.verify, kv, [2] * M, buf.ptr)
        assert hip.hipStreamEndCapture(st, ctypes.byref(graph)) == 0
    finally:
        gctx.set_stream(None)
        if graph.value:
            hip.hipGraphDestroy(graph)
        hip.hipStreamDestroy(st)
    assert setup.pool.available == 3 and kv.pointers()[2] == 64
    for x, y in zip(kv.read(), before):
        np.testing.assert_array_equal(x, y)
    setup.step([(kv, [2] * M, None, True)])
    assert setup.pool.available == 2
    buf.free()


@KINDS
def test_one_window_over_caches_of_two_sizes(setup):
    """More first tokens than one cache can hold: one window, sinks and step."""
    a, b = (setup.gm.kv_paged(setup.pool, cap, window=8, sinks=100) for cap in (40, 150))
    whole = setup.gm.kv_paged(setup.pool, 40)
    setup.kvs += [a, b, whole]
    toks = list(range(30))
    got = setup.step([(a, toks, None, True), (b, toks, None, True)])
    np.testing.assert_array_equal(got[0], got[1])
    # every position is one of the first 100: no window
    np.testing.assert_array_equal(setup.step([(whole, toks, None, True), ])[0], got[0])
    far = setup.gm.kv_paged(setup.pool, 150, window=8, sinks=1 << 40)
    setup.kvs.append(far)
    np.testing.assert_array_equal(setup.step([(far, toks, None, True)])[0], got[0])
