"""Steps in which single tokens and chunks meet: a chunk, whose rows go to the kernel of many,
leaves the tokens' outputs bit for bit what they are without it; and chunks by plans set from
the host and built on the GPU."""
import numpy as np
import pytest

from test_gpu_paged import Cache, Rows, queries
from test_gpu_paged_build import ALL, Built, every_type  # noqa: F401
from xwfes_amd import ftx

pytestmark = pytest.mark.gpu


@ALL
@pytest.mark.parametrize("hd,kv,heads,few,chunk,window", [
    # lists that stay whole, that are split, of 8 rows, under a window
    (128, 8, 32, [(37 * s + 20, 1) for s in range(16)], (300, 40), 0),
    (128, 8, 32, [(8000, 1), (2900, 1)], (64, 33), 0),
    (128, 2, 8, [(700, 2), (70, 1), (0, 2)], (0, 128), 0),
    (64, 2, 16, [(1500, 1), (63, 1), (64, 1)], (10, 20), 0),
    (64, 4, 16, [(900, 1), (10, 1)], (500, 64), 200)])
def test_single_tokens_beside_a_chunk(gctx, kvt, hd, kv, heads, few, chunk, window):
    rng = np.random.default_rng(hd + heads + len(few))
    force = ftx.load().paged_force_rows
    force(128)
    try:
        c = Cache(gctx, rng, kvt, hd, kv, heads, few[:1] + [chunk] + few[1:], window, 4 if window else 0)
        c.write_new()
        q = queries(rng, c, 2.0)
        got = c.check(q)
        m, n = few[0][1], few[0][1] + chunk[1]
        alone = c.pool.plan(c.seqs[:1] + c.seqs[2:], heads, window, 4 if window else 0)
        pick = lambda x: np.concatenate([x[:m], x[n:]])  # noqa: E731
        qd, out = Rows(gctx, pick(q)), Rows(gctx, pick(q) * 0)
        alone.attend(0, qd.ptr, out.ptr)
        gctx.sync()
        np.testing.assert_array_equal(pick(got), out.get().reshape(-1, heads, hd))
    finally:
        force(0)
    for x in (qd, out):
        x.buf.free()
    alone.free(), c.free()


@ALL
@pytest.mark.parametrize("hd,kv,heads,seqs", [
    (128, 2, 8, [(0, 100), (20, 40), (3, 1)]), (64, 1, 16, [(1, 5), (60, 64), (0, 128)]), (256, 1, 4, [(9, 90), (0, 0), (5, 17)])])
def test_chunks_in_plans_built_on_the_gpu(gctx, kvt, hd, kv, heads, seqs):
    """Chunks over lists that neither plan splits: bit for bit what a plan set from the host gives
    by row tiles of the same size."""
    rng = np.random.default_rng(hd)
    force = ftx.load().paged_force_rows
    c = Built(gctx, rng, kvt, hd, kv, heads, seqs)
    c.write_new()
    q = queries(rng, c, 2.0)
    got = c.check(q)
    force(128)
    try:
        host = c.pool.plan(c.seqs, heads)
    finally:
        force(0)
    qd, out = Rows(gctx, q), Rows(gctx, q * 0)
    host.attend(0, qd.ptr, out.ptr)
    gctx.sync()
    want, at = out.get().reshape(-1, heads, hd), 0
    for _, m in seqs:
        if m * heads // kv > 64:
            np.testing.assert_array_equal(got[at:at + m], want[at:at + m])
        at += m
    for x in (qd, out):
        x.buf.free()
    host.free(), c.free()
