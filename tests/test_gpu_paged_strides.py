"""Strided and unaligned rows where the kernels of many rows and the joins read
and write them: bit for bit what dense rows give."""
import numpy as np
import pytest

from test_gpu_paged import F16, TYPES, Cache, Rows, queries
from test_paged_plan import probe

pytestmark = pytest.mark.gpu

WAYS = [(4, 4), (3, 0), (0, 1), (8, 2), (1, 3), (64, 0)]


def made(ctx, kvt, hd, kv, heads, seqs, rows):
    ctx.lib.paged_force_rows(rows)
    try:
        c = Cache(ctx, np.random.default_rng(15), kvt, hd, kv, heads, seqs)
        _, _, items, joins = probe(c.seqs, kv, heads, n_pages=10 ** 4, hd=hd)
    finally:
        ctx.lib.paged_force_rows(0)
    return c, items, joins


@TYPES
@pytest.mark.parametrize("hd,kv,heads,seqs,rows", [
    (64, 2, 6, [(80, 40), (1, 30)], 128), (64, 2, 6, [(80, 40), (1, 300)], 256), (128, 1, 8, [(100, 70)], 256),
    (128, 2, 2, [(100, 70), (30, 140)], 128), (256, 1, 4, [(70, 50)], 128)])
def test_many_rows(gctx, kvt, hd, kv, heads, seqs, rows):
    c, items, _ = made(gctx, kvt, hd, kv, heads, seqs, rows)
    assert (items[:, 7] > 0).all()
    c.write_new()
    q = queries(np.random.default_rng(1), c)
    want = c.check(q)
    for pad, off in WAYS:
        c.write_new(pad=pad, off=off)
        np.testing.assert_array_equal(c.attend(q, pad=pad, off=off), want)
    c.free()


@TYPES
@pytest.mark.parametrize("hd,kv,heads,seqs,rows,parts", [
    (64, 1, 4, [(1500, 1)], 0, (2, 8)), (128, 1, 4, [(3000, 3), (900, 1)], 0, (9, 999)), (256, 1, 3, [(800, 2)], 0, (2, 8)),
    (256, 1, 3, [(2600, 2)], 0, (9, 999)), (64, 1, 2, [(2000, 90)], 128, (9, 999)), (64, 1, 2, [(700, 90)], 128, (2, 8)), (128, 1, 4, [(3000, 90)], 256, (9, 999)),
    (256, 1, 2, [(2000, 50)], 128, (2, 999)), (128, 1, 2, [(2500, 60)], 16, (2, 999))])
def test_joins(gctx, kvt, hd, kv, heads, seqs, rows, parts):
    c, items, joins = made(gctx, kvt, hd, kv, heads, seqs, rows)
    assert len(joins) and parts[0] <= joins[:, 3].max() <= parts[1], joins[:, 3].max(initial=0)
    c.write_new()
    q = queries(np.random.default_rng(2), c)
    want = c.check(q)
    for pad, off in WAYS:
        np.testing.assert_array_equal(c.attend(q, pad=pad, off=off), want)
    c.free()


@pytest.mark.parametrize("rows", [128, 256])
def test_many_rows_of_q_k_v_in_one_matrix(gctx, rows):
    """Rows of q | k | v as a projection leaves them, out in their padding."""
    c, items, _ = made(gctx, F16, 64, 2, 4, [(10, 90)], rows)
    assert (items[:, 7] > 0).all()
    q = queries(np.random.default_rng(3), c)
    w = (4 + 2 + 2) * 64
    m = Rows(gctx, np.concatenate([q, c.k[0][10:].reshape(90, -1), c.v[0][10:].reshape(90, -1)], 1), 256)
    c.plan.write(0, m.ptr + 4 * 256, m.ptr + 4 * 384, m.ld, m.ld)
    c.plan.attend(0, m.ptr, m.ptr + 4 * w, m.ld, m.ld)
    gctx.sync()
    got = m.buf.read(np.float32, m.host.size)[:90 * m.ld].reshape(90, m.ld)[:, w:w + 256].reshape(90, 4, 64)
    np.testing.assert_array_equal(got, c.check(q))
    m.buf.free()
    c.free()
