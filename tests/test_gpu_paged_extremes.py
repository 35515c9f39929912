"""Paged attention at the ends of its ranges: the last positions, the most
sequences, many query heads for a kv head and many kv heads."""
import numpy as np
import pytest

from test_gpu_paged import F16, Q8, TILES, TYPES, Cache, Rows, queries, stored, tiles, tree  # noqa: F401

pytestmark = pytest.mark.gpu


@TILES
@TYPES
@pytest.mark.parametrize("M,sinks,branches", [(1, 0, 0), (70, 0, 0), (70, 3, 0), (40, 64, 2)])
def test_the_last_positions(gctx, kvt, M, sinks, branches):
    """2^30 positions of which a window's are held: the outputs are bit for bit
    those of a short sequence that ends in the same way."""
    rng = np.random.default_rng(41)
    W, heads, far = 100, 4, (1 << 30) - M
    n = 64 * 4 + far % 64  # as long as the window and a page more
    par = tree(M, branches) if branches else None
    near = Cache(gctx, rng, kvt, 64, 2, heads, [(n, M, par) if branches else (n, M)], W, sinks)
    near.write_new()
    q = queries(rng, near)
    want = near.check(q)
    table = near.tables[0]
    long = np.full(1 << 24, -1, np.int32)
    keep = len(table) - 1
    long[-keep:] = table[-keep:]
    long[0] = table[0]
    near.plan.set([(long, far, M, par)], heads, W, sinks)
    near.write_new()
    np.testing.assert_array_equal(near.attend(q), want)
    near.free()


@TYPES
def test_the_most_sequences(gctx, kvt):
    """65535 sequences of one token over one shared page, each with a page of its own."""
    n = 65535
    rng = np.random.default_rng(42)
    pool = gctx.pool(1, 1, 64, n + 1, kvt)
    ids = np.array(pool.take(n + 1), np.int32)
    own = rng.permutation(ids[1:])
    seqs = [((ids[0], own[i]), 64, 1) for i in range(n)]
    ctx_k, ctx_v = rng.standard_normal((2, 64, 64)).astype(np.float32)
    k, v, q = rng.standard_normal((3, n, 64)).astype(np.float32)
    fill = pool.plan([(ids[:1], 0, 64)])
    plan = pool.plan(seqs, 1)
    mats = [Rows(gctx, x) for x in (ctx_k, ctx_v, k, v, q, np.zeros_like(q))]
    fill.write(0, mats[0].ptr, mats[1].ptr)
    plan.write(0, mats[2].ptr, mats[3].ptr)
    plan.attend(0, mats[4].ptr, mats[5].ptr)
    gctx.sync()
    got = mats[5].get()
    back = [Rows(gctx, np.zeros_like(k)) for _ in range(2)]
    plan.read(0, back[0].ptr, back[1].ptr)
    gctx.sync()
    for b, x in zip(back, (k, v)):
        np.testing.assert_array_equal(b.get(), stored(x, kvt))
    ck, cv, k, v = (stored(x, kvt).astype(np.float64) for x in (ctx_k, ctx_v, k, v))
    q = q.astype(np.float64)
    s = np.concatenate([q @ ck.T, (q * k).sum(1, keepdims=True)], 1) / 8
    p = np.exp(s - s.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    mag = np.maximum((np.abs(q) @ np.abs(ck).T).max(1), (np.abs(q) * np.abs(k)).sum(1))[:, None] / 8
    b = p[:, :64] @ np.abs(cv) + p[:, 64:] * np.abs(v)
    tol = np.expm1(2 * 2.0 ** -18 * mag + 2.0 ** -20 + 10 * 2.0 ** -23) * b + 65 * 2.0 ** -32 * 6
    assert (np.abs(got - (p[:, :64] @ cv + p[:, 64:] * v)) <= tol).all()
    for x in (*mats, *back):
        x.buf.free()
    fill.free(), plan.free(), pool.free()


@TILES
@TYPES
@pytest.mark.parametrize("kv,heads,seqs", [(1, 999, [(70, 3), (5, 1)]), (1, 65, [(300, 1)]), (300, 300, [(100, 2)]), (257, 514, [(64, 40)])])
def test_many_heads(gctx, kvt, kv, heads, seqs):
    rng = np.random.default_rng(43)
    c = Cache(gctx, rng, kvt, 64, kv, heads, seqs)
    c.write_new()
    c.check(queries(rng, c))
    c.free()
