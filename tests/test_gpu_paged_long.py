"""Long page lists that one workgroup walks by itself: 128 sequences over one
shared context, so that there are workgroups enough and no list is split."""
import numpy as np
import pytest

from test_gpu_paged import TYPES, Rows, stored
from test_paged_plan import probe

pytestmark = pytest.mark.gpu

NSEQ, KV, HD = 128, 8, 64
# new tokens, rows of a tile (one query head a kv head); 65 rows and more: 128 or 256
SHAPES = pytest.mark.parametrize("M,rows", [(1, 0), (40, 0), (70, 128), (70, 256)], ids=["one", "few", "many", "many-256"])


def attend(ctx, kvt, k, v, q, M, rows):
    """Outputs [M][KV][HD] of the first and the last of NSEQ sequences, all with
    new rows k[-M:], v[-M:] and queries q [M][KV][HD] after the same context."""
    n, own = len(k) - M, (M + 63) // 64
    ctx.lib.paged_force_rows(rows)
    pool = ctx.pool(1, KV, HD, n // 64 + NSEQ * own, kvt)
    ids = pool.take(n // 64 + NSEQ * own)
    shared = np.random.default_rng(1).permutation(ids[:n // 64])
    own = np.array(ids[n // 64:]).reshape(NSEQ, own)
    seqs = [(np.append(shared, x), n, M) for x in own]
    try:
        plan = pool.plan(seqs, KV)
        rc, msg, items, joins = probe(seqs, KV, KV, n_pages=len(ids), hd=HD)
        assert rc == 0 and len(joins) == 0 and ((items[:, 7] > 0) == (rows > 0)).all(), msg
        assert (items[:, 2] == 0).all() and (items[:, 3] > n // 64).all()
    finally:
        ctx.lib.paged_force_rows(0)
    fill = pool.plan([(shared, 0, n)])
    mats = [Rows(ctx, x[:n]) for x in (k, v)]
    mats += [Rows(ctx, np.tile(x.reshape(len(x), -1), (NSEQ, 1))) for x in (k[n:], v[n:], q, np.zeros_like(q))]
    fill.write(0, mats[0].ptr, mats[1].ptr)
    plan.write(0, mats[2].ptr, mats[3].ptr)
    plan.attend(0, mats[4].ptr, mats[5].ptr)
    ctx.sync()
    got = mats[5].get().reshape(NSEQ, M, KV, HD)
    for x in mats:
        x.buf.free()
    fill.free(), plan.free(), pool.free()
    np.testing.assert_array_equal(got[1:], got[:-1])
    return got[0]


def exact(kvt, k, v, q, M):
    """Outputs, sum p |v| and the scores' largest sum of magnitudes, [M][KV][HD or 1]."""
    n = len(k) - M
    k, v = (stored(x, kvt).astype(np.float64).transpose(1, 0, 2) for x in (k, v))
    q = q.astype(np.float64).transpose(1, 0, 2)
    see = np.arange(n + M) <= n + np.arange(M)[:, None]
    s = np.where(see, q @ k.transpose(0, 2, 1) / np.sqrt(HD), -np.inf)
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    mag = (np.abs(q) @ np.abs(k).transpose(0, 2, 1)).max(-1, keepdims=True) / np.sqrt(HD)
    return [x.transpose(1, 0, 2) for x in (p @ v, p @ np.abs(v), mag)]


@TYPES
@SHAPES
def test_pages_past_the_first_64(gctx, kvt, M, rows):
    """Every page of a list of more than 64 for each wave (few rows: four waves
    deal the pages among them) is the right one: scores that differ much, each row's
    weight on slots all over the list."""
    n = 64 * (300 if rows == 0 else 150)
    rng = np.random.default_rng(M)
    k, v, q = (rng.standard_normal((m, KV, HD)).astype(np.float32) for m in (n + M, n + M, M))
    got = attend(gctx, kvt, k, v, q * 2, M, rows)
    want, b, mag = exact(kvt, k, v, q * 2, M)
    # (the bound of the stores' tests; 2^-32 of |v| < 6 for each slot)
    tol = np.expm1(2 * 2.0 ** -18 * mag + 2.0 ** -20 + 5 * (n // 64 + 2) * 2.0 ** -23) * b + (n + M) * 2.0 ** -32 * 6
    assert tol.max() < 1e-3
    assert (np.abs(got - want) <= tol).all(), np.abs(got - want).max()


@TYPES
@SHAPES
def test_sums_of_alike_weights(gctx, kvt, M, rows):
    """65536 slots of one score under a larger one's, V rows of the first page
    alone: their sum is as good as kept, so that the error is that of the softmax
    sum.  It takes one rounding of 2^-24 for each page, and 16 within a page; the
    rest as in the stores' tests, but for low halves that are lost: every weight is
    more than half of the largest and keeps both halves."""
    n = 65536
    k = np.zeros((n + M, KV, HD), np.float32)
    k[:, :, 0] = 0.1234
    k[0, :, 0] = 0.5
    v = np.zeros_like(k)
    v[:64] = np.random.default_rng(2).uniform(0.5, 1.0, (64, KV, HD))
    q = np.zeros((M, KV, HD), np.float32)
    q[:, :, 0] = np.linspace(5, 9, M)[:, None] if M > 1 else 7.3
    got = attend(gctx, kvt, k, v, q, M, rows)
    want, b, mag = exact(kvt, k, v, q, M)
    tol = np.expm1(2 * 2.0 ** -18 * mag + 2.0 ** -20 + 5 * 2.0 ** -23 + (n // 64 + 18) * 2.0 ** -24) * b
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / b).max()
