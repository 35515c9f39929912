"""Paged KV caches in 4 bits on the GPU: the stores bit for bit, and attention by
the bounds of 8-bit rows (test_gpu_paged.py): what a row stands for is an integer
of up to 2040, exact as a half, times one fp32 scale, as it is there.  The last
term of the bound, up to 2^-34 of the largest |v| for each slot seen, counts the
weights' lost low halves in values of the row's largest: here that is at least
7 * 255 = 1785 of 2040 steps, so the largest |v| stands for any value but for a
factor of 1.15, which the bound's own factor of two covers.
"""
import numpy as np
import pytest

import test_gpu_paged as P
import test_gpu_paged_extremes
import test_gpu_paged_levels
import test_gpu_paged_long
import test_gpu_paged_scores
import test_gpu_paged_steps as S
import test_gpu_paged_strides
from test_gpu_paged import TILES, Cache, Rows, queries, tiles  # noqa: F401
from xwfes_amd import ftx

pytestmark = pytest.mark.gpu

Q4 = ftx.KV_Q4
F = np.float32


def stored4(x, kvt=Q4):
    """What rows [..., hd] stand for once stored, every operation rounded to fp32."""
    assert kvt == Q4
    x = np.asarray(x, F)
    with np.errstate(all="ignore"):
        b = x.reshape(x.shape[:-1] + (x.shape[-1] // 32, 32))
        t = np.maximum(np.maximum(b, F(0)) * (F(1) / F(7)), np.maximum(-b, F(0)) / F(8)).max(-1)
        T = t.max(-1, keepdims=True)
        bad = ~np.isfinite(x).all(-1, keepdims=True)
        none = bad | (T < 2.0 ** -103)
        T = np.where(none, F(1), T).astype(F)
        s = T / F(255)
        c = np.minimum(np.ceil(t * (F(255) / T)), F(255))
        r = F(1) / (c * s)
        q = np.rint(b * r[..., None])
        q = np.where((c > 0)[..., None], q, F(0))
        assert none.any() or not q.size or (q.min() >= -8 and q.max() <= 7)
        y = ((q * c[..., None]).reshape(x.shape) * s).astype(F)
    return np.where(bad, F(np.nan), np.where(none, F(0), y)).astype(F)


@pytest.fixture(autouse=True)
def in_4_bits(monkeypatch):
    for m in (P, test_gpu_paged_extremes, test_gpu_paged_levels, test_gpu_paged_long, test_gpu_paged_scores):
        if hasattr(m, "stored"):
            monkeypatch.setattr(m, "stored", stored4)


def params(f, n=0):
    """The cases of a test of the other types: its n-th parametrisation but the types'."""
    marks = [m for m in f.pytestmark if m.name == "parametrize" and m.args[0] != "kvt"]
    return pytest.mark.parametrize(marks[n].args[0], marks[n].args[1])


# ---------------------------------------------------------------- stores


@params(P.test_rows_come_back_as_they_are_stored)
def test_rows_come_back_as_they_are_stored(gctx, hd, kv, seqs, pad, off):
    P.test_rows_come_back_as_they_are_stored(gctx, Q4, hd, kv, seqs, pad, off)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("M", [1, 14, 90])
def test_rows_of_every_size(gctx, hd, M):
    """Zero, tiny, subnormal, huge and mixed rows; blocks far apart in size; values at the
    borders of the rounding and their neighbours; rows that hold an infinity or a NaN.
    Row by row and page by page."""
    rng = np.random.default_rng(hd)
    base = rng.standard_normal(hd).astype(F)
    rows = [base * F(f) for f in (0, 2.0 ** -105, 2.0 ** -100, 2.0 ** -98, 1e-42, 1e30, 1.0, 1e-7)]
    big = base / np.abs(base).max()
    rows += [big * F(3.4e38), -big * F(3.4e38), np.abs(big), -np.abs(big)]
    # T on both sides of 2^-103
    for sign, most in ((1, 7), (-1, 8)):
        for e in (0.99, 1.0, 1.01):
            y = np.zeros(hd, F)
            y[hd - 1] = F(sign * most * e * 2.0 ** -103)
            rows.append(y)
    # blocks from one end of the multipliers to the other, and below
    y = base.copy()
    for g in range(hd // 32):
        y[32 * g:32 * g + 32] *= F(10.0 ** (-2 * g))
    rows += [y, y[::-1].copy(), -y]
    only = np.zeros(hd, F)
    only[hd // 2 + 3] = -5
    rows.append(only)
    # every border of the rounding, n + 1/2 steps, and its neighbours
    for step in (1.0, 0.37, 1e-3):
        n = (np.arange(hd) % 15) - 7.5
        y = (n * step).astype(F)
        y[::32], y[1::32] = F(7 * step), F(-8 * step)
        rows += [y, np.nextafter(y, F(np.inf)), np.nextafter(y, F(-np.inf))]
    for bad in (np.inf, -np.inf, np.nan):
        y = base.copy()
        y[hd - 9] = bad
        rows.append(y)
    x = np.stack(rows).astype(F)[:, None, :]
    x = np.concatenate([x] * (M // len(x) + 1))
    for at in range(0, len(x), M):
        part = x[at:at + M]
        n = len(part)
        c = Cache(gctx, rng, Q4, hd, 1, 0, [(7, n)],
                  rows=([np.concatenate([x[:7], part])], [np.concatenate([x[:7], -part])]))
        c.write_new()
        for got, s in zip(c.read(), (1, -1)):
            np.testing.assert_array_equal(got, stored4(s * part))
        for got, s in zip(c.read(context=True), (1, -1)):
            np.testing.assert_array_equal(got, stored4(np.concatenate([x[:7], s * part])))
        c.free()


def test_a_page_filled_token_by_token(gctx):
    """Every token's bytes are its own: tokens one at a time and several at once into the
    same page, others' rows as they were."""
    rng = np.random.default_rng(31)
    x = [rng.standard_normal((64, 2, 128)).astype(F) for _ in range(2)]
    pool = gctx.pool(1, 2, 128, 1, Q4)
    pages = pool.take(1)
    c = Cache.__new__(Cache)
    c.ctx, c.kvt, c.hd, c.kv, c.heads, c.layer, c.pool = gctx, Q4, 128, 2, 0, 0, pool
    at = 0
    for n in (1, 2, 1, 7, 15, 1, 20, 17):
        plan = pool.plan([(pages, at, n)])
        c.write(plan, [x[0][at:at + n]], [x[1][at:at + n]])
        at += n
        for got, y in zip(c.read(plan, context=True, n=at), x):
            np.testing.assert_array_equal(got, stored4(y[:at]))
        plan.free()
    assert at == 64
    pool.free()


# ---------------------------------------------------------------- attention


@TILES
@params(P.test_chains)
def test_chains(gctx, hd, kv, heads, seqs):
    P.test_chains(gctx, Q4, hd, kv, heads, seqs)


@TILES
@params(P.test_windows)
def test_windows(gctx, hd, kv, heads, seqs, window, sinks):
    P.test_windows(gctx, Q4, hd, kv, heads, seqs, window, sinks)


@TILES
@params(P.test_trees)
def test_trees(gctx, hd, kv, heads, seqs, window, sinks):
    P.test_trees(gctx, Q4, hd, kv, heads, seqs, window, sinks)


@TILES
@params(P.test_values_of_every_size)
def test_values_of_every_size(gctx, qs, ks, vs):
    P.test_values_of_every_size(gctx, Q4, qs, ks, vs)


@TILES
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("seqs,heads", [([(300, 1)], 4), ([(300, 3), (90, 1)], 2), ([(200, 9)], 8), ([(130, 40)], 2)])
def test_blocks_of_every_size(gctx, hd, seqs, heads):
    """Keys and values whose blocks of 32 dims lie far apart, rows far apart in size."""
    rng = np.random.default_rng(hd + heads)
    rows = []
    for _ in range(2):
        x = [rng.standard_normal((a + b, 1, hd)).astype(F) for a, b in seqs]
        for y in x:
            y *= np.repeat(F(10.0) ** rng.integers(-3, 1, (len(y), 1, hd // 32)), 32, -1).astype(F)
            y *= F(10.0) ** rng.integers(-4, 2, (len(y), 1, 1)).astype(F)
        rows.append(x)
    c = Cache(gctx, rng, Q4, hd, 1, heads, seqs, rows=rows)
    c.write_new()
    c.check(queries(rng, c, 2.0))
    c.free()


@pytest.mark.parametrize("hd,kv,heads,seqs", [
    (128, 1, 4, [(300, 1)]), (64, 1, 4, [(300, 1), (70, 1)]), (128, 1, 8, [(300, 1)]), (64, 2, 8, [(130, 2)]),
    (128, 2, 16, [(900, 1)]), (128, 1, 1, [(200, 1)]), (128, 1, 6, [(64, 1), (200, 1)]), (256, 1, 4, [(200, 1)]), (128, 1, 16, [(200, 1)])])
def test_blocks_of_one_value(gctx, hd, kv, heads, seqs):
    """Keys whose blocks hold one value each, in dims where the query is small: what the
    other dims, zeros held as 8 less 8, leave of a score is its rounding.

    A block's sum starts at -8 sum q and takes nibbles of up to 15: partial sums of up to
    23 sum |q|, rounded four times by 2^-23 (each product of 32 dims in up to two steps, for
    both halves of q), in steps c s; the block's largest |k| is at least 3.5 of them (c is
    less than twice what it covers): 4 * 23 / 3.5 2^-23 < 2^-18 of sum |q| max |k|."""
    rng = np.random.default_rng(hd + heads)
    g = heads // kv
    ks, vs = [], []
    for a, b in seqs:
        k = np.zeros((a + b, kv, hd // 32, 32), F)
        k[..., 5] = rng.standard_normal(k.shape[:-1]) * 3
        ks.append(k.reshape(a + b, kv, hd))
        vs.append(rng.standard_normal((a + b, kv, hd)).astype(F))
    c = Cache(gctx, rng, Q4, hd, kv, heads, seqs, rows=(ks, vs))
    c.write_new()
    q = rng.standard_normal((c.new, heads, hd)).astype(F) * 4
    q.reshape(c.new, heads, -1, 32)[..., 5] *= F(1 / 64)
    got, at = c.attend(q.reshape(c.new, -1)), 0
    for (_, npast, M, _), k, v in zip(c.seqs, ks, vs):
        k64, v64 = (np.repeat(stored4(x).astype(np.float64), g, axis=1) for x in (k, v))
        qs = q[at:at + M].astype(np.float64)
        s = np.einsum("ihd,jhd->hij", qs, k64) / np.sqrt(hd)
        top = np.abs(k64).reshape(npast + M, heads, -1, 32).max(-1)
        mag = np.einsum("ihb,jhb->hij", np.abs(qs).reshape(M, heads, -1, 32).sum(-1), top).max() / np.sqrt(hd)
        see = np.arange(npast + M) <= npast + np.arange(M)[:, None]
        p = np.where(see, np.exp(s - s.max()), 0)
        p /= p.sum(-1, keepdims=True)
        want, b = (np.einsum("hij,jhd->ihd", p, x) for x in (v64, np.abs(v64)))
        tol = 2 * 2.0 ** -18 * mag + 2.0 ** -20 + 5 * ((npast + M) // 64 + 1) * 2.0 ** -23
        err = np.abs(got[at:at + M] - want)
        assert (err <= np.expm1(tol) * b + (npast + M) * 2.0 ** -34 * np.abs(v64).max()).all()
        at += M
    c.free()


def test_dims_of_zeros_stay_zero(gctx):
    """An output dim over values that are all held as zero is zero, whatever lies beside it."""
    rng = np.random.default_rng(77)
    for hd, heads, M in ((128, 4, 1), (64, 8, 1), (128, 8, 1), (64, 4, 1), (128, 16, 1), (128, 4, 30), (256, 4, 1)):
        v = rng.standard_normal((200 + M, 1, hd)).astype(F) * 100
        zero = rng.permutation(hd)[:hd // 3]
        v[:, :, zero] = rng.uniform(-1e-3, 1e-3, (200 + M, 1, len(zero)))
        c = Cache(gctx, rng, Q4, hd, 1, heads, [(200, M)], rows=([rng.standard_normal((200 + M, 1, hd)).astype(F)], [v]))
        c.write_new()
        got = c.check(queries(rng, c))
        assert not stored4(v)[:, :, zero].any() and not got[:, :, zero].any() and got.any()
        c.free()


@TILES
def test_large_values_in_hidden_places_change_nothing(gctx):
    P.test_large_values_in_hidden_places_change_nothing(gctx, Q4)


@TILES
def test_a_row_hidden_by_the_window(gctx):
    P.test_a_row_hidden_by_the_window(gctx, Q4)


@TILES
def test_pages_that_held_other_things(gctx):
    P.test_pages_that_held_other_things(gctx, Q4)


@TILES
@params(P.test_strides_and_alignment)
def test_strides_and_alignment(gctx, pad, off):
    P.test_strides_and_alignment(gctx, Q4, pad, off)


@TILES
def test_chunks_give_what_one_chunk_gives(gctx):
    P.test_chunks_give_what_one_chunk_gives(gctx, Q4)


@TILES
def test_shared_prefix_pages(gctx):
    P.test_shared_prefix_pages(gctx, Q4)


def test_two_graphs_replayed(gctx):
    P.test_two_graphs_replayed(gctx, Q4)


@params(test_gpu_paged_strides.test_many_rows)
def test_strides_of_many_rows(gctx, hd, kv, heads, seqs, rows):
    test_gpu_paged_strides.test_many_rows(gctx, Q4, hd, kv, heads, seqs, rows)


@params(test_gpu_paged_strides.test_joins)
def test_joins(gctx, hd, kv, heads, seqs, rows, parts):
    test_gpu_paged_strides.test_joins(gctx, Q4, hd, kv, heads, seqs, rows, parts)


@params(test_gpu_paged_long.test_pages_past_the_first_64)
def test_pages_past_the_first_64(gctx, M, rows):
    test_gpu_paged_long.test_pages_past_the_first_64(gctx, Q4, M, rows)


@params(test_gpu_paged_long.test_sums_of_alike_weights)
def test_sums_of_alike_weights(gctx, M, rows):
    test_gpu_paged_long.test_sums_of_alike_weights(gctx, Q4, M, rows)


@TILES
@params(test_gpu_paged_scores.test_scores_past_fp32_are_nan)
def test_scores_past_fp32_are_nan(gctx, sign):
    test_gpu_paged_scores.test_scores_past_fp32_are_nan(gctx, Q4, sign)


def test_offsets_past_32_bits(gctx):
    """A pool of 9.6 GB: the last pages of its last layer."""
    rng = np.random.default_rng(19)
    pages = 32600
    pool = gctx.pool(4, 8, 128, pages, Q4)
    ids = pool.take(pages)
    c = Cache.__new__(Cache)
    c.ctx, c.kvt, c.hd, c.kv, c.heads, c.window, c.sinks, c.layer, c.pool = gctx, Q4, 128, 8, 8, 0, 0, 3, pool
    c.seqs, c.new = [(ids[-3:][::-1], 0, 150, None)], 150
    c.k, c.v = ([rng.standard_normal((150, 8, 128)).astype(F)] for _ in range(2))
    c.plan = pool.plan(c.seqs, 8)
    c.write_new()
    c.check(queries(rng, c))
    c.free()


# ---------------------------------------------------------------- verify steps


@params(S.test_rows_of_a_step_are_stored_as_the_store_does)
def test_rows_of_a_step_are_stored_as_the_store_does(gctx, orc, monkeypatch, cfg, neox, M):
    monkeypatch.setattr(S, "stored", stored4)
    S.test_rows_of_a_step_are_stored_as_the_store_does(gctx, orc, Q4, cfg, neox, M)


def test_commit_of_a_tree_path(gctx, orc):
    """A path's rows move to the next slots, across a page's end, byte for byte; the step
    after it is the step after the chain of the path.

    Projections of up to 8 tokens and of more differ by some 1e-4 of a row's size.  By that
    one value in 1400 crosses its rounding (15 steps to four times the row's spread, 0.57 of
    it a step): sqrt(1 / 1400) 0.57 = 1.5e-2.  One multiplier in 40 does (255 to T): its block
    moves by up to 1/255 and one value in 60 of it with it: sqrt(1 / 40) (0.004 + sqrt(1 / 60)
    0.57) = 1.2e-2.  Together 2e-2 of a row's size in the rows that differ, as a share of the
    logits less, by the rows seen; 8-bit rows' 3e-3 are given 5 LOGIT_TOL."""
    t = S.Setup(gctx, orc, S.CFG64, S.Q8, Q4)
    toks = np.random.default_rng(3).integers(0, 300, 20).tolist()
    par = [-1, -1, 0, 1, 2, 2, 3, 4, 5, 6, 7, 7, 8, 9, 10, 11, 12, 13, 14, 15]
    path = [1, 3, 6, 9, 13, 17]
    a, _, _ = t.context(60, 90)
    b, _, _ = t.context(60, 90)
    t.step([(a, toks, par, False)])
    before = a.read()
    a.commit(path)
    for x, y in zip(before, a.read()):
        np.testing.assert_array_equal(y[:, :60], x[:, :60])
        np.testing.assert_array_equal(y[:, 60:66], x[:, [60 + j for j in path]])
    t.step([(b, [toks[j] for j in path], None, True)])
    assert a.pointers()[2] == b.pointers()[2] == 66
    x, y = (t.step([(z, [7], None, True)])[0] for z in (a, b))
    assert S.rel_err_rows(x, y) < 34 * S.LOGIT_TOL
    t.free()


def test_steps_near_those_of_halves(gctx, orc):
    """Steps over 4-bit rows are steps over the rows that they stand for: a cache of halves
    given those rows (they are within halves' reach) has the same logits, but for halves'
    rounding of them and of the new rows that are kept in 4 bits here."""
    t = S.Setup(gctx, orc, S.CFG64, S.Q8, Q4)
    u = S.Setup(gctx, orc, S.CFG64, S.Q8, ftx.KV_F16)
    kv, _, _ = t.context(200, 230)
    k, v = kv.read()
    half = u.gm.kv_paged(u.pool, 230)
    u.kvs.append(half)
    half.write(k, v)
    half.truncate(200)
    x, = t.step([(kv, [5], None, False)])
    y, = u.step([(half, [5], None, False)])
    # one new row of 201 in 4 bits: off by 0.08 of its size at most (a step of 0.27 of a block's
    # spread, rounded evenly), a 201st part of what is seen, and halves' 2^-11 of every row
    assert S.rel_err_rows(x, y) < 5 * S.LOGIT_TOL
    t.free(), u.free()


def test_steps_of_a_batch_and_under_a_window(gctx, orc):
    """Sequences of one batch as each by itself (their rows' last bits may differ by the
    batch's width: the bound of test_commit_of_a_tree_path); a window leaves its pages behind."""
    t = S.Setup(gctx, orc, S.CFG128, S.Q8, Q4)
    kvs = [t.context(n, 230, seed=n)[0] for n in (10, 128, 200)]
    alone = [t.step([(kv, [7, 9], None, False)])[0] for kv in kvs]
    for x, y in zip(t.step([(kv, [7, 9], None, False) for kv in kvs]), alone):
        assert S.rel_err_rows(x, y) < 34 * S.LOGIT_TOL
    free = t.pool.available
    kv = t.gm.kv_paged(t.pool, 400, window=70, sinks=4)
    t.kvs.append(kv)
    for i in range(6):
        x, = t.step([(kv, list(range(i, i + 50)), None, True)])
        assert np.isfinite(x).all()
    # the last step's 250 before it and 50: the first page, and from 250 - 69 on
    assert free - t.pool.available == 1 + 3
    t.free()


@pytest.mark.parametrize("hd,heads,kv,seqs", [
    (64, 4, 1, [(300, 1), (5, 1)]), (128, 8, 2, [(300, 1)]), (128, 8, 1, [(1000, 1), (70, 1)]), (64, 6, 1, [(40, 1)]),
    (128, 2, 2, [(700, 4)]), (64, 16, 2, [(2000, 1)]), (128, 1, 1, [(130, 8)])])
def test_strides_of_few_rows(gctx, hd, heads, kv, seqs):
    rng = np.random.default_rng(15)
    c = Cache(gctx, rng, Q4, hd, kv, heads, seqs)
    c.write_new()
    q = queries(rng, c)
    want = c.check(q)
    for pad, off in test_gpu_paged_strides.WAYS:
        c.write_new(pad=pad, off=off)
        np.testing.assert_array_equal(c.attend(q, pad=pad, off=off), want)
    c.free()


@pytest.mark.parametrize("heads,M,window,sinks", [(1, 1, 0, 0), (4, 1, 0, 0), (3, 1, 100, 3), (8, 1, 0, 0), (2, 3, 0, 0), (2, 4, 40, 66),
                                                  (1, 7, 0, 0), (5, 1, 1, 0), (7, 1, 64, 64)])
@pytest.mark.parametrize("hd", [64, 128])
def test_few_rows_of_every_number(gctx, hd, heads, M, window, sinks):
    """One to eight query rows a kv head: sequences of no token to many, whole and cut lists."""
    rng = np.random.default_rng(heads * 8 + M)
    seqs = [(n, M) for n in (0, 1, 15, 16, 63 - M, 64, 191, 700, 3000)]
    c = Cache(gctx, rng, Q4, hd, 1, heads, seqs, window, sinks)
    c.write_new()
    c.check(queries(rng, c, 2.0))
    c.free()


def test_many_sequences(gctx):
    """More lists than the chip takes at once, long ones among short ones."""
    rng = np.random.default_rng(41)
    seqs = [(int(n), 1) for n in rng.integers(0, 130, 600)] + [(5000, 1), (2500, 1)]
    c = Cache(gctx, rng, Q4, 64, 2, 4, seqs)
    c.write_new()
    c.check(queries(rng, c))
    c.free()


@pytest.mark.parametrize("hd,heads,M", [(64, 4, 1), (128, 4, 1), (128, 3, 1), (64, 8, 1), (128, 8, 1), (128, 2, 4), (128, 16, 1),
                                        (256, 4, 1), (64, 2, 50)])
def test_queries_that_are_no_numbers(gctx, hd, heads, M):
    """A query row that holds an infinity or a NaN is NaN, the others are what they were bit
    for bit, also those whose products share its instructions."""
    rng = np.random.default_rng(hd + heads + M)
    c = Cache(gctx, rng, Q4, hd, 1, heads, [(700, M), (40, M)])
    c.write_new()
    q = queries(rng, c)
    want = c.check(q)
    rows = q.reshape(-1, hd)
    for n, bad in enumerate((np.nan, np.inf, -np.inf)):
        for r in (0, len(rows) // 2, len(rows) - 1):
            x = rows.copy()
            x[r, (37 * n + 5 * r) % hd] = bad
            got = c.attend(x.reshape(q.shape)).reshape(-1, hd)
            assert np.isnan(got[r]).all()
            np.testing.assert_array_equal(np.delete(got, r, 0), np.delete(want.reshape(-1, hd), r, 0))
    c.free()


@pytest.mark.parametrize("qe,ke", [(117, -98), (120, -60), (126, -98), (126, -20), (-126, 110), (-140, 100)])
@pytest.mark.parametrize("hd,heads,M", [(64, 4, 1), (128, 4, 1), (64, 8, 1), (128, 8, 1), (128, 16, 1), (64, 2, 40), (256, 3, 1)])
def test_queries_of_every_size(gctx, hd, heads, M, qe, ke):
    """The largest and smallest queries over rows that are all alike: whatever the score, an
    output is the mean of the values seen."""
    rng = np.random.default_rng(qe + 200)
    k = np.repeat(rng.uniform(-1, 1, (1, 1, hd)).astype(F) * F(2.0 ** ke), 300 + M, 0)
    v = rng.standard_normal((300 + M, 1, hd)).astype(F)
    c = Cache(gctx, rng, Q4, hd, 1, heads, [(300, M)], rows=([k], [v]))
    c.write_new()
    got = c.attend((rng.uniform(-1, 1, (M, heads * hd)) * 2.0 ** qe).astype(F))
    want = np.cumsum(stored4(v).astype(np.float64), 0)[300:] / np.arange(301, 301 + M)[:, None, None]
    # (the weights are alike to a bit: what is left are the sums of six pages, 2^-20 each of the mean |v|)
    assert (np.abs(got - want) <= 2.0 ** -16 * np.abs(v).max()).all()
    c.free()


@pytest.mark.parametrize("hd,kv,heads", [(64, 2, 8), (128, 2, 8), (128, 1, 8), (64, 1, 1)])
def test_scores_of_two_slots(gctx, hd, kv, heads):
    """Two slots, where an output is off by what a score is.  Query elements of 2^6 to 2^7
    times nibbles of up to 15 2^-20 keep 24 bits below 2^7 2^-14, 2^-18 |q|max of a nibble's unit a
    product; a block's sum |q_i| max |k| is some 32 / 3 |q|max times 7 units, so that its two
    products and the sums in fp32 stay below 2^-22 of it."""
    rng = np.random.default_rng(hd + heads)
    c = Cache(gctx, rng, Q4, hd, kv, heads, [(1, 1)] * 200)
    c.write_new()
    q = queries(rng, c)
    got = c.attend(q).reshape(200, kv, heads // kv, hd)
    q64 = np.asarray(q, np.float64).reshape(200, kv, heads // kv, hd) / np.sqrt(hd)
    k, v = (np.stack([stored4(x) for x in y]).astype(np.float64) for y in (c.k, c.v))  # [200][2 slots][kv][hd]
    s = np.einsum("skhd,sjkd->skhj", q64, k)
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    big = np.repeat(np.abs(k).reshape(200, 2, kv, hd // 32, 32).max(-1), 32, -1)
    mag = np.einsum("skhd,sjkd->skhj", np.abs(q64), big).max(-1)[..., None]
    err = np.abs(got - np.einsum("skhj,sjkd->skhd", p, v))
    tol = (np.expm1(2 * 2.0 ** -22 * mag) + 2.0 ** -20 + 5 * 2.0 ** -23) * np.einsum("skhj,sjkd->skhd", p, np.abs(v))
    assert (err <= tol).all(), (err - tol).max()
    c.free()
