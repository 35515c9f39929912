"""Paged KV caches on the GPU: rows quantised as they are written and read
back, and the attention of new tokens over pages, against 64-bit numpy.

Stores are exact: the scale is one IEEE division, the rounding's border is
decided in 64 bits, a read-back value is one product.

Attention's bound for a row, relative to sum_j p_j |v_j|.  A score is off by at
most 2^-18 sum |q_i k_ji| / sqrt(hd) (q's two halves: 2^-22; up to 16 MFMA
accumulations that round by 2^-23; the products with the row's and slot's
scale 2^-23), which moves every p by as much, twice (p and the sum).  P's two
halves: 2^-21; of a p so small that its low half is lost, 2^-25 of what the
halves are scaled to (2^10 to 2^14 for the row's largest p and V scale), so up
to 2^-35 (2^-34 with the scale's own factor of two) of the largest |v| for each
slot seen: a bound relative to sum p |v| alone does not hold where the few large
p meet v near 0.  The outputs' sums round 4 times a page by 2^-23, the softmax
sum 16 times by 2^-24; a join of partials adds 2^-21.
"""
import ctypes

import numpy as np
import pytest

from xwfes_amd import ftx
from test_paged_plan import depths, visible
from test_zz_no_alloc import _hip

pytestmark = pytest.mark.gpu

F16, Q8 = ftx.KV_F16, ftx.KV_Q8
TYPES = pytest.mark.parametrize("kvt", [F16, Q8], ids=["f16", "q8"])


@pytest.fixture(params=[0, 16, 128, 256], ids=["est", "r16", "r128", "r256"])
def tiles(request):
    """The row tiles of sequences of 65 rows and more: by the estimate, or given."""
    force = ftx.load().paged_force_rows
    force(request.param)
    yield request.param
    force(0)


TILES = pytest.mark.usefixtures("tiles")


def stored(x, kvt):
    """What rows [..., hd] stand for once stored."""
    x = np.asarray(x, np.float32)
    a = np.abs(x).max(-1, keepdims=True)
    bad = ~np.isfinite(x).all(-1, keepdims=True)
    tiny = bad | (a < 2.0 ** -100)
    a1 = np.where(tiny, np.float32(1), a)
    if kvt == Q8:
        q = np.rint(np.where(tiny, 0, x).astype(np.float64) * 127.0 / a1)
        y = q.astype(np.float32) * (a1 / np.float32(127))
    else:
        e = np.where((a1 >= 2.0 ** -8) & (a1 <= 65504), 0, np.frexp(a1)[1] - 1 - 14)
        y = np.ldexp(np.ldexp(np.where(tiny, 0, x).astype(np.float64), -e).astype(np.float16).astype(np.float64), e)
    return np.where(bad, np.float32(np.nan), np.where(tiny, np.float32(0), y)).astype(np.float32)


class Rows:
    """A float matrix on the device, `pad` floats between rows, `off` floats in front."""

    def __init__(self, ctx, a, pad=0, off=0, fill=-7.0):
        a = np.ascontiguousarray(a, np.float32)
        a = a.reshape(a.shape[0], -1)
        self.n, self.w, self.off = a.shape[0], a.shape[1], off
        self.ld = self.w + pad
        self.host = np.full(off + max(self.n, 1) * self.ld + 4, fill, np.float32)
        self.view(self.host)[:] = a
        self.buf = ctx.buffer(self.host.nbytes)
        self.buf.write(self.host)

    def view(self, flat):
        return flat[self.off:self.off + self.n * self.ld].reshape(self.n, self.ld)[:, :self.w]

    @property
    def ptr(self):
        return self.buf.ptr + 4 * self.off

    def get(self):
        """The matrix; what lies around it must be as it was."""
        flat = self.buf.read(np.float32, self.host.size)
        out = self.view(flat).copy()
        self.view(flat)[:] = self.view(self.host)
        np.testing.assert_array_equal(flat, self.host)
        return out


class Cache:
    """A pool with the contexts of `seqs` = [(npast, M[, parents])] written to
    layer `layer`, pages in a shuffled order, and a plan for the new tokens."""

    def __init__(self, ctx, rng, kvt, hd, kv, heads, seqs, window=0, sinks=0, layer=0, n_layer=1, scale=1.0,
                 spare=2, rows=None, drop=True):
        self.ctx, self.kvt, self.hd, self.kv, self.heads = ctx, kvt, hd, kv, heads
        self.window, self.sinks, self.layer = window, sinks, layer
        need = [(s[0] + s[1] + 63) // 64 for s in seqs]
        self.pool = ctx.pool(n_layer, kv, hd, sum(need) + spare, kvt)
        ids = rng.permutation(self.pool.take(sum(need)))
        ends = np.cumsum([0] + need)
        self.tables = [ids[ends[i]:ends[i + 1]] for i in range(len(seqs))]
        self.seqs = [(self.tables[i], s[0], s[1], s[2] if len(s) > 2 else None) for i, s in enumerate(seqs)]
        self.k, self.v = rows or [[(rng.standard_normal((s[0] + s[1], kv, hd)) * scale).astype(np.float32)
                                   for s in seqs] for _ in range(2)]
        self.new = sum(s[1] for s in seqs)
        if sum(s[0] for s in seqs):
            fill = self.pool.plan([(t, 0, s[0]) for t, s in zip(self.tables, seqs)])
            self.write(fill, [k[:s[0]] for k, s in zip(self.k, seqs)], [v[:s[0]] for v, s in zip(self.v, seqs)])
            fill.free()
        self.plan = self.pool.plan(self.seqs, heads, window, sinks)

    def write(self, plan, ks, vs, pad=0, off=0):
        k, v = (Rows(self.ctx, np.concatenate(x), pad, off) for x in (ks, vs))
        plan.write(self.layer, k.ptr, v.ptr, k.ld if pad else 0, v.ld if pad else 0)
        self.ctx.sync()
        for x in (k, v):
            x.buf.free()

    def write_new(self, **kw):
        self.write(self.plan, [k[s[1]:] for k, s in zip(self.k, self.seqs)],
                   [v[s[1]:] for v, s in zip(self.v, self.seqs)], **kw)

    def read(self, plan=None, context=False, pad=0, off=0, n=None):
        n = n if n is not None else sum(s[1] + s[2] for s in self.seqs) if context else self.new
        out = [Rows(self.ctx, np.zeros((n, self.kv * self.hd)), pad, off) for _ in range(2)]
        (plan or self.plan).read(self.layer, out[0].ptr, out[1].ptr, context, out[0].ld, out[1].ld)
        self.ctx.sync()
        got = [x.get().reshape(n, self.kv, self.hd) for x in out]
        for x in out:
            x.buf.free()
        return got

    def attend(self, q, pad=0, off=0, spare=0):
        qd = Rows(self.ctx, q, pad, off)
        out = Rows(self.ctx, np.full((self.new, self.heads * self.hd), 9.0), pad, off)
        self.plan.attend(self.layer, qd.ptr, out.ptr, qd.ld, out.ld)
        self.ctx.sync()
        got = out.get().reshape(self.new, self.heads, self.hd)
        qd.buf.free(), out.buf.free()
        return got

    def want(self, q):
        """(outputs, bounds) in 64 bits over the stored values."""
        q = np.asarray(q, np.float64).reshape(self.new, self.heads, self.hd)
        outs, tols, at, g = [], [], 0, self.heads // self.kv
        for (_, npast, M, par), k, v in zip(self.seqs, self.k, self.v):
            see = visible(npast, M, par, self.window, self.sinks)
            k64, v64 = (np.repeat(stored(x, self.kvt).astype(np.float64), g, axis=1) for x in (k, v))
            qs = q[at:at + M]
            at += M
            with np.errstate(all="ignore"):
                s = np.einsum("ihd,jhd->hij", qs, k64) / np.sqrt(self.hd)
                s = np.where(see[None], s, -np.inf)
                p = np.exp(s - np.nanmax(s, -1, keepdims=True, initial=-np.inf))
                p = np.where(np.isnan(s), np.nan, p)
                p /= p.sum(-1, keepdims=True)
                pz = np.where(see[None], p, 0)
                vz = np.where(np.isfinite(v64), v64, np.nan)
                o = np.zeros((M, self.heads, self.hd))
                b = np.zeros((M, self.heads, self.hd))
                for i in range(M):
                    o[i] = np.einsum("hj,jhd->hd", pz[:, i, see[i]], vz[see[i]])
                    b[i] = np.einsum("hj,jhd->hd", pz[:, i, see[i]], np.abs(vz[see[i]]))
                mag = np.einsum("ihd,jhd->hij", np.abs(qs), np.abs(k64)) / np.sqrt(self.hd)
                mag = np.where(see[None], mag, 0).max(-1, initial=0).T[..., None]
            pages = (npast + M) // 64 + 1
            tol = 2 * 2.0 ** -18 * mag + 2.0 ** -20 + 5 * pages * 2.0 ** -23
            outs.append(o)
            n = see.sum(1)[:, None, None]
            tols.append(np.expm1(np.minimum(tol, 50)) * b + n * 2.0 ** -34 * np.abs(np.nan_to_num(v64)).max(initial=0))
        return np.concatenate(outs), np.concatenate(tols)

    def check(self, q, **kw):
        got = self.attend(q, **kw)
        want, tol = self.want(q)
        assert (np.isnan(got) == np.isnan(want)).all()
        err = np.abs(got - want)
        bad = np.nan_to_num(err) > np.nan_to_num(tol)
        assert not bad.any(), (np.argwhere(bad)[:4], np.nanmax(err / tol))
        return got

    def free(self):
        self.plan.free()
        self.pool.free()


def tree(M, b):
    return [-1 if i < b else max(i - b - i % 3, 0) for i in range(M)]


def queries(rng, c, scale=1.0):
    return (rng.standard_normal((c.new, c.heads * c.hd)) * scale).astype(np.float32)


# ---------------------------------------------------------------- stores


@TYPES
@pytest.mark.parametrize("hd,kv,seqs,pad,off", [
    (64, 1, [(0, 1)], 0, 0), (128, 8, [(2047, 1)], 0, 0), (256, 2, [(60, 9), (0, 64), (5, 0), (64, 130)], 0, 0),
    (128, 3, [(63, 2), (64, 1), (1, 62), (0, 63)], 5, 1), (64, 8, [(37, 300)], 4, 4), (128, 1, [(10, 1)] * 40, 0, 2)])
def test_rows_come_back_as_they_are_stored(gctx, kvt, hd, kv, seqs, pad, off):
    rng = np.random.default_rng(hd + kv)
    c = Cache(gctx, rng, kvt, hd, kv, 0, seqs, layer=1, n_layer=3)
    c.write_new(pad=pad, off=off)
    for got, x in zip(c.read(pad=pad, off=off), (c.k, c.v)):
        np.testing.assert_array_equal(got, stored(np.concatenate([r[s[1]:] for r, s in zip(x, c.seqs)]), kvt))
    for got, x in zip(c.read(context=True), (c.k, c.v)):
        np.testing.assert_array_equal(got, stored(np.concatenate(x), kvt))
    # the layers on either side hold nothing
    for layer in (0, 2):
        c.layer = layer
        assert not any(x.any() for x in (np.nan_to_num(y) for y in c.read(context=True)) if kvt == F16)
    c.free()


@TYPES
def test_rows_of_every_size(gctx, kvt):
    """Zero, tiny, subnormal, huge and mixed rows, borders of the rounding,
    rows that hold an infinity or a NaN."""
    hd = 128
    rng = np.random.default_rng(5)
    base = rng.standard_normal((1, hd)).astype(np.float32)
    rows = [base * 0, base * 2.0 ** -105, base * 2.0 ** -98, base * 1e-42, base * 1e30, base * 2.0 ** -7, base * 2.0 ** -9,
            base / np.abs(base).max() * 65504, base / np.abs(base).max() * 65505, base / np.abs(base).max() * 3.4e38,
            base / np.abs(base).max() * 2.0 ** -100, base / np.abs(base).max() * 2.0 ** -8]
    mixed = base.copy()
    mixed[0, 3] = 1e20
    mixed[0, 5] = 1e-30
    rows.append(mixed)
    # halves of steps: (n + 1/2) a / 127 exactly, and their neighbours
    for a in (127.0, 254.0, 1.0, 3.7):
        n = np.arange(hd) - 64 + 0.5
        y = (n / 127.0 * a).astype(np.float32)
        y[0] = a
        rows += [y[None], np.nextafter(y, np.float32(np.inf))[None], np.nextafter(y, np.float32(-np.inf))[None]]
        rows[-2][0, 0] = rows[-1][0, 0] = a
    for bad in (np.inf, -np.inf, np.nan):
        y = base.copy()
        y[0, 77] = bad
        rows.append(y)
    x = np.concatenate(rows).astype(np.float32)[:, None, :]
    c = Cache(gctx, rng, kvt, hd, 1, 0, [(7, len(x))], rows=([np.concatenate([x[:7], x])], [np.concatenate([x[:7], -x])]))
    c.write_new()
    for got, s in zip(c.read(), (1, -1)):
        np.testing.assert_array_equal(got, stored(s * x, kvt))
    c.free()


# ---------------------------------------------------------------- attention


@TILES
@TYPES
@pytest.mark.parametrize("hd,kv,heads,seqs", [
    (64, 8, 8, [(128, 1)]), (128, 8, 32, [(0, 1)]), (128, 2, 16, [(63, 1), (64, 1), (65, 1), (700, 1), (0, 1)]),
    (128, 1, 1, [(1900, 1)]), (256, 1, 3, [(100, 5), (0, 0), (3, 70)]), (64, 2, 14, [(33, 17), (1, 1), (0, 130)]),
    (128, 2, 8, [(200, 8), (59, 8)]), (128, 1, 24, [(300, 30)]), (64, 1, 64, [(5, 3)]), (128, 2, 8, [(70, 333)]),
    (128, 1, 8, [(4000, 1), (20, 3)]), (64, 1, 2, [(2500, 40)]), (128, 8, 32, [(640, 1), (1, 1), (0, 2)]),
    (64, 8, 8, [(900, 9)] * 3)])
def test_chains(gctx, kvt, hd, kv, heads, seqs):
    rng = np.random.default_rng(heads + hd)
    c = Cache(gctx, rng, kvt, hd, kv, heads, seqs)
    c.write_new()
    c.check(queries(rng, c, 2.0))
    c.free()


@TILES
@TYPES
@pytest.mark.parametrize("hd,kv,heads,seqs,window,sinks", [
    (128, 2, 8, [(300, 1), (1000, 1)], 1, 0), (128, 2, 8, [(300, 1), (1000, 3)], 64, 0), (64, 2, 8, [(500, 70)], 65, 4),
    (64, 1, 4, [(1000, 40), (20, 90)], 130, 65), (128, 1, 8, [(0, 300)], 20, 1), (128, 1, 1, [(900, 1)], 200, 64),
    (128, 1, 2, [(30, 5)], 1000, 4), (128, 1, 2, [(640, 9)], 3, 1000), (256, 1, 2, [(200, 70)], 64, 128)])
def test_windows(gctx, kvt, hd, kv, heads, seqs, window, sinks):
    rng = np.random.default_rng(window)
    c = Cache(gctx, rng, kvt, hd, kv, heads, seqs, window, sinks)
    c.write_new()
    c.check(queries(rng, c, 2.0))
    c.free()


@TILES
@TYPES
@pytest.mark.parametrize("hd,kv,heads,seqs,window,sinks", [
    (128, 2, 8, [(300, 52, 4)], 0, 0), (64, 2, 8, [(0, 33, 1), (61, 7, 3)], 0, 0), (128, 1, 8, [(900, 256, 2), (5, 3)], 0, 0),
    (128, 1, 4, [(300, 64, 2)], 5, 3), (128, 1, 4, [(0, 130, 2), (2, 40, 1)], 4, 3), (64, 1, 4, [(70, 90, 5)], 64, 66)])
def test_trees(gctx, kvt, hd, kv, heads, seqs, window, sinks):
    rng = np.random.default_rng(heads)
    seqs = [(s[0], s[1], tree(s[1], s[2])) if len(s) > 2 else s for s in seqs]
    c = Cache(gctx, rng, kvt, hd, kv, heads, seqs, window, sinks)
    c.write_new()
    c.check(queries(rng, c, 2.0))
    c.free()


@TILES
@TYPES
@pytest.mark.parametrize("qs,ks,vs", [(1e30, 1e-30, 1.0), (1e-25, 1e25, 1e30), (1.0, 1.0, 1e-28), (30.0, 3.0, 1.0),
                                      (1e3, 1e2, 1e-3), (0.0, 1.0, 1.0), (1.0, 0.0, 0.0)])
def test_values_of_every_size(gctx, kvt, qs, ks, vs):
    rng = np.random.default_rng(11)
    k, v = (rng.standard_normal((310, 2, 128)) for _ in range(2))
    c = Cache(gctx, rng, kvt, 128, 2, 8, [(270, 40)], rows=([(k * ks).astype(np.float32)], [(v * vs).astype(np.float32)]))
    c.write_new()
    c.check(queries(rng, c, qs))
    c.free()


@TILES
@TYPES
def test_large_values_in_hidden_places_change_nothing(gctx, kvt):
    """Rows that a token does not see may be huge, infinite or NaN: its output
    is bit for bit what it is without them; a token that sees one is NaN."""
    rng = np.random.default_rng(12)
    seqs, M = [(100, 50), (30, 9)], 50
    base = [[rng.standard_normal((a + b, 2, 128)).astype(np.float32) for a, b in seqs] for _ in range(2)]
    q = None
    got = {}
    for what in (None, np.nan, np.inf, 1e30):
        rows = [[x.copy() for x in y] for y in base]
        if what is not None:
            for x in rows:
                x[0][100 + 20, 1, 7] = what  # token 20 of the first sequence, kv head 1
        c = Cache(gctx, rng, kvt, 128, 2, 8, seqs, rows=rows)
        c.write_new()
        q = queries(rng, c) if q is None else q
        got[what] = c.attend(q)
        if what is None or what != 1e30:
            c.check(q)
        c.free()
    for what in (np.nan, np.inf, 1e30):
        np.testing.assert_array_equal(got[what][:20], got[None][:20])
        np.testing.assert_array_equal(got[what][20:50, :4], got[None][20:50, :4])
        np.testing.assert_array_equal(got[what][50:], got[None][50:])
    assert np.isnan(got[np.nan][20:50, 4:]).all() and np.isnan(got[np.inf][20:50, 4:]).all()


@TILES
@TYPES
def test_a_row_hidden_by_the_window(gctx, kvt):
    """NaN rows between the first tokens and the window, in pages that are read
    and in pages that are not."""
    rng = np.random.default_rng(13)
    k, v = ([rng.standard_normal((600, 1, 64)).astype(np.float32)] for _ in range(2))
    outs = []
    for poison in (False, True):
        rows = [[x[0].copy()] for x in (k, v)]
        if poison:
            for x in rows:
                x[0][4:500 - 130 + 1] = np.nan
        c = Cache(gctx, rng, kvt, 64, 1, 2, [(500, 100)], 130, 4, rows=rows)
        c.write_new()
        outs.append(c.check(np.ones((100, 128), np.float32)))
        c.free()
    np.testing.assert_array_equal(*outs)
    assert np.isfinite(outs[0]).all()


@TILES
@TYPES
def test_pages_that_held_other_things(gctx, kvt):
    """A page that another sequence left full of NaN, then used for a few tokens."""
    rng = np.random.default_rng(14)
    pool = gctx.pool(1, 1, 128, 2, kvt)
    pages = pool.take(2)
    c = Cache.__new__(Cache)
    c.ctx, c.kvt, c.hd, c.kv, c.heads, c.window, c.sinks, c.layer, c.pool = gctx, kvt, 128, 1, 4, 0, 0, 0, pool
    junk = np.full((128, 1, 128), np.nan, np.float32)
    fill = pool.plan([(pages, 0, 128)])
    c.write(fill, [junk], [junk])
    fill.free()
    c.seqs, c.new = [(pages[::-1], 0, 70, None)], 70
    c.k, c.v = ([rng.standard_normal((70, 1, 128)).astype(np.float32)] for _ in range(2))
    c.plan = pool.plan(c.seqs, 4)
    c.write_new()
    assert np.isfinite(c.check(queries(rng, c))).all()
    c.free()


@TILES
@TYPES
@pytest.mark.parametrize("pad,off", [(4, 4), (3, 0), (0, 1), (8, 2)])
def test_strides_and_alignment(gctx, kvt, pad, off):
    rng = np.random.default_rng(15)
    c = Cache(gctx, rng, kvt, 64, 2, 6, [(80, 20), (1, 3)])
    c.write_new(pad=pad, off=off)
    q = queries(rng, c)
    np.testing.assert_array_equal(c.attend(q, pad=pad, off=off), c.check(q))
    c.free()


@TILES
def test_q_k_v_in_one_matrix(gctx):
    """Rows of q | k | v as a projection leaves them, out over q's place of a
    second matrix's columns."""
    rng = np.random.default_rng(16)
    c = Cache(gctx, rng, F16, 64, 2, 4, [(10, 30)])
    q = queries(rng, c)
    w = (4 + 2 + 2) * 64
    m = Rows(gctx, np.concatenate([q, c.k[0][10:].reshape(30, -1), c.v[0][10:].reshape(30, -1)], 1), 256)
    c.plan.write(0, m.ptr + 4 * 256, m.ptr + 4 * 384, m.ld, m.ld)
    c.plan.attend(0, m.ptr, m.ptr + 4 * w, m.ld, m.ld)  # into the rows' padding
    gctx.sync()
    got = m.buf.read(np.float32, m.host.size)[:30 * m.ld].reshape(30, m.ld)[:, w:w + 256].reshape(30, 4, 64)
    np.testing.assert_array_equal(got, c.check(q))
    m.buf.free()
    c.free()


@TILES
@TYPES
def test_chunks_give_what_one_chunk_gives(gctx, kvt):
    """A prompt in chunks of uneven length over one growing table: each chunk's
    rows as of the whole prompt at once, to the bound of each."""
    rng = np.random.default_rng(17)
    whole = Cache(gctx, rng, kvt, 128, 2, 8, [(0, 200)], spare=4)
    whole.write_new()
    q = queries(rng, whole)
    want, tol = whole.want(q)
    table, at = whole.tables[0], 0
    fresh = whole.pool.take(4)
    for n in (1, 62, 1, 5, 131):
        whole.plan.set([(fresh[:(at + n + 63) // 64], at, n)], 8)
        k, v = (Rows(gctx, x[0][at:at + n]) for x in (whole.k, whole.v))
        qd, out = Rows(gctx, q[at:at + n]), Rows(gctx, np.zeros((n, 1024)))
        whole.plan.write(0, k.ptr, v.ptr)
        whole.plan.attend(0, qd.ptr, out.ptr)
        gctx.sync()
        got = out.get().reshape(n, 8, 128)
        assert (np.abs(got - want[at:at + n]) <= tol[at:at + n]).all()
        for x in (k, v, qd, out):
            x.buf.free()
        at += n
    assert len(table) == 4
    whole.free()


@TILES
@TYPES
def test_shared_prefix_pages(gctx, kvt):
    """Two sequences over one sequence's first pages, each with its own last page."""
    rng = np.random.default_rng(18)
    c = Cache(gctx, rng, kvt, 64, 1, 4, [(128, 0)], spare=2)
    own = c.pool.take(2)
    k, v = (rng.standard_normal((2, 5, 1, 64)).astype(np.float32) for _ in range(2))
    c.seqs = [(np.append(c.tables[0], own[i]), 128, 5, None) for i in range(2)]
    c.k = [np.concatenate([c.k[0], k[i]]) for i in range(2)]
    c.v = [np.concatenate([c.v[0], v[i]]) for i in range(2)]
    c.new = 10
    c.plan.set(c.seqs, 4)
    c.write_new()
    c.check(queries(rng, c))
    c.free()


def test_offsets_past_32_bits(gctx):
    """A pool of 8 GB: the last pages of its last layer."""
    rng = np.random.default_rng(19)
    pages = 8200
    pool = gctx.pool(4, 8, 128, pages, F16)
    ids = pool.take(pages)
    c = Cache.__new__(Cache)
    c.ctx, c.kvt, c.hd, c.kv, c.heads, c.window, c.sinks, c.layer, c.pool = gctx, F16, 128, 8, 8, 0, 0, 3, pool
    c.seqs, c.new = [(ids[-3:][::-1], 0, 150, None)], 150
    c.k, c.v = ([rng.standard_normal((150, 8, 128)).astype(np.float32)] for _ in range(2))
    c.plan = pool.plan(c.seqs, 8)
    c.write_new()
    c.check(queries(rng, c))
    np.testing.assert_array_equal(c.read()[0], stored(c.k[0], F16))
    c.free()


# ---------------------------------------------------------------- refusals, pool, graphs


def refused(code, f, *a, **kw):
    with pytest.raises(ftx.FtxError) as e:
        f(*a, **kw)
    assert e.value.code == code, e.value


def test_refused_calls(gctx):
    rng = np.random.default_rng(20)
    for bad in ((0, 1, 64, 1, F16), (1, 0, 64, 1, F16), (1, 1, 64, 0, F16), (1, 1, 64, (1 << 24) + 1, F16)):
        refused(-1, gctx.pool, *bad)
    for hd, t in ((80, F16), (32, Q8), (512, F16), (64, ftx.KV_F32), (64, 7)):
        refused(-2, gctx.pool, 1, 1, hd, 1, t)
    c = Cache(gctx, rng, F16, 64, 1, 2, [(70, 5)])
    c.write_new()
    m = Rows(gctx, np.zeros((5, 4 * 128)))
    host = np.zeros((5, 128), np.float32)
    p = c.plan
    refused(-1, p.write, 0, host.ctypes.data, m.ptr)
    refused(-1, p.write, 0, None, m.ptr)
    refused(-1, p.write, 0, m.ptr, m.ptr, 63, 64)
    refused(-1, p.write, 0, m.ptr + 2, m.ptr)
    refused(-5, p.write, 1, m.ptr, m.ptr)
    refused(-5, p.write, -1, m.ptr, m.ptr)
    refused(-1, p.read, 0, m.ptr, m.ptr)
    refused(-1, p.read, 0, m.ptr, m.ptr + 4 * 63, False, 512, 512)
    refused(-1, p.attend, 0, m.ptr, m.ptr)
    refused(-1, p.attend, 0, m.ptr, m.ptr + 4 * 127, 512, 512)
    refused(-1, p.attend, 0, m.ptr, m.ptr + 4 * 512, 128, 256)
    refused(-1, p.attend, 0, host.ctypes.data, m.ptr)
    refused(-1, c.pool.free)
    far = c.pool.plan([([-1, c.tables[0][1]], 70, 5)], 2, 3)
    refused(-5, far.read, 0, m.ptr, m.ptr + 4 * 256, True, 512, 512)
    far.read(0, m.ptr, m.ptr + 4 * 256, False, 512, 512)
    far.free()
    no_heads = c.pool.plan([(c.tables[0], 70, 5)])
    refused(-1, no_heads.attend, 0, m.ptr, m.ptr + 4 * 256, 512, 512)
    # a refused set leaves the plan as it was
    refused(-1, no_heads.set, [(c.tables[0][:1], 70, 5)])
    no_heads.read(0, m.ptr, m.ptr + 4 * 256, False, 512, 512)
    got = m.buf.read(np.float32, 5 * 512).reshape(5, 512)
    np.testing.assert_array_equal(got[:, :64], stored(c.k[0][70:, 0], F16))
    no_heads.free()
    m.buf.free()
    c.free()


def test_pool_bookkeeping(gctx):
    pool = gctx.pool(1, 1, 64, 5, Q8)
    a = pool.take(3)
    assert a == [0, 1, 2] and pool.available == 2
    refused(-4, pool.take, 3)
    assert pool.available == 2
    refused(-1, pool.give, [0, 0])
    refused(-1, pool.give, [1, 3])
    refused(-1, pool.give, [5])
    refused(-1, pool.give, [-1])
    assert pool.available == 2
    pool.give([1])
    assert pool.take(2) == [1, 3] and pool.available == 1
    refused(-1, pool.plan, [([4], 0, 1)])
    pool.give([0, 1, 2, 3])
    assert pool.take(5) == [0, 1, 2, 3, 4] and pool.take(0) == []
    pool.free()


def test_sequences_without_new_tokens(gctx):
    rng = np.random.default_rng(21)
    c = Cache(gctx, rng, Q8, 64, 1, 2, [(70, 0), (0, 0)])
    c.plan.write(0, None, None)
    c.plan.attend(0, None, None)
    np.testing.assert_array_equal(c.read(context=True)[1], stored(c.v[0], Q8))
    c.free()


@TILES
@TYPES
def test_two_graphs_replayed(gctx, kvt):
    """Two plans of one pool, each step captured on its own stream; replays side
    by side, with eager calls of other plans between, give the eager results."""
    hip = _hip()
    rng = np.random.default_rng(22)
    cs = [Cache(gctx, rng, kvt, 128, 2, 8, s) for s in ([(1000, 1), (300, 1)], [(1500, 20)])]
    qs = [queries(rng, c) for c in cs]
    for c in cs:
        c.write_new()
    want = [c.check(q) for c, q in zip(cs, qs)]
    held, streams = [], []
    try:
        for c, q in zip(cs, qs):
            st, graph, exe = (ctypes.c_void_p() for _ in range(3))
            assert hip.hipStreamCreate(ctypes.byref(st)) == 0
            streams.append(st)
            new = [np.concatenate([x[s[1]:] for x, s in zip(y, c.seqs)]) for y in (c.k, c.v)]
            mats = [Rows(gctx, x) for x in (*new, q, np.zeros_like(q))]
            gctx.set_stream(st.value)
            assert hip.hipStreamBeginCapture(st, 2) == 0
            c.plan.write(0, mats[0].ptr, mats[1].ptr)
            c.plan.attend(0, mats[2].ptr, mats[3].ptr)
            assert hip.hipStreamEndCapture(st, ctypes.byref(graph)) == 0
            gctx.set_stream(None)
            assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0) == 0
            held.append((st, graph, exe, mats))
            refused(-1, c.plan.set, c.seqs, 8)
        other = Cache(gctx, rng, kvt, 128, 2, 8, [(777, 9)])
        other.write_new()
        for _ in range(4):
            for *_, mats in held:
                mats[3].buf.write(mats[3].host)
            other.check(queries(rng, other))
            for st, _, exe, _ in held:
                assert hip.hipGraphLaunch(exe, st) == 0
            for st in streams:
                assert hip.hipStreamSynchronize(st) == 0
            for (*_, mats), w in zip(held, want):
                np.testing.assert_array_equal(mats[3].get().reshape(w.shape), w)
        other.free()
    finally:
        gctx.set_stream(None)
        for st, graph, exe, _ in held:
            hip.hipGraphExecDestroy(exe)
            hip.hipGraphDestroy(graph)
        for st in streams:
            hip.hipStreamSynchronize(st)
            hip.hipStreamDestroy(st)
    for *_, mats in held:
        for x in mats:
            x.buf.free()
    for c in cs:
        c.free()


def test_calls_on_another_stream_than_the_tables(gctx):
    """A plan set on one stream, behind work there, and called at once on
    another; then set again while the calls there may still run."""
    hip = _hip()
    rng = np.random.default_rng(31)
    busy = Cache(gctx, rng, Q8, 128, 2, 8, [(3000, 500)])
    busy.write_new()
    bq = Rows(gctx, queries(rng, busy))
    bo = Rows(gctx, np.zeros((busy.new, busy.heads * busy.hd), np.float32))
    c = Cache(gctx, rng, F16, 128, 2, 8, [(900, 3)])
    c.write_new()
    q = queries(rng, c)
    want = c.check(q)
    qd, out = Rows(gctx, q), Rows(gctx, np.zeros_like(q))
    st = ctypes.c_void_p()
    assert hip.hipStreamCreate(ctypes.byref(st)) == 0
    try:
        for k in range(3):
            out.buf.write(out.host)
            c.plan.set([([], 0, 0)], 8)
            for _ in range(20):
                busy.plan.attend(0, bq.ptr, bo.ptr)
            c.plan.set(c.seqs, 8)
            gctx.set_stream(st.value)
            c.plan.attend(0, qd.ptr, out.ptr)
            gctx.set_stream(None)
            c.plan.set([([], 0, 0)], 8)
            gctx.sync()
            assert hip.hipStreamSynchronize(st) == 0
            np.testing.assert_array_equal(out.get().reshape(want.shape), want)
    finally:
        gctx.set_stream(None)
        hip.hipStreamSynchronize(st)
        hip.hipStreamDestroy(st)
    for x in (bq, bo, qd, out):
        x.buf.free()
    c.free()
    busy.free()


@pytest.mark.parametrize("mode", [0, 1, 2], ids=["global", "thread", "relaxed"])
def test_capture_modes(gctx, mode):
    """A plan whose tables went up on another stream, captured in every mode."""
    hip = _hip()
    rng = np.random.default_rng(32)
    c = Cache(gctx, rng, Q8, 64, 2, 8, [(500, 2)])
    c.write_new()
    q = queries(rng, c)
    want = c.check(q)
    qd, out = Rows(gctx, q), Rows(gctx, np.zeros_like(q))
    st, graph, exe = (ctypes.c_void_p() for _ in range(3))
    assert hip.hipStreamCreate(ctypes.byref(st)) == 0
    gctx.set_stream(st.value)
    try:
        assert hip.hipStreamBeginCapture(st, mode) == 0
        c.plan.attend(0, qd.ptr, out.ptr)
        assert hip.hipStreamEndCapture(st, ctypes.byref(graph)) == 0
        assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0) == 0
        for _ in range(3):
            out.buf.write(out.host)
            assert hip.hipGraphLaunch(exe, st) == 0
            assert hip.hipStreamSynchronize(st) == 0
            np.testing.assert_array_equal(out.get().reshape(want.shape), want)
    finally:
        gctx.set_stream(None)
        hip.hipStreamSynchronize(st)
        if exe:
            hip.hipGraphExecDestroy(exe)
        if graph:
            hip.hipGraphDestroy(graph)
        hip.hipStreamDestroy(st)
    qd.buf.free(), out.buf.free()
    c.free()


def test_set_while_captured_is_refused(gctx):
    hip = _hip()
    c = Cache(gctx, np.random.default_rng(23), F16, 64, 1, 1, [(3, 1)])
    st, graph = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamCreate(ctypes.byref(st)) == 0
    try:
        gctx.set_stream(st.value)
        assert hip.hipStreamBeginCapture(st, 2) == 0
        refused(-1, c.plan.set, c.seqs, 1)
        assert hip.hipStreamEndCapture(st, ctypes.byref(graph)) == 0
    finally:
        gctx.set_stream(None)
        if graph.value:
            hip.hipGraphDestroy(graph)
        hip.hipStreamDestroy(st)
    c.plan.set(c.seqs, 1)
    c.free()


def test_traced_calls(gctx):
    c = Cache(gctx, np.random.default_rng(24), F16, 64, 1, 2, [(300, 3)])
    gctx.trace(True)
    c.write_new()
    c.check(queries(np.random.default_rng(1), c))
    tr = gctx.trace_read()
    gctx.trace(False)
    assert tr["paged_kv"]["launches"] == 1 and tr["attention"]["launches"] == 1
    c.free()
