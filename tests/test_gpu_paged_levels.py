"""Attention over pages whose V rows differ much in size, against 64-bit numpy.

A row of halves is stored as it is from 2^-8 to 65504 and under a power of two
elsewhere, so that rows of one page have scales of 1 and of 2^-23 and less side
by side.  The bound is the stores' tests', but for the term of weights so small
that their low half is lost.  Such a weight is off by 2^-25 of what the halves
are scaled to, the row's largest weight is 2^12 to 2^15, and a stored value of
2^k stands for 2^k times its scale: relative to the largest |v| that the row
sees in that kv head (the kind of row that sets the scale: 8-bit rows reach 127
steps of a scale at most 16 times below the level, halves 2^14 at most 8 times
below, rows kept as they are 2^16 under a level of larger ones), 2^-25 2^-12 2^5
= 2^-32 for each slot seen.
"""
import numpy as np
import pytest

from test_gpu_paged import F16, Q8, TILES, TYPES, Cache, queries, stored, tiles, tree  # noqa: F401
from test_paged_plan import visible

pytestmark = pytest.mark.gpu


def bound(c, q, factor=1e-2):
    """(outputs, bounds, the largest |v| seen) of Cache c's plan, each for its row and head."""
    q = np.asarray(q, np.float64).reshape(c.new, c.heads, c.hd)
    outs, tols, at, g = [], [], 0, c.heads // c.kv
    for (_, npast, M, par), k, v in zip(c.seqs, c.k, c.v):
        see = visible(npast, M, par, c.window, c.sinks)
        k64, v64 = (np.repeat(stored(x, c.kvt).astype(np.float64), g, axis=1).transpose(1, 0, 2) for x in (k, v))
        qs = q[at:at + M].transpose(1, 0, 2)
        at += M
        s = np.where(see, qs @ k64.transpose(0, 2, 1) / np.sqrt(c.hd), -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        mag = np.where(see, np.abs(qs) @ np.abs(k64).transpose(0, 2, 1) / np.sqrt(c.hd), 0).max(-1)[..., None]
        tol = np.expm1(2 * 2.0 ** -18 * mag + 2.0 ** -20 + 5 * ((npast + M) // 64 + 1) * 2.0 ** -23)
        assert tol.max() < factor
        top = np.where(see, np.abs(v64).max(-1)[:, None, :], 0).max(-1)[..., None]
        outs.append((p @ v64).transpose(1, 0, 2))
        tols.append((tol * (p @ np.abs(v64)) + see.sum(1)[:, None] * 2.0 ** -32 * top).transpose(1, 0, 2))
    return np.concatenate(outs), np.concatenate(tols)


def check(c, q):
    got = c.attend(q)
    want, tol = bound(c, q)
    err = np.abs(got - want)
    assert (err <= tol).all(), (np.argwhere(~(err <= tol))[:4], np.nanmax(err / tol))
    return got


def made(ctx, rng, kvt, hd, seqs, size, window=0, sinks=0, kv=1, heads=4, faint=(), strong=4.0):
    """A cache whose V row j of each sequence is of size size(j) in every head;
    slots faint(j) get next to no weight."""
    rows = [[], []]
    for npast, M, *_ in seqs:
        n = npast + M
        k, v = rng.standard_normal((2, n, kv, hd))
        k[:, :, 0] = strong
        if faint:
            k[faint(np.arange(n)), :, 0] = -10 * strong
        v *= (size(np.arange(n)) * np.ones(n))[:, None, None]
        rows[0].append(k.astype(np.float32)), rows[1].append(v.astype(np.float32))
    c = Cache(ctx, rng, kvt, hd, kv, heads, seqs, window, sinks, rows=rows)
    c.write_new()
    q = queries(rng, c).reshape(c.new, heads, hd)
    q[:, :, 0] = 6.0
    return c, q


SEQS = [(270, 40)]
SIZES = {
    # one row just above 2^-8 of next to no weight, the others below it
    "one-above": (lambda j: np.where(j == 30, 0.004, 1e-6), lambda j: j == 30),
    "one-above-near": (lambda j: np.where(j == 30, 0.004, 3.8e-4), lambda j: j == 30),
    "one-above-far": (lambda j: np.where(j == 30, 1.0, 1e-20), lambda j: j == 30),
    # every fifth row of ordinary size and next to no weight
    "fifths": (lambda j: np.where(j % 5 == 0, 0.02, 1e-5), lambda j: j % 5 == 0),
    # whole pages above and below, in turn
    "pages": (lambda j: np.where(j // 64 % 2, 1e-6, 0.05), lambda j: j // 64 % 2 == 0),
    "pages-from-below": (lambda j: np.where(j // 64 % 2, 0.05, 1e-6), lambda j: j // 64 % 2 == 1),
    # rows of zeros, which are of no size
    "zeros": (lambda j: np.where(j % 3 == 0, 0.0, 1e-6), lambda j: j < 0),
    "zeros-far": (lambda j: np.where(j % 3 == 0, 0.0, 1e-25), lambda j: j < 0),
    # above 65504, as they are, below 2^-8
    "three": (lambda j: np.choose(j % 3, [1e5, 0.1, 1e-5]), lambda j: j % 3 == 0),
    "three-far": (lambda j: np.choose(j % 3, [1e12, 1.0, 1e-9]), lambda j: j % 3 != 2),
    # by powers of two from 2^-30 to 2^-1
    "spread": (lambda j: 2.0 ** -(1 + j * 7 % 30), lambda j: j % 4 == 0),
}


@TILES
@TYPES
@pytest.mark.parametrize("what", SIZES)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_rows_of_two_sizes(gctx, kvt, hd, what):
    rng = np.random.default_rng(hd)
    size, faint = SIZES[what]
    c, q = made(gctx, rng, kvt, hd, SEQS, size, faint=faint)
    check(c, q)
    c.free()


@TYPES
@pytest.mark.parametrize("what", SIZES)
@pytest.mark.parametrize("seqs", [[(129, 1)], [(5, 3), (700, 1), (64, 1)], [(1500, 12)], [(100, 30, 3)], [(300, 140, 4)]],
                         ids=["one", "three", "split", "tree", "big-tree"])
def test_rows_of_two_sizes_in_other_shapes(gctx, kvt, what, seqs):
    rng = np.random.default_rng(7)
    size, faint = SIZES[what]
    seqs = [(s[0], s[1], tree(s[1], s[2])) if len(s) > 2 else s for s in seqs]
    c, q = made(gctx, rng, kvt, 64, seqs, size, kv=2, heads=8, faint=faint)
    check(c, q)
    c.free()


@TILES
@TYPES
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("small", [1e-3, 1e-6, 1e-7, 1e-20])
@pytest.mark.parametrize("window,sinks", [(130, 0), (64, 0), (100, 2), (200, 66)])
def test_large_rows_behind_the_window(gctx, kvt, hd, small, window, sinks):
    """Pages of ordinary rows that the window hides from the later tokens, whose
    rows are all small: their bound is that of the small rows."""
    rng = np.random.default_rng(window)
    edge = 256 + 64
    c, q = made(gctx, rng, kvt, hd, [(edge + 100, 90)], lambda j: np.where((j >= 66) & (j < edge), 1.0, small),
                window, sinks, faint=lambda j: (j >= 66) & (j < edge))
    check(c, q)
    c.free()
