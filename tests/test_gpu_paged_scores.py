"""Attention over pages of scores of every size: a row whose largest score leads
by far is its slot's V row, also where a score's last place is worth more than
the exponent of a half; scores past fp32 make a row NaN; what one row of a tile
sees does not reach its neighbours."""
import numpy as np
import pytest

from test_gpu_paged import F16, Q8, TILES, TYPES, Cache, queries, stored, tiles, tree  # noqa: F401

pytestmark = pytest.mark.gpu


@TILES
@TYPES
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("at", [3, 100, 199])
@pytest.mark.parametrize("lo,hi", [(20, 32), (32, 60), (60, 120)])
def test_the_largest_score_takes_all(gctx, kvt, hd, at, lo, hi):
    """Scores of 2^lo to 2^hi, the others 2% below: all of the weight is one
    slot's, whose V row comes back to its weight's two halves and the rounding of a
    product and a division (2^-22 + 2^-23 + 2^-23 < 2^-20)."""
    rng = np.random.default_rng(at)
    k, v = np.zeros((330, 1, hd)), rng.uniform(0.5, 1.0, (330, 1, hd)) * rng.choice([-1, 1], (330, 1, hd))
    k[:, :, 0] = rng.uniform(0.5, 0.98, (330, 1))
    k[at, :, 0] = 1.0
    c = Cache(gctx, rng, kvt, hd, 1, 1, [(200, 130)], rows=([k.astype(np.float32)], [v.astype(np.float32)]))
    c.write_new()
    q = np.zeros((130, 1, hd), np.float32)
    q[:, 0, 0] = 2.0 ** rng.uniform(lo, hi, 130) * np.sqrt(hd) / 1.4427
    got = c.attend(q)
    want = stored(c.v[0][at], kvt)
    assert (np.abs(got - want) <= 2.0 ** -20 * np.abs(want)).all(), np.abs(got / want - 1).max()
    c.free()


@TILES
@TYPES
def test_scores_that_climb(gctx, kvt):
    """Every slot's score is above the one before by less than, or just as much
    as, an offset is worth: the newest slot leads."""
    rng = np.random.default_rng(5)
    for step in (8.0, 12.0, 15.0, 16.0, 24.0):
        n = 300
        k, v = np.zeros((n, 1, 128)), rng.uniform(0.5, 1.0, (n, 1, 128))
        # halves: k = j / 512 exactly, q so that a slot is worth `step` in log2
        k[:, :, 0] = 0.25 + np.arange(n)[:, None] / 512
        c = Cache(gctx, rng, F16, 128, 1, 1, [(200, 100)], rows=([k.astype(np.float32)], [v.astype(np.float32)]))
        c.write_new()
        q = np.zeros((100, 128), np.float32)
        q[:, 0] = step * 512 * np.sqrt(128) / 1.4426950408889634
        c.check(q)
        c.free()


@TILES
@TYPES
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_past_fp32_are_nan(gctx, kvt, sign):
    rng = np.random.default_rng(6)
    c = Cache(gctx, rng, kvt, 64, 1, 2, [(70, 40)],
              rows=([np.full((110, 1, 64), sign * 1e25, np.float32)], [np.ones((110, 1, 64), np.float32)]))
    c.write_new()
    q = np.full((40, 2, 64), 1e25, np.float32)
    q[5], q[20, 1] = 1e-25, 0.0
    got = c.attend(q)
    fine = np.zeros((40, 2), bool)
    fine[5], fine[20, 1] = True, True
    assert np.isnan(got[~fine]).all()
    np.testing.assert_allclose(got[fine], 1.0, rtol=2.0 ** -20)
    c.free()


@TILES
@TYPES
@pytest.mark.parametrize("seqs", [[(100, 9)], [(60, 50)], [(90, 30, 3)]], ids=["few", "many", "tree"])
@pytest.mark.parametrize("size", [30.0, 1e4, 1e-4])
def test_neighbours_of_a_large_slot(gctx, kvt, seqs, size):
    """K and V rows of some new tokens taken `size` times: the rows of tokens that
    do not see them stay as they were, bit for bit, in the same tile too."""
    rng = np.random.default_rng(8)
    seqs = [(s[0], s[1], tree(s[1], s[2])) if len(s) > 2 else s for s in seqs]
    npast, M = seqs[0][:2]
    base = [rng.standard_normal((npast + M, 2, 128)).astype(np.float32) for _ in range(2)]
    q, got = None, []
    for big in (False, True):
        rows = [[x.copy()] for x in base]
        if big:
            for x in rows:
                x[0][npast + M // 2 - 1] *= size
        c = Cache(gctx, rng, kvt, 128, 2, 8, seqs, rows=rows)
        c.write_new()
        q = queries(rng, c) if q is None else q
        got.append(c.attend(q))
        c.free()
    from test_paged_plan import visible
    par = seqs[0][2] if len(seqs[0]) > 2 else None
    sees = visible(npast, M, par)[:, npast + M // 2 - 1]
    assert 0 < sees.sum() < M
    np.testing.assert_array_equal(got[0][~sees], got[1][~sees])
    assert not np.array_equal(got[0][sees], got[1][sees])
