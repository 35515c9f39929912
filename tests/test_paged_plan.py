"""The host side of a paged cache's plan, without a device: what it refuses,
and that its items cover every (query row, visible page) pair once."""
import ctypes as C

import numpy as np
import pytest

from xwfes_amd import ftx

I32 = np.int32


def probe(seqs, n_kv=2, n_head=4, window=0, sinks=0, n_pages=64, taken=None, cu=256, hd=64, most=100000):
    """(code, message, items [n][8] (without their sequences), joins [n][8]) of a step's tables."""
    a, keep = ftx.plan_args(seqs, n_head, window, sinks)
    tk = np.ones(n_pages, np.uint8) if taken is None else np.asarray(taken, np.uint8)
    items, combs = np.zeros((most, 24), I32), np.zeros((most, 8), I32)
    ni, nc, msg = C.c_int64(0), C.c_int64(0), C.create_string_buffer(256)
    f = ftx.load().paged_probe
    f.restype = C.c_int
    f.argtypes = [C.c_void_p, C.c_int64, C.c_int64, C.c_int64, C.c_void_p, C.c_int, C.c_void_p,
                  C.c_void_p, C.c_void_p, C.c_void_p, C.c_int64, C.c_char_p, C.c_int64]
    rc = f(C.byref(a), n_kv, hd, n_pages, tk.ctypes.data, cu, items.ctypes.data, C.byref(ni),
           combs.ctypes.data, C.byref(nc), most, msg, 256)
    return rc, msg.value.decode(), items[:ni.value, :8], combs[:nc.value]


def tree_mask(par):
    n = len(par)
    a = np.zeros((n, n), bool)
    for i, p in enumerate(par):
        if p >= 0:
            a[i] = a[p]
        a[i, i] = True
    return a


def depths(par):
    d = []
    for p in par:
        d.append(0 if p < 0 else d[p] + 1)
    return np.array(d)


def visible(npast, M, par=None, window=0, sinks=0):
    """[M][npast + M]: what each new token sees."""
    at = np.arange(npast + M)
    if par is not None:
        at[npast:] = npast + depths(par)
    see = at[None, :] <= at[npast:, None]
    see[:, npast:] &= np.tril(np.ones((M, M), bool)) if par is None else tree_mask(par)
    if window:
        see &= (at[npast:, None] - at[None, :] < window) | (at[None, :] < sinks)
    return see


@pytest.mark.parametrize("seqs,code", [
    ([([0], 60, 4)], 0),
    ([([0], 60, 5)], -1),               # too few pages
    ([([0, 64], 60, 5)], -5),           # a page past the pool
    ([([0, -2], 60, 5)], -5),
    ([([0, -1], 60, 5)], -1),           # new tokens' page absent
    ([([-1, 1], 64, 5)], -1),           # a seen page absent
    ([([0, 0], 60, 5)], -1),            # read and written
    ([([3, 1], 64, 2), ([3, 2], 64, 2)], 0),   # a shared prefix
    ([([3], 10, 2), ([3], 10, 2)], -1),        # written twice
    ([([3], 10, 2), ([3, 4], 64, 2)], -1),     # written, then read by another
    ([([3, 4], 64, 2), ([3], 10, 2)], -1),     # read by another, then written
    ([([], 0, 0)], 0),                  # nothing at all
    ([([5], 64, 0)], 0),
    ([([5], 3, -1)], -5), ([([5], -1, 1)], -5),
    ([([0], 3, 3, [-1, 0, 2])], -1), ([([0], 3, 3, [-1, -2, 0])], -1), ([([0], 3, 3, [-1, 0, 0])], 0),
    ([(list(range(6)), 0, 257, [-1] * 257)], -1), ([(list(range(6)), 0, 256, [-1] * 256)], 0),
    ([([0], (1 << 30) + 1, 0)], -5),
    ([], -1),
])
def test_sequences_that_are_refused(seqs, code):
    rc, msg, _, _ = probe(seqs)
    assert rc == code, msg
    assert bool(msg) == bool(code)


def test_refusals_of_the_plan():
    one = [([0], 0, 1)]
    assert probe(one, n_head=3)[0] == -1          # 2 kv heads
    assert probe(one, n_head=-2)[0] == -1
    assert probe(one, window=-1)[0] == -1
    assert probe(one, sinks=-1)[0] == -1
    taken = np.ones(64)
    taken[0] = 0
    rc, msg, _, _ = probe(one, taken=taken)
    assert rc == -1 and "taken" in msg
    # outside the window a page may be absent, with sinks the first may not
    far = [([-1, -1, 2, 3], 200, 3)]
    assert probe(far, window=50)[0] == 0
    assert probe(far, window=50, sinks=1)[0] == -1
    assert probe([([0, -1, 2, 3], 200, 3)], window=50, sinks=64)[0] == 0
    assert probe([([0, -1, 2, 3], 200, 3)], window=50, sinks=65)[0] == -1
    # without attention nothing is seen
    assert probe(far, n_head=0)[0] == 0
    # more rows than a plan holds
    many = list(range(64))
    assert probe([(many, 0, 4096)] * 1, n_head=4, n_kv=2)[0] == 0
    a = [(np.zeros(1 << 20, I32), 0, 1 << 26)]
    assert probe(a, n_head=64)[0] == -5


CASES = [
    dict(seqs=[(0, 1)]), dict(seqs=[(63, 1)]), dict(seqs=[(64, 1)]), dict(seqs=[(0, 200), (5, 0), (130, 7), (64, 64)]),
    dict(seqs=[(700, 100)], window=1), dict(seqs=[(700, 100)], window=65, sinks=4),
    dict(seqs=[(700, 300), (10, 500)], window=200, sinks=70), dict(seqs=[(3, 9)], window=5, sinks=1000),
    dict(seqs=[(900, 40, 3)], window=30, sinks=2), dict(seqs=[(0, 200, 2), (70, 64, 4)], window=3, sinks=3),
    dict(seqs=[(500, 256, 1)]), dict(seqs=[(1900, 1)], cu=1), dict(seqs=[(1900, 1)], cu=4096),
    dict(seqs=[(1500, 33), (1, 1)], n_kv=8, n_head=8), dict(seqs=[(300, 20)], n_kv=1, n_head=48),
    dict(seqs=[(1900, 260), (40, 50), (3, 2)], cu=1), dict(seqs=[(1900, 260), (500, 30)], cu=9),
    dict(seqs=[(3000, 64), (3000, 64), (3000, 70)], n_kv=8, n_head=32), dict(seqs=[(250, 40)], n_kv=8, n_head=32),
]


@pytest.fixture(params=[0, 16, 128, 256], ids=["est", "r16", "r128", "r256"])
def rows(request):
    """The row tiles of sequences of 65 rows and more: by the estimate, or given."""
    force = ftx.load().paged_force_rows
    force(request.param)
    yield request.param
    force(0)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_items_cover_every_visible_page_once(case, hd, rows):
    n_kv, n_head = case.get("n_kv", 2), case.get("n_head", 6)
    window, sinks = case.get("window", 0), case.get("sinks", 0)
    seqs, pages = [], 0
    for npast, M, *b in case["seqs"]:
        n = (npast + M + 63) // 64
        par = [-1 if i < b[0] else max(i - b[0] - i % 3, 0) for i in range(M)] if b else None
        seqs.append((np.arange(pages, pages + n), npast, M, par))
        pages += n
    rc, msg, items, combs = probe(seqs, n_kv, n_head, window, sinks, n_pages=pages + 1, cu=case.get("cu", 256), hd=hd)
    assert rc == 0, msg
    gqa = n_head // n_kv
    # row tiles of 16 (all of sequences of up to 64 rows), then those of 128 or
    # 256, the longest first in each
    many = items[:, 7] > 0
    big = np.array([seqs[s][2] * gqa > 64 for s in items[:, 0]], bool)
    assert not many[~big].any()
    if rows:
        assert (many[big] == (rows > 16)).all() and (items[:, 7] <= max(min(rows, 256 if hd <= 128 else 128) // 128, 0)).all()
    assert (np.diff(many.astype(int)) >= 0).all()
    for part in (items[~many], items[many]):
        assert (np.diff((part[:, 3] - part[:, 2]) * np.where(part[:, 7] == 2, 7, 4)) <= 0).all()
    # a partial is a block of 16 rows: every place once, each joined once
    places = {}
    for (s, row0, _, _, _, _, p, nt), mn in zip(items, many):
        assert nt in ((0, 1, 2) if hd <= 128 else (0, 1))
        for x in range((8 * nt if mn else 1) if p >= 0 else 0):
            assert p + x not in places
            places[p + x] = (s, row0 + 16 * x)
    assert sorted(places) == list(range(len(places)))
    joined = {p: (c[0], c[1]) for c in combs for p in range(c[2], c[2] + c[3] * c[4], c[4])}
    assert (combs[:, 3] > 1).all() and len(joined) == combs[:, 3].sum()
    live = {p: at for p, at in places.items() if at[1] < seqs[at[0]][2] * gqa}
    assert joined == live
    for s, (_, npast, M, par) in enumerate(seqs):
        see = visible(npast, M, par, window, sinks)
        n = (npast + M + 63) // 64
        pad = np.zeros((M, n * 64), bool)
        pad[:, :npast + M] = see
        want = np.repeat(pad.reshape(M, n, 64).any(2), gqa, axis=0)
        got = np.zeros((M * gqa, n), int)
        for _, row0, i0, i1, sp, a, _, nt in items[items[:, 0] == s]:
            tr = 128 * nt or 16
            assert row0 % tr == 0 and i0 < i1
            pg = np.array([i if i < sp else a + i - sp for i in range(i0, i1)])
            assert (pg >= 0).all() and (pg < n).all() and sp <= a
            got[row0:row0 + tr, pg] += 1
        assert got.max(initial=0) <= 1 and (got[want] == 1).all()


@pytest.mark.parametrize("hd,M,npast,nseq,nt", [
    (128, 256, 4000, 16, {2}), (128, 17, 4000, 4, {1}), (128, 64, 300, 1, {0}), (64, 1, 100000, 1, {0}),
    (256, 256, 4000, 16, {1}), (128, 80, 4000, 4, {1, 2}), (128, 16, 5000, 8, {0}),
])
def test_tiles_by_the_work(hd, M, npast, nseq, nt):
    n = (npast + M + 63) // 64
    seqs = [(np.arange(i * n, i * n + n), npast, M) for i in range(nseq)]
    rc, msg, items, _ = probe(seqs, 8, 32, n_pages=nseq * n, hd=hd)
    assert rc == 0, msg
    assert set(items[:, 7]) == nt


def test_null_arguments_are_status_codes():
    lib = ftx.load()
    assert lib.ftx_pool_create(None, 1, 1, 64, 1, 1, None) == -1
    assert lib.ftx_pool_free(None) == 0 and lib.ftx_plan_free(None) == 0
    assert lib.ftx_pool_available(None) == 0
    assert lib.ftx_pool_take(None, 1, None) == -1 and lib.ftx_pool_give(None, None, 0) == -1
    assert lib.ftx_plan_create(None, None, None, None) == -1 and lib.ftx_plan_set(None, None) == -1
    assert lib.ftx_paged_write(None, 0, None, 0, None, 0) == -1
    assert lib.ftx_paged_read(None, 0, 0, None, 0, None, 0) == -1
    assert lib.ftx_paged_attention(None, 0, None, 0, None, 0) == -1
