"""The division of a step whose tables are built on the GPU, without a device:
what a plan's room refuses, and that the lists of any lengths that fit it cover
every (query row, visible page) pair once, inside the room's entries."""
import ctypes as C

import numpy as np
import pytest

from test_paged_plan import visible
from xwfes_amd import ftx

I32 = np.int32
ROOM = ("nseq", "tokens", "most", "n_pages", "pool_pages", "n_kv", "gqa", "window", "sinks", "cut_many", "slots",
        "cut_few", "wide", "few", "many", "combs", "parts", "touch")


def probe(room, lengths, n_kv=2, hd=64, pool_pages=1 << 20, cu=256, most=400000):
    """(code, message, room, items [n][8], joins [n][8]) for lengths [(npast, M)]."""
    a = ftx.PlanRoom(*room)
    npast, M = (np.array([x[i] for x in lengths], I32) for i in (0, 1))
    r, items, combs = np.zeros(len(ROOM), I32), np.zeros((most, 24), I32), np.zeros((most, 8), I32)
    msg = C.create_string_buffer(256)
    f = ftx.load().paged_build_probe
    f.restype = C.c_int
    f.argtypes = [C.c_void_p] + [C.c_int64] * 3 + [C.c_int, C.c_void_p, C.c_void_p, C.c_int64] + \
        [C.c_void_p] * 3 + [C.c_int64, C.c_char_p, C.c_int64]
    rc = f(C.byref(a), n_kv, hd, pool_pages, cu, npast.ctypes.data, M.ctypes.data, len(lengths), r.ctypes.data,
           items.ctypes.data, combs.ctypes.data, most, msg, 256)
    room = dict(zip(ROOM, r.tolist()))
    return rc, msg.value.decode(), room, items[:room["few"] + room["many"], :8], combs[:room["combs"]]


@pytest.mark.parametrize("room,code", [
    ((1, 1, 1, 1, 4, 0, 0), 0), ((0, 1, 1, 1, 4, 0, 0), -1), ((4097, 5000, 1, 1, 4, 0, 0), -1),
    ((4096, 5000, 1, 1, 4, 0, 0), 0), ((1, 0, 1, 1, 4, 0, 0), -1), ((1, 1, 0, 1, 4, 0, 0), -1),
    ((1, 1, 2, 1, 4, 0, 0), -1), ((1, 1, 1, 0, 4, 0, 0), -1), ((1, 1, 1, (1 << 24) + 1, 4, 0, 0), -1),
    ((1, 1, 1, 1 << 24, 4, 0, 0), 0), ((4096, 4096, 1, 1 << 20, 4, 0, 0), -5), ((1, 1, 1, 1, 3, 0, 0), -1),
    ((1, 1, 1, 1, -2, 0, 0), -1), ((1, 1, 1, 1, 0, 0, 0), 0), ((1, 1, 1, 1, 4, -1, 0), -1), ((1, 1, 1, 1, 4, 0, -1), -1),
    ((1, 1 << 30, 1 << 30, 1, 4, 0, 0), -5), ((1, (1 << 30) + 1, 1, 1, 0, 0, 0), -1), ((2, 1 << 27, 1 << 27, 1, 8, 0, 0), -5), ((2, 1 << 26, 1 << 26, 1, 8, 0, 0), 0),
    ((1, 1, 1, 1, 4, 1 << 40, 1 << 40), 0),
])
def test_rooms_that_are_refused(room, code):
    rc, msg, _, _, _ = probe(room, [(0, 1)], most=40 << 20 if room[1] > 1 << 20 else 400000)
    assert rc == code, msg
    assert bool(msg) == bool(code)


@pytest.mark.parametrize("lengths,code", [
    ([(0, 0)], 0), ([(-1, 1)], -5), ([(1, -1)], -5), ([(0, 9)], -5), ([(250, 7)], -5), ([(250, 6)], 0),
    ([(0, 8), (0, 8)], -5), ([(1 << 30, 1)], -5), ([((1 << 31) - 1, 8)], -5), ([(5, 3), (100, 8), (9, 0)], 0)])
def test_lengths_that_do_not_fit(lengths, code):
    assert probe((3, 15, 8, 4, 4, 0, 0), lengths)[0] == code


def check(room, lengths, n_kv, hd, cu):
    rc, msg, r, items, combs = probe(room, lengths, n_kv, hd, cu=cu)
    assert rc == 0, msg
    gqa, (window, sinks) = room[4] // n_kv, room[5:]
    places, blocks = {}, {}
    many = np.arange(len(items)) >= r["few"]
    live = items[:, 0] >= 0
    for (s, row0, i0, i1, _, _, p, nt), mn in zip(items[live], many[live]):
        assert nt == mn and row0 % (128 if mn else 16) == 0 and i0 < i1
        assert mn == (lengths[s][1] * gqa >= 65)
        for x in range((8 if mn else 1) if p >= 0 else 0):
            assert p + x not in places and 0 <= p + x < r["parts"]
            places[p + x] = (s, row0 + 16 * x)
    real = combs[combs[:, 6] > 0]
    for s, row0, part0, n, step, tok0, M, _ in real:
        assert M == lengths[s][1] and row0 < M * gqa and tok0 == sum(x[1] for x in lengths[:s]) and n >= 1
        for p in range(part0, part0 + n * step, step):
            assert p not in blocks
            blocks[p] = (s, row0)
    assert blocks == {p: at for p, at in places.items() if at[1] < lengths[at[0]][1] * gqa}
    for s, (npast, M) in enumerate(lengths):
        if M == 0:
            assert not (items[live][:, 0] == s).any()
            continue
        see = visible(npast, M, None, window, sinks)
        n = (npast + M + 63) // 64
        pad = np.zeros((M, n * 64), bool)
        pad[:, :npast + M] = see
        want = np.repeat(pad.reshape(M, n, 64).any(2), gqa, axis=0)
        got = np.zeros((M * gqa, n), int)
        for _, row0, i0, i1, sp, a, _, nt in items[live][items[live][:, 0] == s]:
            pg = np.array([i if i < sp else a + i - sp for i in range(i0, i1)])
            assert (pg >= 0).all() and (pg < n).all() and sp <= a
            got[row0:row0 + (128 if nt else 16), pg] += 1
        assert got.max(initial=0) <= 1 and (got[want] == 1).all()
    return r, real


CASES = [
    dict(lengths=[(0, 1)]), dict(lengths=[(63, 1), (64, 1), (65, 1), (0, 0), (0, 1)]), dict(lengths=[(4000, 1)]),
    dict(lengths=[(4000, 1), (10, 1), (2000, 1), (0, 0)]), dict(lengths=[(700, 100), (3, 2)], window=1),
    dict(lengths=[(700, 100), (900, 1)], window=65, sinks=4), dict(lengths=[(700, 300), (10, 200)], window=200, sinks=70),
    dict(lengths=[(3, 9)], window=5, sinks=1000), dict(lengths=[(1900, 1)], cu=1), dict(lengths=[(1900, 1)], cu=4096),
    dict(lengths=[(1500, 33), (1, 1)], n_kv=8, n_head=8), dict(lengths=[(300, 20)], n_kv=1, n_head=48),
    dict(lengths=[(1900, 260), (40, 50), (3, 2), (3000, 1)], cu=9), dict(lengths=[(3000, 64), (3000, 3), (3000, 70)], n_kv=8, n_head=32),
    dict(lengths=[(100, 5)] * 30, n_kv=1, n_head=7), dict(lengths=[(2500, 1)] * 3, n_kv=300, n_head=300, cu=60),
    dict(lengths=[(200, 64), (130, 65), (4000, 16), (5, 1)], n_kv=4, n_head=4), dict(lengths=[(6000, 2)], window=3000, sinks=64),
]


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("spare", [0, 3])
@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_items_cover_every_visible_page_once(case, spare, hd):
    n_kv, n_head, lengths = case.get("n_kv", 2), case.get("n_head", 6), case["lengths"]
    most = max(max(m for _, m in lengths), 1)
    room = (len(lengths) + spare, max(sum(m for _, m in lengths), 1) + 70 * spare, most + 20 * spare,
            max((p + m + 63) // 64 for p, m in lengths) + spare, n_head, case.get("window", 0), case.get("sinks", 0))
    check(room, lengths, n_kv, hd, case.get("cu", 256))


@pytest.mark.parametrize("seed", range(40))
def test_any_lengths_fit_the_room(seed):
    """Lengths drawn against rooms that are just large enough."""
    rng = np.random.default_rng(seed)
    n_kv, gqa = int(rng.integers(1, 9)), int(rng.choice([1, 2, 4, 7, 8, 24]))
    n = int(rng.integers(1, 40))
    most = int(rng.choice([1, 4, 30, 200]))
    lengths = [(int(2 ** rng.uniform(0, 11)) - 1, int(rng.integers(0, most + 1))) for _ in range(n)]
    window = int(rng.choice([0, 0, 1, 64, 300]))
    room = (n, max(sum(m for _, m in lengths), 1), max(max(m for _, m in lengths), 1),
            max(max((p + m + 63) // 64 for p, m in lengths), 1), n_kv * gqa, window, int(rng.choice([0, 4, 100])))
    check(room, lengths, n_kv, int(rng.choice([64, 128, 256])), int(rng.choice([1, 20, 256])))


def test_lists_are_cut_where_there_are_few():
    r, joins = check((1, 1, 1, 600, 8, 0, 0), [(38000, 1)], 8, 128, 256)
    assert len(joins) == 1 and joins[0, 3] > 48
    r, joins = check((1, 1, 1, 600, 8, 0, 0), [(38, 1)], 8, 128, 256)
    assert len(joins) == 0
    # short rooms of few sequences: whole lists for eight waves
    assert check((4, 4, 1, 8, 8, 0, 0), [(400, 1)] * 4, 8, 128, 256)[0]["wide"] == 1


def test_null_arguments_are_status_codes():
    lib = ftx.load()
    assert lib.ftx_plan_create_device(None, None, None, None) == -1
    assert lib.ftx_plan_build(None, None) == -1
