"""Steps whose tables are built on the GPU: block tables, starts, slots and positions
against numpy, the plan's calls against the bounds of plans set from the host
(test_gpu_paged.py), faults of a step that only the GPU sees, and whole decode steps in a
graph whose lengths change between its replays."""
import ctypes

import numpy as np
import pytest

import test_gpu_paged as P
from test_gpu_paged import F16, Q8, Cache, Rows, queries, refused
from test_gpu_paged_q4 import Q4, stored4
from test_zz_no_alloc import _hip
from xwfes_amd import ftx

pytestmark = pytest.mark.gpu

I32 = np.int32
ALL = pytest.mark.parametrize("kvt", [F16, Q8, Q4], ids=["f16", "q8", "q4"])


@pytest.fixture(autouse=True)
def every_type(monkeypatch):
    by8 = P.stored
    monkeypatch.setattr(P, "stored", lambda x, kvt: stored4(x) if kvt == Q4 else by8(x, kvt))


class Lists:
    """The device arrays of a build."""

    def __init__(self, ctx, npast, M, tables, free, used=0, tokens=None, n_free=None, in_place=False, ldt=None):
        self.ctx, self.nseq, self.ldt = ctx, len(npast), ldt or tables.shape[1]
        self.tokens = tokens or int(np.sum(M))
        self.n_free = len(free) if n_free is None else n_free
        self.host = dict(npast=np.array(npast, I32), M=np.array(M, I32), tables=np.array(tables, I32),
                         free=np.array(free, I32), used=np.array([used], I32), after=np.full(1, -77, I32),
                         status=np.full(1, 55, I32), starts=np.full(self.nseq + 1, -7, I32),
                         slots=np.full(self.tokens + 3, -7, I32), positions=np.full(self.tokens + 3, -7, I32))
        self.buf = {n: ctx.buffer(max(x.nbytes, 4)) for n, x in self.host.items()}
        if in_place:
            self.buf["after"] = self.buf["used"]
        self.reset()

    def reset(self, **new):
        for n, x in new.items():
            self.host[n] = np.array(x, I32).reshape(self.host[n].shape)
        for n, x in self.host.items():
            if x.size and not (n == "after" and self.buf["after"] is self.buf["used"]):
                self.buf[n].write(x)

    def ptr(self, n):
        return self.buf[n].ptr

    def build(self, plan, skip=()):
        opt = {n + "_ptr": self.ptr(n) for n in ("starts", "slots", "positions") if n not in skip}
        plan.build(self.ptr("npast"), self.ptr("M"), self.nseq, self.ptr("tables"), self.ldt, self.ptr("free"), self.n_free,
                   self.ptr("used"), self.ptr("after"), self.ptr("status"), **opt)

    def get(self):
        self.ctx.sync()
        return {n: self.buf[n].read(I32, x.size).reshape(x.shape) for n, x in self.host.items() if x.size}

    def want(self):
        h = self.host
        t, at, starts, slots, pos = h["tables"].copy(), int(h["used"][0]), [0], [], []
        for s, (p, m) in enumerate(zip(h["npast"], h["M"])):
            for i in range((p + 63) // 64, (p + m + 63) // 64):
                t[s, i] = h["free"][at]
                at += 1
            x = np.arange(p, p + m)
            slots.append(t[s, x // 64] * 64 + x % 64)
            pos.append(x)
            starts.append(starts[-1] + m)
        pad = lambda x: np.concatenate(x + [np.full(self.tokens - starts[-1], -1, I32), np.full(3, -7, I32)])  # noqa: E731
        return dict(tables=t, after=np.array([at]), status=np.zeros(1), starts=np.array(starts), slots=pad(slots), positions=pad(pos))

    def check(self, skip=()):
        got, want = self.get(), self.want()
        for n, x in want.items():
            np.testing.assert_array_equal(got[n], self.host[n] if n in skip else x, err_msg=n)

    def refused(self, code):
        """Nothing but the fault: what the tables and the list of pages were, no tokens."""
        got, h = self.get(), self.host
        assert got["status"][0] == code
        for n in ("npast", "M", "tables", "free"):
            if n in got:
                np.testing.assert_array_equal(got[n], h[n])
        assert got["after"][0] == h["used"][0] and not got["starts"].any()
        for n in ("slots", "positions"):
            assert (got[n][:self.tokens] == -1).all() and (got[n][self.tokens:] == -7).all()

    def free(self):
        for x in {id(x): x for x in self.buf.values()}.values():
            x.free()


def lists_of(ctx, rng, lengths, used=0, spare=0, ld=2, tokens=None, pages=None, **kw):
    """Lists of sequences [(npast, M)] over pages in a random order."""
    have = [(p + 63) // 64 for p, _ in lengths]
    need = [(p + m + 63) // 64 for p, m in lengths]
    total = sum(need) + used + spare
    ids = rng.permutation(total if pages is None else pages)[:total]
    tables, at = np.full((len(lengths), max(need + [1]) + ld), -5, I32), 0
    for s, n in enumerate(have):
        tables[s, :n] = ids[at:at + n]
        at += n
    return Lists(ctx, [p for p, _ in lengths], [m for _, m in lengths], tables, ids[at:], used, tokens, **kw)


def some(rng, n, past, most):
    return [(int(2 ** rng.uniform(0, np.log2(past + 1))) - 1, int(rng.integers(0, most + 1))) for _ in range(n)]


@pytest.mark.parametrize("lengths,used,tokens", [
    ([(0, 1)], 0, None), ([(0, 0)], 0, 1), ([(63, 1), (64, 1), (65, 1)], 0, None), ([(128, 64), (0, 0), (1, 127), (0, 128)], 3, 500),
    ([(0, 1000)], 1, None), ([(100000, 1)], 0, 9), ([(640, 1)] * 16, 2, None), ((7, 20, 3000, 1), 0, None),
    ((8, 200, 900, 3), 5, 700), ((9, 1024, 500, 1), 0, None), ((10, 1025, 300, 2), 0, 4000), ((11, 4096, 130, 1), 0, None),
    ((12, 4095, 2000, 70), 0, None), ((13, 60, 20000, 300), 1, None), ((14, 1, 5000, 9000), 0, 10000)])
def test_tables(gctx, lengths, used, tokens):
    rng = np.random.default_rng(len(lengths))
    if isinstance(lengths, tuple):
        lengths = some(np.random.default_rng(lengths[0]), *lengths[1:])
    ls = lists_of(gctx, rng, lengths, used, spare=2, tokens=tokens)
    pool = gctx.pool(1, 1, 64, int(max(ls.host["tables"].max(), ls.host["free"].max())) + 1, Q4)
    most = max(max(m for _, m in lengths), 1)
    for room in (0, 1):
        plan = pool.device_plan(min(ls.nseq + 5 * room, 4096), ls.tokens, min(most + 9 * room, ls.tokens), ls.ldt + 30 * room - 2, 1)
        ls.reset()
        ls.build(plan)
        ls.check()
        ls.reset()
        ls.build(plan, skip=("slots", "starts") if room else ("positions",))
        ls.check(skip=("slots", "starts") if room else ("positions",))
        plan.free()
    ls.free()
    pool.free()


def test_used_in_place_through_many_steps(gctx):
    """Tables that grow by what one step after another takes from the list."""
    rng = np.random.default_rng(3)
    lengths = [(int(rng.integers(0, 200)), 1) for _ in range(33)]
    ls = lists_of(gctx, rng, lengths, used=4, spare=200, ld=8, tokens=33 * 40, in_place=True)
    pool = gctx.pool(1, 1, 64, 1000, F16)
    plan = pool.device_plan(33, 33 * 40, 40, ls.ldt, 1)
    for step in range(8):
        ls.build(plan)
        ls.check()
        w = ls.want()
        ls.reset(tables=w["tables"], used=w["after"], npast=ls.host["npast"] + ls.host["M"], M=rng.integers(0, 41, 33))
    ls.free(), plan.free(), pool.free()


BAD = [
    # npast, M, what else is wrong, code
    ([5, -1], [1, 1], {}, -5), ([5, 0], [1, -1], {}, -5), ([5, 0], [1, 9], {}, -5), ([5, 250], [1, 7], {}, -5),
    ([5, (1 << 31) - 1], [1, 8], {}, -5), ([5, 5], [8, 8], dict(tokens=15), -5), ([60, 60], [5, 5], dict(n_free=1), -4),
    ([60, 60], [5, 5], dict(used=2), -4), ([60, 60], [5, 5], dict(used=-1), -5), ([60, 60], [5, 5], dict(used=9), -5),
    ([100, 70], [1, 1], dict(page=(1, 0, -1)), -1), ([100, 70], [1, 1], dict(page=(1, 1, 40)), -1),
    ([100, 128], [1, 1], dict(page=(0, 0, 1 << 30)), -1), ([60, 60], [5, 5], dict(free=(1, -1)), -1),
    ([60, 60], [5, 5], dict(free=(0, 40)), -1), ([60, -3], [5, 5], dict(n_free=0), -5),
    ([100, 70], [0, 0], dict(page=(1, 0, -1)), -1), ([60, 60], [5, 5], dict(ldt=1), -5),
]


@pytest.mark.parametrize("spread", [0, 1], ids=["one", "many"])
@pytest.mark.parametrize("npast,M,wrong,code", BAD)
def test_faults_that_the_gpu_sees(gctx, npast, M, wrong, code, spread):
    """Each leaves the plan without tokens: its calls touch nothing.  By the kernel of one
    workgroup, and (among many sequences of nothing) by those of several."""
    n = 2 + 3000 * spread
    tables = np.full((n, 4), -9, I32)
    tables[:2] = np.arange(8).reshape(2, 4)
    free = np.arange(20, 23, dtype=I32)[:3]
    if "page" in wrong:
        tables[wrong["page"][:2]] = wrong["page"][2]
    if "free" in wrong:
        free[wrong["free"][0]] = wrong["free"][1]
    pool = gctx.pool(1, 1, 64, 32, Q8)
    pool.take(32)
    tokens = wrong.get("tokens", 16)
    plan = pool.device_plan(n, tokens, 8, 4, 2)
    zeros = [0] * (n - 2)
    ls = Lists(gctx, npast + zeros, M + zeros, tables, free, wrong.get("used", 0), tokens, wrong.get("n_free"), ldt=wrong.get("ldt"))
    ls.build(plan)
    ls.refused(code)
    k, out = Rows(gctx, np.ones((tokens, 64))), Rows(gctx, np.full((tokens, 128), 3.0))
    plan.write(0, k.ptr, k.ptr)
    plan.read(0, out.ptr, out.ptr + 4 * 64, False, 128, 128)
    q = Rows(gctx, np.ones((tokens, 128)))
    plan.attend(0, q.ptr, out.ptr)
    gctx.sync()
    assert (out.get() == 3.0).all()
    # no row of the pool was written
    whole = pool.plan([([0, 1, 2, 3, 4, 5, 6, 7], 0, 512)])
    back = Rows(gctx, np.full((512, 128), 5.0))
    whole.read(0, back.ptr, back.ptr + 4 * 64, False, 128, 128)
    gctx.sync()
    assert not back.get().any()
    # and a good step on the same plan works
    good = Lists(gctx, [60, 3] + zeros, [5, 1] + zeros, np.where(tables < 0, 0, tables % 32) if spread == 0 else tables * 0 + 1,
                 [20, 21, 22], 0, tokens)
    good.build(plan)
    good.check()
    for x in (k, q, out, back):
        x.buf.free()
    ls.free(), good.free(), whole.free(), plan.free(), pool.free()


def test_pages_outside_the_window_may_be_absent(gctx):
    pool = gctx.pool(1, 1, 64, 16, Q8)
    pool.take(16)
    tables = np.array([[-1, -1, -1, 3, 4, -1]], I32)
    for sinks, code in ((0, 0), (1, -1)):
        plan = pool.device_plan(1, 4, 4, 6, 2, window=70, sinks=sinks)
        ls = Lists(gctx, [300], [2], tables, [9], 0, 4)
        ls.build(plan)
        assert ls.get()["status"][0] == code
        m = Rows(gctx, np.zeros((400, 128)))
        refused(-5, plan.read, 0, m.ptr, m.ptr + 256, True, 128, 128)
        m.buf.free()
        ls.free(), plan.free()
    pool.free()


class Built(Cache):
    """A Cache whose plan for the new tokens is built on the GPU, with `spare` room."""

    def __init__(self, ctx, rng, kvt, hd, kv, heads, seqs, window=0, sinks=0, room=0, **kw):
        super().__init__(ctx, rng, kvt, hd, kv, heads, seqs, window, sinks, **kw)
        self.plan.free()
        ld = max(max(len(t) for t in self.tables), 1)
        tables, free = np.full((len(seqs), ld), -3, I32), []
        for s, (t, (npast, M)) in enumerate(zip(self.tables, seqs)):
            have = (npast + 63) // 64
            tables[s, :have] = t[:have]
            free += list(t[have:])
        most = max(max(s[1] for s in seqs), 1)
        self.room = max(self.new, 1) + 40 * room
        self.lists = Lists(ctx, [s[0] for s in seqs], [s[1] for s in seqs], tables, free, 0, self.room)
        self.plan = self.pool.device_plan(len(seqs) + 3 * room, self.room, most + 5 * room, ld + 9 * room, heads, window, sinks)
        self.lists.build(self.plan)
        self.lists.check()

    def pad(self, x, fill):
        """Rows as long as the plan's room."""
        x = np.asarray(x, np.float32).reshape(self.new, -1)
        return np.concatenate([x, np.full((self.room - len(x), x.shape[1]), fill, np.float32)])

    def write_new(self):
        new = [np.concatenate([r[s[1]:s[1] + s[2]] for r, s in zip(x, self.seqs)]) for x in (self.k, self.v)]
        mats = [Rows(self.ctx, self.pad(x, 1e30)) for x in new]
        self.plan.write(self.layer, mats[0].ptr, mats[1].ptr)
        self.ctx.sync()
        for m in mats:
            m.buf.free()

    def read(self, context=False):
        if context:
            return super().read(context=True)
        mats = [Rows(self.ctx, np.full((self.room, self.kv * self.hd), 8.0)) for _ in range(2)]
        self.plan.read(self.layer, mats[0].ptr, mats[1].ptr)
        self.ctx.sync()
        got = [m.get() for m in mats]
        for m, x in zip(mats, got):
            assert (x[self.new:] == 8).all()
            m.buf.free()
        return [x[:self.new].reshape(self.new, self.kv, self.hd) for x in got]

    def attend(self, q):
        mats = [Rows(self.ctx, self.pad(q, np.nan)), Rows(self.ctx, np.full((self.room, self.heads * self.hd), 9.0))]
        self.plan.attend(self.layer, mats[0].ptr, mats[1].ptr)
        self.ctx.sync()
        got = mats[1].get()
        assert (got[self.new:] == 9).all()
        for m in mats:
            m.buf.free()
        return got[:self.new].reshape(self.new, self.heads, self.hd)

    def free(self):
        self.lists.free()
        super().free()


@ALL
@pytest.mark.parametrize("room", [0, 1])
@pytest.mark.parametrize("hd,kv,heads,seqs,window,sinks", [
    (64, 8, 8, [(128, 1)], 0, 0), (128, 8, 32, [(0, 1)], 0, 0), (128, 2, 16, [(63, 1), (64, 1), (65, 1), (700, 1), (0, 1)], 0, 0),
    (128, 1, 1, [(5900, 1)], 0, 0), (256, 1, 3, [(100, 5), (0, 0), (3, 70)], 0, 0), (64, 2, 14, [(33, 17), (1, 1), (0, 130)], 0, 0),
    (128, 2, 8, [(70, 333), (900, 1)], 0, 0), (64, 1, 2, [(2500, 40), (100, 1)], 0, 0), (128, 8, 32, [(640, 1), (1, 1), (0, 2)], 0, 0),
    (128, 2, 8, [(300, 1), (1000, 3)], 64, 0), (64, 2, 8, [(500, 70), (9, 2)], 65, 4), (64, 1, 4, [(1000, 40), (20, 90)], 130, 65),
    (128, 1, 8, [(300, 1)] * 30, 0, 0), (256, 2, 4, [(900, 1), (1500, 60)], 0, 0), (128, 1, 4, [(4000, 200)], 0, 0)])
def test_calls(gctx, kvt, hd, kv, heads, seqs, window, sinks, room):
    rng = np.random.default_rng(hd + heads)
    c = Built(gctx, rng, kvt, hd, kv, heads, seqs, window, sinks, room)
    c.write_new()
    c.check(queries(rng, c, 2.0))
    new = [np.concatenate([r[s[1]:] for r, s in zip(x, c.seqs)]) for x in (c.k, c.v)]
    for got, x in zip(c.read(), new):
        np.testing.assert_array_equal(got, P.stored(x, kvt))
    if not window:
        for got, x in zip(c.read(context=True), (c.k, c.v)):
            np.testing.assert_array_equal(got, P.stored(np.concatenate(x), kvt))
    c.free()


def test_attention_without_heads_and_before_a_build(gctx):
    pool = gctx.pool(1, 1, 64, 4, Q4)
    pool.take(4)
    m = Rows(gctx, np.full((9, 128), 4.0))
    plan = pool.device_plan(2, 9, 9, 2)
    refused(-1, plan.attend, 0, m.ptr, m.ptr + 256)
    plan.free()
    plan = pool.device_plan(2, 9, 9, 2, 2)
    out = Rows(gctx, np.full((9, 128), 6.0))
    plan.attend(0, m.ptr, out.ptr)
    plan.write(0, m.ptr, m.ptr, 128, 128)
    plan.read(0, out.ptr, out.ptr + 256, False, 128, 128)
    gctx.sync()
    assert (out.get() == 6.0).all()
    plan.free()
    m.buf.free(), out.buf.free()
    pool.free()


def test_refused_calls(gctx):
    pool = gctx.pool(1, 2, 64, 4, Q4)
    pool.take(4)
    for bad, code in (((0, 1, 1, 1, 2), -1), ((4097, 1, 1, 1, 2), -1), ((1, 0, 1, 1, 2), -1), ((1, 1, 2, 1, 2), -1),
                      ((1, 1, 1, 0, 2), -1), ((1, 1, 1, 1, 3), -1), ((1, 1, 1, 1, 2, -1), -1), ((4096, 4096, 1, 1 << 20, 2), -5)):
        refused(code, pool.device_plan, *bad)
    plan = pool.device_plan(2, 8, 4, 2, 2)
    ls = lists_of(gctx, np.random.default_rng(1), [(3, 2), (0, 1)], tokens=8)
    a = [ls.ptr("npast"), ls.ptr("M"), 2, ls.ptr("tables"), ls.ldt, ls.ptr("free"), ls.n_free, ls.ptr("used"), ls.ptr("after"),
         ls.ptr("status")]
    host = np.zeros(8, I32)
    for i, x, code in ((0, None, -1), (1, host.ctypes.data, -1), (2, 3, -5), (2, 0, -5), (3, ls.ptr("tables") + 2, -1), (4, 0, -1),
                       (5, None, -1), (6, -1, -1), (6, 1 << 31, -1), (7, None, -1), (8, host.ctypes.data, -1), (9, None, -1)):
        refused(code, plan.build, *[x if j == i else y for j, y in enumerate(a)])
    refused(-1, plan.build, *a, slots_ptr=host.ctypes.data)
    refused(-1, plan.build, *a[:4], (1 << 40) + 1, *a[5:])
    # arrays over each other, by one number (the table's two rows, the list, and the outputs)
    end = ls.ptr("tables") + 4 * (ls.ldt + min(ls.ldt, 2))
    for i, x in ((0, ls.ptr("M")), (7, end - 4), (8, ls.ptr("free")), (8, ls.ptr("npast") + 4), (9, ls.ptr("used"))):
        refused(-1, plan.build, *[x if j == i else y for j, y in enumerate(a)])
    for n in ("npast", "M", "tables", "free", "used", "after", "status"):
        for opt in ("starts_ptr", "slots_ptr", "positions_ptr"):
            refused(-1, plan.build, *a, **{opt: ls.ptr(n)})
    refused(-1, plan.build, *a, slots_ptr=ls.ptr("slots"), positions_ptr=ls.ptr("slots") + 4 * 7)
    refused(-1, plan.build, *a, starts_ptr=ls.ptr("slots") + 4 * 8 - 4, slots_ptr=ls.ptr("slots"))
    refused(-1, plan.set, [([0], 0, 1)], 2)
    plan.build(*a)
    assert ls.get()["status"][0] == 0
    other = pool.plan([([0], 0, 1)], 2)
    refused(-1, other.build, *a)
    refused(-1, pool.free)
    other.free(), plan.free(), ls.free(), pool.free()


@ALL
def test_decode_steps_in_a_graph(gctx, kvt):
    """Build, store and attention of a step in one graph, replayed over lengths that move on
    (pages are taken as it goes, eager work of another plan between): every replay bit for bit
    as eager calls, and within the bounds."""
    hip = _hip()
    rng = np.random.default_rng(22)
    seqs, heads, kv, hd, steps = [(1000, 1), (62, 1), (0, 1), (317, 1)], 8, 2, 128, 5
    c = Built(gctx, rng, kvt, hd, kv, heads, seqs, room=1, spare=12)
    extra = c.pool.take(c.pool.available)
    ls = c.lists
    base = ls.want()
    free = np.concatenate([ls.host["free"], extra]).astype(I32)
    ls.free()
    c.plan.free()
    tables = np.full((len(seqs), 20), -1, I32)
    tables[:, :base["tables"].shape[1]] = ls.host["tables"]
    c.lists = ls = Lists(gctx, [s[0] for s in seqs], [1] * 4, tables, free, 0, 4)
    c.plan = c.pool.device_plan(4, 4, 1, 20, heads)
    mats = [Rows(gctx, np.zeros((4, n * hd))) for n in (kv, kv, heads, heads)]

    def step():
        ls.build(c.plan)
        c.plan.write(0, mats[0].ptr, mats[1].ptr)
        c.plan.attend(0, mats[2].ptr, mats[3].ptr)

    st, graph, exe = (ctypes.c_void_p() for _ in range(3))
    assert hip.hipStreamCreate(ctypes.byref(st)) == 0
    other = Cache(gctx, rng, kvt, hd, kv, heads, [(777, 9)])
    other.write_new()
    try:
        gctx.set_stream(st.value)
        assert hip.hipStreamBeginCapture(st, 2) == 0
        # a call whose build is not in the capture
        refused(-1, c.plan.attend, 0, mats[2].ptr, mats[3].ptr)
        step()
        assert hip.hipStreamEndCapture(st, ctypes.byref(graph)) == 0
        assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0) == 0
        gctx.set_stream(None)
        for i in range(steps):
            new = [rng.standard_normal((4, kv, hd)).astype(np.float32) for _ in range(2)]
            q = rng.standard_normal((4, heads * hd)).astype(np.float32)
            for m, x in zip(mats, (*new, q, q * 0 + 9)):
                m.view(m.host)[:] = x.reshape(4, -1)
                m.buf.write(m.host)
            for s in range(4):
                for rows, x in ((c.k, new[0]), (c.v, new[1])):
                    rows[s] = np.concatenate([rows[s][:seqs[s][0] + i], x[s:s + 1]])
            ls.reset()
            other.check(queries(rng, other))
            assert hip.hipGraphLaunch(exe, st) == 0
            assert hip.hipStreamSynchronize(st) == 0
            ls.check()
            got = mats[3].get()
            mats[3].buf.write(mats[3].host)
            step()
            gctx.sync()
            np.testing.assert_array_equal(mats[3].get(), got)
            c.seqs = [(t, s[0] + i, 1, None) for t, s in zip(c.tables, seqs)]
            want, tol = c.want(q)
            assert (np.abs(got.reshape(want.shape) - want) <= tol).all()
            w = ls.want()
            ls.host.update(tables=w["tables"].astype(I32), used=w["after"].astype(I32), npast=ls.host["npast"] + 1)
        # the lists run out: the graph's step does nothing
        ls.reset(used=[ls.n_free], npast=[s[0] // 64 * 64 + 64 * (s[0] % 64 > 0) for s in seqs])
        mats[3].buf.write(mats[3].host)
        assert hip.hipGraphLaunch(exe, st) == 0
        assert hip.hipStreamSynchronize(st) == 0
        ls.refused(-4)
        assert (mats[3].get() == 9).all()
    finally:
        gctx.set_stream(None)
        hip.hipStreamSynchronize(st)
        if exe:
            hip.hipGraphExecDestroy(exe)
        if graph:
            hip.hipGraphDestroy(graph)
        hip.hipStreamDestroy(st)
    other.free()
    for m in mats:
        m.buf.free()
    c.free()


def test_build_and_calls_on_two_streams(gctx):
    """Built on one stream behind work there, called at once on another; then built again for
    nothing while the calls there may still run."""
    hip = _hip()
    rng = np.random.default_rng(31)
    busy = Cache(gctx, rng, Q8, 128, 2, 8, [(3000, 500)])
    busy.write_new()
    bq, bo = Rows(gctx, queries(rng, busy)), Rows(gctx, np.zeros((busy.new, busy.heads * busy.hd), np.float32))
    c = Built(gctx, rng, F16, 128, 2, 8, [(900, 3)])
    c.write_new()
    q = queries(rng, c)
    want = c.check(q)
    none = Lists(gctx, [0], [0], c.lists.host["tables"], [], 0, c.room)
    qd, out = Rows(gctx, q), Rows(gctx, np.zeros_like(q))
    st = ctypes.c_void_p()
    assert hip.hipStreamCreate(ctypes.byref(st)) == 0
    try:
        for _ in range(3):
            out.buf.write(out.host)
            none.build(c.plan)
            for _ in range(20):
                busy.plan.attend(0, bq.ptr, bo.ptr)
            c.lists.build(c.plan)
            gctx.set_stream(st.value)
            c.plan.attend(0, qd.ptr, out.ptr)
            gctx.set_stream(None)
            none.build(c.plan)
            gctx.sync()
            assert hip.hipStreamSynchronize(st) == 0
            np.testing.assert_array_equal(out.get().reshape(want.shape), want)
    finally:
        gctx.set_stream(None)
        hip.hipStreamSynchronize(st)
        hip.hipStreamDestroy(st)
    for x in (bq, bo, qd, out):
        x.buf.free()
    none.free(), c.free(), busy.free()


def test_captures_hold_their_builds(gctx):
    """Two graphs of one plan, each with its own build and lengths, replayed in turn with eager
    steps of the plan between; a capture without a build, and another stream of a capture than
    the build's, are refused."""
    hip = _hip()
    rng = np.random.default_rng(41)
    c = Built(gctx, rng, Q4, 128, 2, 8, [(900, 3), (62, 5), (0, 0)], room=1)
    c.write_new()
    q = queries(rng, c)
    want = c.check(q)
    # the same sequences some tokens shorter: other tables of the same pages
    less = Lists(gctx, [899, 60, 0], [3, 6, 0], c.lists.host["tables"], c.lists.host["free"], 0, c.room)
    less.host["tables"][1, 0] = c.tables[1][0]
    less.reset()
    pair = [c.lists, less]
    qd = Rows(gctx, c.pad(q, np.nan))
    out = Rows(gctx, np.full((c.room, c.heads * c.hd), 9.0))

    def step(ls):
        ls.build(c.plan)
        c.plan.attend(0, qd.ptr, out.ptr)

    def taken():
        got = out.get()
        out.buf.write(out.host)
        return got

    eager = []
    for ls in pair:
        out.buf.write(out.host)
        step(ls)
        gctx.sync()
        eager.append(taken())
    np.testing.assert_array_equal(eager[0][:c.new].reshape(want.shape), want)
    assert (eager[1] != eager[0]).any() and (eager[1][9:] == 9).all()
    st, side, forked, joined = (ctypes.c_void_p() for _ in range(4))
    graphs, exes = [ctypes.c_void_p() for _ in pair], [ctypes.c_void_p() for _ in pair]
    for x in (st, side):
        assert hip.hipStreamCreate(ctypes.byref(x)) == 0
    for x in (forked, joined):
        assert hip.hipEventCreate(ctypes.byref(x)) == 0
    try:
        for ls, g, e in zip(pair, graphs, exes):
            gctx.set_stream(st.value)
            assert hip.hipStreamBeginCapture(st, 2) == 0
            refused(-1, c.plan.attend, 0, qd.ptr, out.ptr)
            step(ls)
            assert hip.hipEventRecord(forked, st) == 0
            assert hip.hipStreamWaitEvent(side, forked, 0) == 0
            gctx.set_stream(side.value)
            refused(-1, c.plan.attend, 0, qd.ptr, out.ptr)
            refused(-1, ls.build, c.plan)
            assert hip.hipEventRecord(joined, side) == 0
            assert hip.hipStreamWaitEvent(st, joined, 0) == 0
            assert hip.hipStreamEndCapture(st, ctypes.byref(g)) == 0
            assert hip.hipGraphInstantiate(ctypes.byref(e), g, None, None, 0) == 0
            gctx.set_stream(None)
        for i in (0, 1, 1, 0, 0, 1):
            out.buf.write(out.host)
            assert hip.hipGraphLaunch(exes[i], st) == 0
            assert hip.hipStreamSynchronize(st) == 0
            np.testing.assert_array_equal(taken(), eager[i])
            step(pair[1 - i])
            gctx.sync()
            np.testing.assert_array_equal(taken(), eager[1 - i])
    finally:
        gctx.set_stream(None)
        hip.hipStreamSynchronize(st)
        for e in exes:
            if e:
                hip.hipGraphExecDestroy(e)
        for g in graphs:
            if g:
                hip.hipGraphDestroy(g)
        for x in (forked, joined):
            hip.hipEventDestroy(x)
        for x in (st, side):
            hip.hipStreamDestroy(x)
    for x in (qd, out):
        x.buf.free()
    less.free(), c.free()


def test_a_page_twice_in_a_table(gctx):
    """Sequences that share their first pages, and one that has a page in two places."""
    rng = np.random.default_rng(43)
    for kvt in (F16, Q8, Q4):
        c = Built(gctx, rng, kvt, 64, 1, 4, [(256, 2), (200, 1)])
        t = c.lists.host["tables"].copy()
        t[0, 2] = t[0, 0]
        t[1, :2] = t[0, :2]
        for s, src, at in ((0, 0, 2), (1, 0, 0), (1, 1, 1)):
            for x in (c.k, c.v):
                x[s][at * 64:at * 64 + 64] = x[0][src * 64:src * 64 + 64]
            c.tables[s][at] = t[s, at]
        c.lists.reset(tables=t)
        c.lists.build(c.plan)
        c.lists.check()
        c.write_new()
        c.check(queries(rng, c, 2.0))
        c.free()
