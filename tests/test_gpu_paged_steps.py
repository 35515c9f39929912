"""Verify steps over paged caches: the same steps over the same tokens as the
oracle's (halves; LOGIT_TOL as for contiguous caches) or as the same steps in
other shapes (8-bit rows), the cache's bookkeeping (growth, truncation, commit,
window, refusals) and generate over paged caches."""
import numpy as np
import pytest

import pyoracle as P
from xwfes_amd import ftx, spec
from test_gpu_batch import LOGIT_TOL, random_tree, rel_err_rows, upload
from test_gpu_paged import refused, stored

pytestmark = pytest.mark.gpu

Q4K = dict(tok_embd=P.Q8_0, output=P.Q8_0, q=P.Q4_K, k=P.Q4_K, v=P.Q4_K, o=P.Q4_K, gate=P.Q4_K, up=P.Q4_K, down=P.Q4_K)
Q8 = dict(Q4K, q=P.Q8_0, k=P.Q8_0, v=P.Q8_0, o=P.Q8_0, gate=P.Q8_0, up=P.Q8_0)
CFG64 = P.model_cfg(2, 512, 8, 4, 64, 1024, 300, rope_theta=10000.0)
CFG128 = P.model_cfg(2, 1024, 8, 2, 128, 1024, 300, rope_theta=500000.0)


class Setup:
    def __init__(self, ctx, orc, cfg, dts, kvt=ftx.KV_F16, pages=40, max_tokens=256, seed=3, **kw):
        self.ctx, self.orc, self.cfg = ctx, orc, cfg
        self.model = P.make_model(orc, cfg, dts, seed=seed, **kw)
        self.tensors = upload(ctx, self.model)
        self.gm = ctx.model(cfg, self.tensors, max_tokens=max_tokens)
        self.pool = ctx.pool(cfg["n_layer"], cfg["n_head_kv"], cfg["head_dim"], pages, kvt)
        self.kvs, self.pages = [], pages

    def context(self, npast, cap, seed=40, kv=None, **kw):
        """A cache of `npast` random rows (halves), and the rows."""
        rng = np.random.default_rng(seed)
        kv = kv or self.gm.kv_paged(self.pool, cap, **kw)
        if kv not in self.kvs:
            self.kvs.append(kv)
        k, v = np.zeros((2,) + kv.shape, np.float16)
        k[:, :npast], v[:, :npast] = rng.standard_normal((2, kv.shape[0], npast, kv.shape[2]))
        kv.write(k, v)
        kv.truncate(npast)
        return kv, k, v

    def step(self, seqs):
        """Logits of one step: seqs = [(kv, tokens, parents, advance)]."""
        V = self.cfg["vocab"]
        bufs = [self.ctx.buffer(len(s[1]) * V * 4) for s in seqs]
        self.gm.verify_batch([(s[0], s[1], b.ptr, s[2], s[3]) for s, b in zip(seqs, bufs)])
        self.ctx.sync()
        out = [b.read(np.float32, len(s[1]) * V).reshape(-1, V) for s, b in zip(seqs, bufs)]
        for b in bufs:
            b.free()
        return out

    def free(self):
        for kv in self.kvs:
            kv.free()
        assert self.pool.available == self.pages  # every page came back
        self.gm.free()
        for t in self.tensors.values():
            t.free()
        self.pool.free()


@pytest.mark.parametrize("cfg,dts,neox,extras", [
    (CFG64, Q4K, 0, ()), (CFG128, Q8, 0, ()), (CFG128, Q4K, 1, ()),
    (CFG64, Q8, 1, ("q_bias", "k_bias", "v_bias", "q_norm", "k_norm"))])
@pytest.mark.parametrize("M,npast,tree", [(1, 0, False), (1, 130, False), (8, 61, False), (20, 64, False), (200, 5, False),
                                          (7, 60, True), (52, 100, True)])
def test_steps_equal_the_oracle(gctx, orc, cfg, dts, neox, extras, M, npast, tree):
    cfg = dict(cfg, rope_neox=neox)
    t = Setup(gctx, orc, cfg, dts, extras=extras)
    rng = np.random.default_rng(M)
    toks = rng.integers(0, 300, M).tolist()
    par = random_tree(rng, M, 10, 4) if tree else None
    kv, k, v = t.context(npast, npast + M + 9)
    got, = t.step([(kv, toks, par, True)])
    want = orc.forward(t.model, k, v, npast, toks, parents=par)
    assert rel_err_rows(got, want) < LOGIT_TOL
    kg, vg = kv.read()
    np.testing.assert_array_equal(kg[:, :npast], k[:, :npast].astype(np.float32))
    for a, b in ((kg, k), (vg, v)):
        np.testing.assert_allclose(a[:, :npast + M], b[:, :npast + M].astype(np.float32), rtol=3e-3, atol=3e-3)
    assert kv.pointers() == (None, None, npast + M)
    t.free()


@pytest.mark.parametrize("kvt", [ftx.KV_F16, ftx.KV_Q8], ids=["f16", "q8"])
def test_one_step_is_many(gctx, orc, kvt):
    """A chain of 70 tokens in one step, in steps of 1, 5 and 64, and in a
    batch beside others, leaves the same logits and rows."""
    t = Setup(gctx, orc, CFG64, Q8, kvt)
    rng = np.random.default_rng(9)
    toks = rng.integers(0, 300, 70).tolist()
    kvs = [t.context(50, 130)[0] for _ in range(3)]
    whole, = t.step([(kvs[0], toks, None, True)])
    parts = [t.step([(kvs[1], toks[a:b], None, True)])[0] for a, b in ((0, 1), (1, 6), (6, 70))]
    other, _, _ = t.context(64, 90, seed=41)
    batch = t.step([(other, toks[:9], None, False), (kvs[2], toks, None, True)])[1]
    # 8-bit rows: projections of up to 8 tokens and of more differ by some 1e-4,
    # 127 values of that move one value in a hundred across its rounding, by
    # 1/127 of the row's largest (four times the row's spread): 0.1 * 4 / 127 =
    # 3e-3 of a row's size in one row, less by averaging over the rows seen
    tol = LOGIT_TOL if kvt == ftx.KV_F16 else 5 * LOGIT_TOL
    assert rel_err_rows(np.concatenate(parts), whole) < tol
    assert rel_err_rows(batch, whole) < tol
    t.free()


def test_8_bit_rows_near_halves(gctx, orc):
    """8-bit rows move the logits by what their rounding moves the scores: the
    rows a step leaves are the oracle's rows quantised, to half a step more."""
    t = Setup(gctx, orc, CFG128, Q8, ftx.KV_Q8)
    kv, k, v = t.context(90, 130)
    toks = np.random.default_rng(2).integers(0, 300, 30).tolist()
    t.step([(kv, toks, None, True)])
    kg, vg = kv.read()
    for a, b in ((kg, k), (vg, v)):
        b4 = b[:, :90].astype(np.float32).reshape(2, 90, 2, 128)
        np.testing.assert_array_equal(a[:, :90].reshape(b4.shape), stored(b4, ftx.KV_Q8))
    orc.forward(t.model, k, v, 90, toks)
    # the first layer's new rows do not depend on the cache
    for a, b in ((kg, k), (vg, v)):
        b4 = b[0, 90:120].astype(np.float32).reshape(30, 2, 128)
        step = np.abs(b4).max(-1, keepdims=True) / 127
        assert (np.abs(a[0, 90:120].reshape(b4.shape) - b4) <= 0.51 * step + 3e-3 * np.abs(b4)).all()
    t.free()


@pytest.mark.parametrize("kvt", [ftx.KV_F16, ftx.KV_Q8], ids=["f16", "q8"])
@pytest.mark.parametrize("cfg,neox,M", [
    (CFG64, False, 1), (CFG64, True, 15), (CFG128, False, 8), (CFG128, True, 3), (CFG128, False, 16),
    (P.model_cfg(2, 1024, 4, 2, 256, 512, 300), False, 5), (P.model_cfg(2, 1024, 4, 2, 256, 512, 300), True, 12)])
def test_rows_of_a_step_are_stored_as_the_store_does(gctx, orc, kvt, cfg, neox, M):
    """The first layer's rows of a step, over the end of a page, against the fp32
    rows of the same step over a contiguous fp32 cache: bit for bit."""
    t = Setup(gctx, orc, dict(cfg, rope_neox=neox), Q8, kvt=kvt)
    npast, cap, V = 60, 90, cfg["vocab"]
    kv, k, v = t.context(npast, cap)
    full = t.gm.kv(cap, ftx.KV_F32)
    full.write(*(np.float32(x) for x in (k, v)))
    full.truncate(npast)
    buf = gctx.buffer(M * V * 4)
    for c in (kv, full):
        t.gm.verify(c, list(range(M)), buf.ptr)
    gctx.sync()
    hd = cfg["head_dim"]
    for got, want in zip(kv.read(), full.read()):
        rows = want[0, npast:npast + M].reshape(M, -1, hd)
        np.testing.assert_array_equal(got[0, npast:npast + M].reshape(M, -1, hd), stored(rows, kvt))
    buf.free()
    full.free()
    t.free()


@pytest.mark.parametrize("kvt", [ftx.KV_F16, ftx.KV_Q8], ids=["f16", "q8"])
def test_commit_of_a_tree_path(gctx, orc, kvt):
    """A path's rows move to the next slots, across a page's end; the step
    after it is the step after the chain of the path."""
    t = Setup(gctx, orc, CFG64, Q8, kvt)
    rng = np.random.default_rng(3)
    toks = rng.integers(0, 300, 20).tolist()
    par = [-1, -1, 0, 1, 2, 2, 3, 4, 5, 6, 7, 7, 8, 9, 10, 11, 12, 13, 14, 15]
    path = [1, 3, 6, 9, 13, 17]
    a, k, v = t.context(60, 90)
    b, _, _ = t.context(60, 90)
    t.step([(a, toks, par, False)])
    before = a.read()
    a.commit(path)
    after = a.read()
    for x, y in zip(before, after):
        np.testing.assert_array_equal(y[:, :60], x[:, :60])
        np.testing.assert_array_equal(y[:, 60:66], x[:, [60 + j for j in path]])
    t.step([(b, [toks[j] for j in path], None, True)])
    assert a.pointers()[2] == b.pointers()[2] == 66
    tol = LOGIT_TOL if kvt == ftx.KV_F16 else 5 * LOGIT_TOL
    assert rel_err_rows(t.step([(a, [7], None, True)])[0], t.step([(b, [7], None, True)])[0]) < tol
    # nothing moves: a chain's commit
    t.step([(a, toks[:5], None, False)])
    a.commit([0, 1])
    assert a.pointers()[2] == 69
    refused(-5, a.commit, [0, 70])
    t.free()


def test_pages_grow_and_are_given_back(gctx, orc):
    t = Setup(gctx, orc, CFG64, Q8, pages=4)
    a, b = (t.gm.kv_paged(t.pool, 1000) for _ in range(2))
    t.kvs = [a, b]
    toks = list(range(200))
    t.step([(a, toks[:64], None, True)])
    assert t.pool.available == 3
    t.step([(a, toks[:1], None, False)])
    assert t.pool.available == 2
    t.step([(a, toks[:9], None, True)])
    assert t.pool.available == 2
    t.step([(b, toks[:100], None, True)])
    assert t.pool.available == 0
    refused(-4, t.step, [(a, toks[:200], None, True)])
    assert a.pointers()[2] == 73
    a.truncate(64)
    assert t.pool.available == 1
    refused(-5, a.truncate, 65)
    a.truncate(0)
    assert t.pool.available == 2
    want, = t.step([(a, toks[:30], None, True)])
    b.truncate(0)
    got, = t.step([(b, toks[:30], None, True)])
    np.testing.assert_array_equal(got, want)
    refused(-1, t.pool.free)
    t.free()


def test_a_refused_step_takes_nothing(gctx, orc):
    t = Setup(gctx, orc, CFG64, Q8)
    kv = t.gm.kv_paged(t.pool, 100)
    w = t.gm.kv_paged(t.pool, 100, window=20)
    plain = t.gm.kv(100)
    pool2 = gctx.pool(2, 4, 64, 4)
    other = t.gm.kv_paged(pool2, 100)
    t.kvs = [kv, w, plain, other]
    for x in (w, plain, other):
        refused(-1, t.step, [(kv, [1], None, False), (x, [1], None, False)])
    refused(-1, t.step, [(kv, [1], None, False), (kv, [1], None, False)])
    refused(-5, t.step, [(kv, list(range(101)), None, False)])
    refused(-5, t.step, [(kv, [300], None, False)])
    assert t.pool.available == 40
    bad = gctx.pool(2, 4, 128, 2)
    refused(-1, t.gm.kv_paged, bad, 10)
    refused(-1, t.gm.kv_paged, t.pool, 0)
    refused(-1, t.gm.kv_paged, t.pool, 10, -1)
    bad.free()
    t.free()
    pool2.free()


def test_a_refused_batch_or_write_takes_nothing(gctx, orc):
    su = Setup(gctx, orc, CFG64, Q4K, pages=6)
    a, k, v = su.context(60, 128)
    b, _, _ = su.context(64, 128, seed=41)
    hog = su.gm.kv_paged(su.pool, 256)
    su.kvs.append(hog)
    kb = np.zeros((2,) + hog.shape, np.float16)
    spare = su.pool.take(su.pool.available - 1)
    # a grows by the last page, b finds none: neither has it
    refused(-4, su.step, [(a, [1] * 8, None, False), (b, [2] * 8, None, False)])
    assert su.pool.available == 1
    # writing all of cap takes 4 pages: refused, and a's rows stay as they were
    refused(-4, hog.write, *kb)
    big, before = su.gm.kv_paged(su.pool, 300), a.read()
    su.kvs.append(big)
    refused(-4, big.write, *np.zeros((2,) + big.shape, np.float16))
    for x, y in zip(a.read(), before):
        np.testing.assert_array_equal(x, y)
    assert su.pool.available == 1
    su.pool.give(spare)
    got = su.step([(a, [1] * 8, None, False), (b, [2] * 8, None, False)])
    assert all(np.isfinite(x).all() for x in got)
    su.free()


@pytest.mark.parametrize("M", [1, 30])
def test_window_steps(gctx, orc, M):
    """What lies outside the window and past the first tokens has no effect,
    what lies at its edge has; a window past everything is none."""
    t = Setup(gctx, orc, dict(CFG128, n_layer=2), Q8, pages=60)
    toks = np.random.default_rng(5).integers(0, 300, M).tolist()
    W, S, n = 100, 3, 400

    def run(at=None, window=W, sinks=S):
        kv = t.gm.kv_paged(t.pool, n + M, window=window, sinks=sinks)
        rng = np.random.default_rng(40)
        k, v = rng.standard_normal((2,) + kv.shape).astype(np.float32)
        if at is not None:
            v[0, at] += 3.0
        kv.write(k, v)
        kv.truncate(n)
        out, = t.step([(kv, toks, None, True)])
        held = t.pool.available
        kv.free()
        return out, held

    base, held = run()
    np.testing.assert_array_equal(run(S)[0], base)
    np.testing.assert_array_equal(run(n - W)[0], base)
    for at in (0, S - 1, n - W + 1):
        assert not np.array_equal(run(at)[0][0], base[0]), at
    full, all_held = run(window=0, sinks=0)
    np.testing.assert_array_equal(run(window=10000)[0], full)
    assert not np.array_equal(full, base)
    assert held - all_held == (n - W + 1) // 64 - 1  # pages past the first, before the window
    t.free()


def test_window_drops_pages_for_good(gctx, orc):
    t = Setup(gctx, orc, CFG64, Q8, pages=6)
    kv = t.gm.kv_paged(t.pool, 5000, window=70, sinks=2)
    t.kvs = [kv]
    rng = np.random.default_rng(6)
    for i in range(12):  # 1200 tokens through 6 pages
        t.step([(kv, rng.integers(0, 300, 100).tolist(), None, True)])
    assert kv.pointers()[2] == 1200
    kv.truncate(1195)
    refused(-5, kv.truncate, 900)
    k, _ = kv.read()
    assert k[:, :64].any() and not k[:, 64:1000].any() and k[:, 1100:1195].any()
    t.step([(kv, [5], None, True)])
    kv.truncate(0)
    assert t.pool.available == 6
    t.free()


@pytest.mark.parametrize("temp", [0.0, 0.7])
def test_generate_over_paged_caches(gctx, orc, temp):
    """Speculative generation, target and drafter over one pool: the oracle's
    tokens; then over 8-bit rows: it runs to its end."""
    def peaked(seed, gain):
        m = P.make_model(orc, CFG64, Q8, seed=seed)
        m["out_norm"]["raw"] = np.full(512, gain, np.float32).view(np.uint8).copy()
        return m

    target, draft = peaked(31, 30.0), peaked(32, 25.0)
    prompt = [3, 17, 5, 40, 11, 9, 30, 2, 21]
    want, st = orc.generate(target, draft, prompt, 30, spec_k=4, temp=temp, cap=128)
    models = []
    for m in (target, draft):
        tensors = upload(gctx, m)
        gm = gctx.model(CFG64, tensors, max_tokens=8)
        gm.owned = list(tensors.values())
        models.append(gm)
    for kvt in (ftx.KV_F16, ftx.KV_Q8):
        pool = gctx.pool(2, 4, 64, 6, kvt)
        tkv, dkv = (m.kv_paged(pool, 128) for m in models)
        drafter = spec.DraftModelDrafter(gctx, models[1], dkv)
        got, stats = spec.generate(gctx, models[0], tkv, drafter, prompt, 30, spec_k=4, temp=temp)
        if kvt == ftx.KV_F16:
            assert got == want and stats == st
        assert len(got) >= 30
        drafter.free()
        for x in (tkv, dkv):
            x.free()
        assert pool.available == 6
        pool.free()
    for m in models:
        m.free()
