"""Caches held in 4 bits, and the tables of a step built on the GPU, as cases to time and compare.

A cache of 4-bit rows holds twice the tokens of an 8-bit one. A row of head_dim values is cut into
blocks of 32; in fp32, every operation rounded to nearest,

  t_b = max over the block of max(x, 0) (1/7) and max(-x, 0) / 8      (1/7: the float next to it)
  T = the largest t_b,  s = T / 255,  c_b = min(255, ceil(t_b (255 / T)))
  q = x (1 / (c_b s)) to the nearest integer, ties to even            (-8 .. 7)

and x is held as q c_b s. Four kinds of work come of it, for every layer of every step or once a step:

  store   the new tokens' rows are quantised as they are written, and read back
  read    whole contexts are read back
  attend  the new tokens attend to their sequences' pages: one token of many sequences, drafts
          (chains and trees), chunks of prompts; with a sliding window and a few first tokens
          that stay visible, or without
  tables  block tables, slots and positions of a step from the lengths that the GPU holds
  step    tables, store and attention of one step, with no word from the host

Head layouts are those of bench.py's models (8 heads of 64; 32 heads of 64 or 128 over 8; 64 of
128 over 8).

listed() / draw(rng): the cases; prepare(case, seed): a program's state; run(state): one pass;
exact(case, seed): the same outputs in 64 bits.
"""
import math

import numpy as np
import torch

own = False
DEV = "cuda"
PAGE = 64
BLOCK = 32
TINY = dict(heads=8, kv=8, hd=64)
LLAMA_1B = dict(heads=32, kv=8, hd=64)
LLAMA_8B = dict(heads=32, kv=8, hd=128)
LLAMA_70B = dict(heads=64, kv=8, hd=128)


def listed():
    return [
        # the smallest calls: one sequence's next token, its row into the cache
        dict(name="store-1-q4", kind="store", seqs=1, M=1, ctx=2047, ragged=0.0, **LLAMA_8B),
        # a prompt's chunk, its first page partly filled by the chunk before
        dict(name="store-2000-q4", kind="store", seqs=1, M=2000, ctx=37, ragged=0.0, **LLAMA_8B),
        # four whole contexts handed on
        dict(name="read-4x16k-q4", kind="read", seqs=4, M=0, ctx=16384, ragged=0.3, **LLAMA_8B),
        # one token of the tiny model after its 128-token prompt: latency
        dict(name="attend-1-tiny-q4", kind="attend", seqs=1, M=1, ctx=128, ragged=0.0, tree=0, window=0, sinks=0,
             **TINY),
        # a decode step of 16 sequences of uneven length
        dict(name="attend-16x1-q4", kind="attend", seqs=16, M=1, ctx=8191, ragged=0.9, tree=0, window=0, sinks=0,
             **LLAMA_8B),
        # one long document, one token
        dict(name="attend-1x128k-q4", kind="attend", seqs=1, M=1, ctx=131071, ragged=0.0, tree=0, window=0, sinks=0,
             **LLAMA_70B),
        # four 64-node draft trees at context 8192
        dict(name="attend-tree4x64-q4", kind="attend", seqs=4, M=64, ctx=8192, ragged=0.0, tree=4, window=0, sinks=0,
             **LLAMA_70B),
        # chunks of three prompts of uneven length in one step
        dict(name="attend-3x1500-q4", kind="attend", seqs=3, M=1500, ctx=4000, ragged=0.6, tree=0, window=0, sinks=0,
             **LLAMA_8B),
        # 8-token drafts under a window, far past it
        dict(name="window-16x8-q4", kind="attend", seqs=16, M=8, ctx=16000, ragged=0.5, tree=0, window=4096, sinks=4,
             **LLAMA_1B),
        # the next token of 16 sequences: some of them need a page
        dict(name="tables-16x1", kind="tables", seqs=16, M=1, ctx=8191, ragged=0.9),
        # a full batch in which chunks of prompts and single tokens meet
        dict(name="tables-512x48", kind="tables", seqs=512, M=48, ctx=16384, ragged=1.0),
        # a whole decode step of 32 sequences in a loop that the host does not enter
        dict(name="step-32x1-q4", kind="step", seqs=32, M=1, ctx=4096, ragged=0.9, window=0, sinks=0, **LLAMA_8B),
    ]


def _log_int(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    kind = rng.choice(["store", "read", "attend", "attend", "window", "window", "tables", "step"])
    ragged = round(rng.choice([0.0, rng.random()]), 2)
    c = dict(kind="attend" if kind == "window" else kind, ragged=ragged)
    if kind == "tables":
        seqs = _log_int(rng, 1, 512)
        return dict(c, seqs=seqs, M=_log_int(rng, 1, max(1, min(2048, 16384 // seqs))), ctx=_log_int(rng, 1, 16384))
    if kind in ("store", "read"):
        seqs = _log_int(rng, 1, 32)
        c.update(seqs=seqs, M=0 if kind == "read" else max(1, _log_int(rng, 1, 2000) // seqs),
                 ctx=_log_int(rng, 1, 65536) // seqs + 1)
        return dict(c, **rng.choice([TINY, LLAMA_1B, LLAMA_8B]))
    shape = rng.choice([TINY, LLAMA_1B, LLAMA_8B, LLAMA_8B, LLAMA_70B])
    window = _log_int(rng, 1, 4096) if kind == "window" or (kind == "step" and rng.random() < 0.3) else 0
    sinks = rng.choice([0, 1, 4, 65]) if window else 0
    if kind == "step":
        seqs = _log_int(rng, 1, 64)
        return dict(c, seqs=seqs, M=rng.choice([1, 1, rng.randint(2, 12)]), ctx=_log_int(rng, 1, 8192), window=window,
                    sinks=sinks, **shape)
    use = rng.choice(["decode", "draft", "tree", "chunk"])
    if use == "decode":
        seqs, M, tree = _log_int(rng, 1, 64), 1, 0
        ctx = min(_log_int(rng, 1, 131072), 262144 // seqs)
    elif use == "draft":
        seqs, M, tree = _log_int(rng, 1, 16), rng.randint(2, 16), 0
        ctx = _log_int(rng, 1, 16384)
    elif use == "tree":
        seqs, M, tree = rng.randint(1, 4), rng.randint(4, 64), rng.choice([2, 4])
        ctx = _log_int(rng, 1, 8192)
    else:
        shape = rng.choice([TINY, LLAMA_1B, LLAMA_8B])
        seqs, tree = rng.randint(1, 3), 0
        M, ctx = _log_int(rng, 17, 3000 // seqs), _log_int(rng, 1, 4000)
    return dict(c, seqs=seqs, M=M, ctx=ctx, tree=tree, window=window, sinks=sinks, **shape)


# ---------------------------------------------------------------- a case's sizes


def _spread(n, longest, ragged, start):
    """n lengths up to `longest`, spread over its last part `ragged` (the first is the longest)."""
    return [max(1, int(longest * (1.0 - ragged * ((start + s) * 0.6180339887 % 1.0)))) if longest else 0
            for s in range(n)]


def _sizes(case):
    """(committed, new) tokens of every sequence."""
    n = case["seqs"]
    past = _spread(n, case["ctx"], case["ragged"], 0)
    if case["kind"] in ("tables", "step"):
        # (not in step with the contexts: sequences end anywhere in their pages)
        return past, _spread(n, case["M"], case["ragged"], 5)
    return past, _spread(n, case["M"], 0.0 if case.get("tree") else case["ragged"], 0)


def _pages(n):
    return (n + PAGE - 1) // PAGE


def _parents(M, tree):
    """A draft tree of M nodes: `tree` roots, then each node below one of the last 2 tree ones."""
    return [-1 if i < tree else i - tree - (i * 7 % tree if i >= 2 * tree else 0) for i in range(M)]


def _depths(par):
    d = []
    for p in par:
        d.append(0 if p < 0 else d[p] + 1)
    return d


def _ancestors(par):
    a = np.zeros((len(par), len(par)), bool)
    for i, p in enumerate(par):
        if p >= 0:
            a[i] = a[p]
        a[i, i] = True
    return a


def _seen(past, M, par, window, sinks):
    """visible[i, j] of one sequence: new token i, slot j."""
    at = np.arange(past + M)
    if par is not None:
        at[past:] = past + np.array(_depths(par))
    see = at[None, :] <= at[past:, None]
    see[:, past:] &= np.tril(np.ones((M, M), bool)) if par is None else _ancestors(par)
    if window:
        see &= (at[past:, None] - at[None, :] < window) | (at[None, :] < sinks)
    return see


# ---------------------------------------------------------------- inputs


def _rows(case, seed, key, total):
    """K and V rows [total][kv][hd]: keys with a few strong channels, as models have them."""
    g = torch.Generator(device=DEV).manual_seed(seed * 8 + key)
    k = torch.randn(total, case["kv"], case["hd"], device=DEV, generator=g)
    v = torch.randn(total, case["kv"], case["hd"], device=DEV, generator=g)
    k[:, :, ::19] *= 4.0
    return k, v


def _inputs(case, seed):
    """Context rows, new rows, queries; rows of sequences one after another."""
    past, new = _sizes(case)
    kc, vc = _rows(case, seed, 0, sum(past))
    kn, vn = _rows(case, seed, 1, sum(new))
    g = torch.Generator(device=DEV).manual_seed(seed * 8 + 2)
    q = torch.randn(sum(new), case["heads"], case["hd"], device=DEV, generator=g)
    return kc, vc, kn, vn, q


def _order(case, seed, total):
    """The pool's pages in the order in which the sequences came by them."""
    return np.random.RandomState(seed % (1 << 31)).permutation(total)


def _lists(case, seed):
    """What a step's tables are built from: the lengths, the tables so far (-1: no page yet), the
    pages that the program set aside for new tokens and how many of them are used up."""
    past, new = _sizes(case)
    ld = max(_pages(p + m) for p, m in zip(past, new)) + 1
    held = [_pages(p) for p in past]
    more = sum(_pages(p + m) - h for p, m, h in zip(past, new, held))
    used = 3
    order = _order(case, seed, sum(held) + more + used + 2).astype(np.int32)
    tables, at = np.full((case["seqs"], ld), -1, np.int32), 0
    for s, h in enumerate(held):
        tables[s, :h] = order[at:at + h]
        at += h
    return dict(npast=np.array(past, np.int32), M=np.array(new, np.int32), tables=tables, free=order[at:],
                used=np.array([used], np.int32)), order


class _Held:
    """The library's handles of one state."""

    def __init__(self, *things):
        self.things = things

    def __del__(self):
        for t in self.things:
            t.free()


_context = []


def _ctx():
    if not _context:
        from xwfes_amd import ftx

        _context.append(ftx.Context(0))
    return _context[0]


def _slots(pages, first, count):
    """(page, slot in page) of `count` tokens from position `first` of one sequence."""
    at = np.arange(first, first + count)
    return pages[at // PAGE], at % PAGE


def _places(tables, first, count):
    got = [_slots(t, f, n) for t, f, n in zip(tables, first, count)]
    return tuple(torch.from_numpy(np.concatenate([g[i] for g in got])).to(DEV).long() for i in (0, 1))


def _plain_cache(case, n_pages):
    shape = (n_pages, PAGE, case["kv"])
    st = {}
    for n in ("K", "V"):
        st[n] = torch.zeros(*shape, case["hd"], dtype=torch.int8, device=DEV)
        st[n + "c"] = torch.zeros(*shape, case["hd"] // BLOCK, dtype=torch.uint8, device=DEV)
        st[n + "s"] = torch.zeros(shape, device=DEV)
    return st


def prepare(case, seed):
    if case["kind"] == "tables":
        return _prepare_tables(case, seed)
    if case["kind"] == "step":
        return _prepare_step(case, seed)
    past, new = _sizes(case)
    S, kv, hd = case["seqs"], case["kv"], case["hd"]
    kc, vc, kn, vn, q = _inputs(case, seed)
    need = [_pages(p + m) for p, m in zip(past, new)]
    order = _order(case, seed, sum(need))
    ends = np.cumsum([0] + need)
    tables = [order[ends[s]:ends[s + 1]] for s in range(S)]
    par = _parents(case["M"], case["tree"]) if case.get("tree") else None
    window, sinks = case.get("window", 0), case.get("sinks", 0)
    attend = case["kind"] == "attend"
    st = dict(case=case, kn=kn, vn=vn, q=q)
    if own:
        from xwfes_amd import ftx

        ctx = _ctx()
        pool = ctx.pool(1, kv, hd, sum(need), ftx.KV_Q4)
        ids = np.array(pool.take(sum(need)))
        seqs = [(ids[tables[s]].tolist(), past[s], new[s], par) for s in range(S)]
        if case["kind"] != "store":
            fill = pool.plan([(t, 0, p, None) for t, p, m, _ in seqs])
            fill.write(0, kc.data_ptr(), vc.data_ptr())
            fill.free()
        plan = pool.plan(seqs, n_head=case["heads"], window=window, sinks=sinks)
        if attend:
            plan.write(0, kn.data_ptr(), vn.data_ptr())
        ctx.sync()
        rows = sum(past) + sum(new) if case["kind"] == "read" else sum(new)
        st.update(plan=plan, held=_Held(plan, pool), out=torch.empty_like(q),
                  k=torch.empty(rows, kv, hd, device=DEV), v=torch.empty(rows, kv, hd, device=DEV))
        return st
    st.update(_plain_cache(case, sum(need)))
    zero = [0] * S
    st["new"] = _places(tables, past, new)
    st["all"] = _places(tables, zero, [p + m for p, m in zip(past, new)])
    if case["kind"] != "store":
        _plain_store(st, _places(tables, zero, past), kc, vc)
    if attend:
        _plain_store(st, st["new"], kn, vn)
        st.update(_plain_plan(case, past, new, tables, par, window, sinks))
    return st


def _prepare_tables(case, seed):
    lists, order = _lists(case, seed)
    past, new = _sizes(case)
    st = dict(case=case, ntok=sum(new), most=max(new), **{k: torch.from_numpy(v).to(DEV) for k, v in lists.items()})
    if own:
        from xwfes_amd import ftx

        ctx = _ctx()
        # (the smallest pool of that many pages: the tables alone are built)
        pool = ctx.pool(1, 1, 64, len(order), ftx.KV_Q4)
        pool.take(len(order))
        plan = pool.device_plan(case["seqs"], sum(new), max(new), lists["tables"].shape[1], n_head=1)
        st.update(plan=plan, held=_Held(plan, pool))
        st.update(_results(case, sum(new)))
    return st


def _results(case, ntok):
    """Where a step's tables go beside the block tables themselves."""
    z = lambda n: torch.zeros(n, dtype=torch.int32, device=DEV)  # noqa: E731
    return dict(starts=z(case["seqs"] + 1), slots=z(ntok), positions=z(ntok), after=z(1), status=z(1))


def _prepare_step(case, seed):
    lists, order = _lists(case, seed)
    past, new = _sizes(case)
    kc, vc, kn, vn, q = _inputs(case, seed)
    st = dict(case=case, kn=kn, vn=vn, q=q, ntok=sum(new), most=max(new),
              **{k: torch.from_numpy(v).to(DEV) for k, v in lists.items()})
    tables = [t[t >= 0] for t in lists["tables"]]
    if own:
        from xwfes_amd import ftx

        ctx = _ctx()
        pool = ctx.pool(1, case["kv"], case["hd"], len(order), ftx.KV_Q4)
        pool.take(len(order))
        fill = pool.plan([(t.tolist(), 0, p, None) for t, p in zip(tables, past)])
        fill.write(0, kc.data_ptr(), vc.data_ptr())
        fill.free()
        plan = pool.device_plan(case["seqs"], sum(new), max(new), lists["tables"].shape[1], n_head=case["heads"],
                                window=case["window"], sinks=case["sinks"])
        ctx.sync()
        st.update(plan=plan, held=_Held(plan, pool), out=torch.empty_like(q))
        st.update(_results(case, sum(new)))
        return st
    st.update(_plain_cache(case, len(order)))
    _plain_store(st, _places(tables, [0] * case["seqs"], past), kc, vc)
    return st


def _plain_plan(case, past, new, tables, par, window, sinks):
    """Padded index tensors of a batch: every sequence's pages that any of its new tokens
    sees, the slots' and tokens' positions, the rows of the packed queries."""
    S, Mm = case["seqs"], max(new)
    lo = [max(0, p - window + 1) // PAGE if window else 0 for p in past]
    vis = [sorted(set(range(0, min(_pages(sinks), len(t)))) | set(range(l, len(t)))) for l, t in zip(lo, tables)]
    Pv = max(len(v) for v in vis)
    page, slot = np.zeros((S, Pv), np.int64), np.full((S, Pv * PAGE), 1 << 40)
    where, qi, live = np.full((S, Pv * PAGE), 1 << 40), np.zeros((S, Mm), np.int64), np.zeros((S, Mm), bool)
    at, first = np.zeros((S, Mm), np.int64), 0
    dep = np.array(_depths(par)) if par is not None else np.arange(Mm)
    for s in range(S):
        page[s, :len(vis[s])] = tables[s][vis[s]]
        sl = (np.array(vis[s])[:, None] * PAGE + np.arange(PAGE)).reshape(-1)
        sl[sl >= past[s] + new[s]] = 1 << 40
        slot[s, :sl.size] = sl
        draft = (sl >= past[s]) & (sl < 1 << 40)
        where[s, :sl.size] = np.where(draft, past[s] + dep[np.clip(sl - past[s], 0, Mm - 1)], sl)
        qi[s, :new[s]] = first + np.arange(new[s])
        live[s, :new[s]] = True
        at[s] = past[s] + dep[:Mm]
        first += new[s]
    st = dict(page=page, slot=slot, where=where, qi=qi, live=live, at=at, past=np.array(past)[:, None])
    if par is not None:
        st["anc"] = _ancestors(par)
    return {k: torch.from_numpy(v).to(DEV) for k, v in st.items()}


# ---------------------------------------------------------------- the plain forms


def _quantise(x):
    """Rows of hd values as (q, c, s). Quotients and the rounding's border in 64 bits, rounded to 32 where the
    definition rounds."""
    b = x.reshape(*x.shape[:-1], -1, BLOCK)
    t = torch.maximum(b.amax(-1).clamp_min(0.0) * (1.0 / 7.0), (-b).amax(-1).clamp_min(0.0) * 0.125)
    T = t.amax(-1, keepdim=True).double().clamp_min(2.0 ** -110)
    s = (T / 255.0).float()
    c = (t.double() * (255.0 / T).float().double()).float().ceil().clamp_max(255.0)
    r = (1.0 / (c * s).double()).float()
    q = torch.round((b.double() * r[..., None].double()).float())
    q = torch.where(c[..., None] > 0, q, torch.zeros_like(q))
    return q.reshape(x.shape).to(torch.int8), c.to(torch.uint8), s[..., 0]


def _plain_store(st, places, k, v):
    for n, x in (("K", k), ("V", v)):
        st[n][places], st[n + "c"][places], st[n + "s"][places] = _quantise(x)


def _held(st, n, at):
    """What the rows at `at` of K or V stand for."""
    q = st[n][at].float()
    q = q.reshape(*q.shape[:-1], -1, BLOCK) * st[n + "c"][at].float()[..., None]
    return q.flatten(-2) * st[n + "s"][at][..., None]


def _plain_read(st, places):
    return [_held(st, n, places) for n in ("K", "V")]


def _plain_attend(st, c):
    S, Mm = st["qi"].shape
    kv, hd, g = c["kv"], c["hd"], c["heads"] // c["kv"]
    k, v = [_held(st, n, st["page"]).reshape(S, -1, kv, hd).transpose(1, 2) for n in ("K", "V")]
    q = st["q"][st["qi"]].reshape(S, Mm, kv, g, hd).permute(0, 2, 1, 3, 4).reshape(S, kv, Mm * g, hd)
    see = st["where"][:, None, :] <= st["at"][:, :, None]
    if "anc" in st:
        node = (st["slot"] - st["past"]).clamp(0, Mm - 1)
        see &= (st["slot"] < st["past"])[:, None, :] | st["anc"][:, node].transpose(0, 1)
        see &= (st["slot"] < 1 << 40)[:, None, :]
    if c["window"]:
        see &= (st["at"][:, :, None] - st["where"][:, None, :] < c["window"]) | (st["where"] < c["sinks"])[:, None, :]
    s = (q @ k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(hd))
    s = s.reshape(S, kv, Mm, g, -1).masked_fill_(~see[:, None, :, None, :], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).reshape(S, kv, Mm * g, -1)
    o = (p @ v.contiguous()).reshape(S, kv, Mm, g, hd).permute(0, 2, 1, 3, 4).reshape(S, Mm, c["heads"], hd)
    return o[st["live"]]


def _plain_tables(st):
    """Block tables with the new pages, starts, slots, positions, pages used, status: all int32."""
    npast, M, tables = st["npast"].long(), st["M"].long(), st["tables"]
    have, want = (npast + PAGE - 1) // PAGE, (npast + M + PAGE - 1) // PAGE
    first = st["used"].long() + torch.cumsum(want - have, 0) - (want - have)
    col = torch.arange(tables.shape[1], device=DEV)
    fresh = (col >= have[:, None]) & (col < want[:, None])
    at = (first[:, None] + col - have[:, None]).clamp(0, st["free"].numel() - 1)
    tables = torch.where(fresh, st["free"][at], tables)
    ends = torch.cumsum(M, 0)
    seq = torch.repeat_interleave(torch.arange(M.numel(), device=DEV), M, output_size=st["ntok"])
    pos = torch.arange(st["ntok"], device=DEV) - (ends - M)[seq] + npast[seq]
    slots = tables[seq, pos // PAGE] * PAGE + pos % PAGE
    after = st["used"] + (want - have).sum()
    bad = (after > st["free"].numel()) | (want > tables.shape[1]).any()
    starts = torch.cat([ends - M, ends[-1:]])
    return dict(tables=tables, starts=starts.int(), slots=slots.int(), positions=pos.int(), after=after.int(),
                status=bad.int())


def _plain_step(st):
    t = _plain_tables(st)
    c = st["case"]
    _plain_store(st, (t["slots"].long() // PAGE, t["slots"].long() % PAGE), st["kn"], st["vn"])
    col = torch.arange(st["most"], device=DEV)
    live = col < st["M"][:, None]
    where = torch.arange(t["tables"].shape[1] * PAGE, device=DEV).expand(c["seqs"], -1)
    view = dict(st, page=t["tables"].long().clamp_min(0), where=where, at=st["npast"].long()[:, None] + col, live=live,
                qi=(t["starts"][:-1].long()[:, None] + col).clamp_max(st["ntok"] - 1))
    return dict(t, out=_plain_attend(view, c))


def _own_tables(st):
    """The library's: block tables in place, the rest where prepare() said."""
    t = st["tables"]
    st["plan"].build(st["npast"].data_ptr(), st["M"].data_ptr(), st["case"]["seqs"], t.data_ptr(), t.shape[1],
                     st["free"].data_ptr(), st["free"].numel(), st["used"].data_ptr(), st["after"].data_ptr(),
                     st["status"].data_ptr(), starts_ptr=st["starts"].data_ptr(), slots_ptr=st["slots"].data_ptr(),
                     positions_ptr=st["positions"].data_ptr())
    return {n: st[n] for n in ("tables", "starts", "slots", "positions", "after", "status")}


def run(st):
    kind = st["case"]["kind"]
    if own:
        plan = st["plan"]
        if kind == "tables":
            return _own_tables(st)
        if kind == "step":
            t = _own_tables(st)
            plan.write(0, st["kn"].data_ptr(), st["vn"].data_ptr())
            plan.attend(0, st["q"].data_ptr(), st["out"].data_ptr())
            return dict(t, out=st["out"])
        if kind == "attend":
            plan.attend(0, st["q"].data_ptr(), st["out"].data_ptr())
            return st["out"]
        if kind == "store":
            plan.write(0, st["kn"].data_ptr(), st["vn"].data_ptr())
        plan.read(0, st["k"].data_ptr(), st["v"].data_ptr(), context=kind == "read")
        return st["k"], st["v"]
    if kind == "tables":
        return _plain_tables(st)
    if kind == "step":
        return _plain_step(st)
    if kind == "attend":
        return _plain_attend(st, st["case"])
    if kind == "store":
        _plain_store(st, st["new"], st["kn"], st["vn"])
        return tuple(_plain_read(st, st["new"]))
    return tuple(_plain_read(st, st["all"]))


# ---------------------------------------------------------------- the least work, and 64 bits


def _row_bytes(case):
    return case["kv"] * (case["hd"] // 2 + case["hd"] // BLOCK + 4)


def work(case):
    past, new = _sizes(case)
    nbytes = flops = 0.0
    if case["kind"] in ("tables", "step"):
        fresh = sum(_pages(p + m) - _pages(p) for p, m in zip(past, new))
        # lengths, starts, slots and positions, the page that a sequence is in, new pages read and written
        nbytes += 16.0 * case["seqs"] + 8.0 * sum(new) + 8.0 * fresh
        flops += 4.0 * sum(new)
        if case["kind"] == "tables":
            return dict(bytes=nbytes, flops=flops)
    rb, wide = _row_bytes(case), 4 * case["kv"] * case["hd"]
    if case["kind"] in ("store", "read", "step"):
        rows = sum(past) + sum(new) if case["kind"] == "read" else sum(new)
        passes = 2 if case["kind"] == "store" else 1
        nbytes += passes * 2 * rows * (rb + wide)
        flops += passes * 4 * rows * case["kv"] * case["hd"]
        if case["kind"] != "step":
            return dict(bytes=nbytes, flops=flops)
    par = _parents(case["M"], case["tree"]) if case.get("tree") else None
    for p, m in zip(past, new):
        see = _seen(p, m, par, case["window"], case["sinks"])
        nbytes += 2.0 * rb * int(see.any(0).sum()) + 8.0 * m * case["heads"] * case["hd"]
        flops += 4.0 * case["heads"] * case["hd"] * float(see.sum())
    return dict(bytes=nbytes, flops=flops)


def _held64(x):
    """What a row stands for once it is stored: the definition, each rounding to fp32 made from 64 bits."""
    f32 = lambda y: y.to(torch.float32).to(torch.float64)  # noqa: E731
    out = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    seventh = float(np.float32(1) / np.float32(7))
    blocks = [x[..., i:i + BLOCK].double() for i in range(0, x.shape[-1], BLOCK)]
    need = torch.stack([torch.maximum(f32(b.max(-1).values.clamp(min=0) * seventh), b.min(-1).values.clamp(max=0) / -8)
                        for b in blocks], -1)
    top = need.max(-1).values
    s, up = f32(top / 255), f32(255 / top)
    for i, b in enumerate(blocks):
        c = torch.ceil(f32(need[..., i] * up)).clamp(max=255)
        q = torch.round(f32(b * f32(1 / f32(c * s))[..., None]))
        out[..., i * BLOCK:(i + 1) * BLOCK] = q * (c * s)[..., None]
    return out


def _exact_tables(case, seed):
    """The lists walked one sequence after another, on the host."""
    lists, _ = _lists(case, seed)
    tables, at = lists["tables"].copy(), int(lists["used"][0])
    starts, slots, positions = [0], [], []
    for s, (p, m) in enumerate(zip(lists["npast"].tolist(), lists["M"].tolist())):
        for pos in range(p, p + m):
            if tables[s, pos // PAGE] < 0:
                tables[s, pos // PAGE] = lists["free"][at]
                at += 1
            slots.append(int(tables[s, pos // PAGE]) * PAGE + pos % PAGE)
            positions.append(pos)
        starts.append(starts[-1] + m)
    t = lambda x: torch.from_numpy(np.asarray(x, np.int32))  # noqa: E731
    return dict(tables=t(tables), starts=t(starts), slots=t(slots), positions=t(positions), after=t([at]),
                status=t([0]))


def exact(case, seed):
    if case["kind"] == "tables":
        return _exact_tables(case, seed)
    past, new = _sizes(case)
    kc, vc, kn, vn, q = _inputs(case, seed)
    kc, vc, kn, vn = (_held64(x) for x in (kc, vc, kn, vn))
    if case["kind"] == "store":
        return kn, vn
    pe, ne = np.cumsum([0] + past), np.cumsum([0] + new)
    ks = [torch.cat([kc[pe[s]:pe[s + 1]], kn[ne[s]:ne[s + 1]]]) for s in range(case["seqs"])]
    vs = [torch.cat([vc[pe[s]:pe[s + 1]], vn[ne[s]:ne[s + 1]]]) for s in range(case["seqs"])]
    if case["kind"] == "read":
        return torch.cat(ks), torch.cat(vs)
    par = _parents(case["M"], case["tree"]) if case.get("tree") else None
    out = torch.empty(sum(new), case["heads"], case["hd"], dtype=torch.float64, device=DEV)
    g = case["heads"] // case["kv"]
    for s in range(case["seqs"]):
        see = torch.from_numpy(_seen(past[s], new[s], par, case["window"], case["sinks"])).to(DEV)
        for h in range(case["heads"]):
            z = q[ne[s]:ne[s + 1], h].double() @ ks[s][:, h // g].T.contiguous() / math.sqrt(case["hd"])
            z = torch.softmax(torch.where(see, z, torch.full_like(z, -math.inf)), dim=-1)
            out[ne[s]:ne[s + 1], h] = z @ vs[s][:, h // g].contiguous()
    return dict(_exact_tables(case, seed), out=out) if case["kind"] == "step" else out
