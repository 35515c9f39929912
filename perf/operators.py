"""The paged KV cache's operators as cases to time and compare.

A serving loop keeps the K / V rows of many sequences in one pool of pages of
64 tokens, as halves or as 8-bit integers with one scale per token and head.
Three kinds of work come of it, for every layer of every step:

  store   the new tokens' rows are quantised as they are written, and read back
  read    whole contexts are read back (to hand a cache on, or to check it)
  attend  the new tokens attend to their sequences' pages: one token of many
          sequences, drafts (chains and trees), chunks of prompts; with a
          sliding window and a few first tokens that stay visible, or without

Head layouts are those of bench.py's models (8 heads of 64; 32 heads of 64 or
128 over 8; 64 of 128 over 8).

listed() / draw(rng): the cases; prepare(case, seed): a program's state;
run(state): one pass; exact(case, seed): the same outputs in 64 bits.
"""
import math

import numpy as np
import torch

own = False
DEV = "cuda"
PAGE = 64
TINY = dict(heads=8, kv=8, hd=64)
LLAMA_1B = dict(heads=32, kv=8, hd=64)
LLAMA_8B = dict(heads=32, kv=8, hd=128)
LLAMA_70B = dict(heads=64, kv=8, hd=128)


def listed():
    return [
        # the smallest calls: one sequence's next token, its row into the cache
        dict(name="store-1-q8", kind="store", type="q8", seqs=1, M=1, ctx=2047, ragged=0.0, **LLAMA_8B),
        # a step of 16 sequences with 8-token drafts, anywhere in their pages
        dict(name="store-16x8-f16", kind="store", type="f16", seqs=16, M=8, ctx=4096, ragged=0.9, **LLAMA_8B),
        # a prompt's chunk, its first page partly filled by the chunk before
        dict(name="store-2000-q8", kind="store", type="q8", seqs=1, M=2000, ctx=37, ragged=0.0, **LLAMA_8B),
        # four whole contexts handed on
        dict(name="read-4x16k-q8", kind="read", type="q8", seqs=4, M=0, ctx=16384, ragged=0.3, **LLAMA_8B),
        # one token of the tiny model after its 128-token prompt: latency
        dict(name="attend-1-tiny-f16", kind="attend", type="f16", seqs=1, M=1, ctx=128, ragged=0.0,
             tree=0, window=0, sinks=0, **TINY),
        # a decode step of 16 sequences of uneven length
        dict(name="attend-16x1-q8", kind="attend", type="q8", seqs=16, M=1, ctx=8191, ragged=0.9,
             tree=0, window=0, sinks=0, **LLAMA_8B),
        # one long document, one token
        dict(name="attend-1x128k-f16", kind="attend", type="f16", seqs=1, M=1, ctx=131071, ragged=0.0,
             tree=0, window=0, sinks=0, **LLAMA_70B),
        # four 64-node draft trees at context 8192
        dict(name="attend-tree4x64-q8", kind="attend", type="q8", seqs=4, M=64, ctx=8192, ragged=0.0,
             tree=4, window=0, sinks=0, **LLAMA_70B),
        # chunks of three prompts of uneven length in one step
        dict(name="attend-3x1500-q8", kind="attend", type="q8", seqs=3, M=1500, ctx=4000, ragged=0.6,
             tree=0, window=0, sinks=0, **LLAMA_8B),
        # a decode step under a window, far past it
        dict(name="window-16x1-q8", kind="attend", type="q8", seqs=16, M=1, ctx=16000, ragged=0.5,
             tree=0, window=4096, sinks=4, **LLAMA_8B),
        # 8-token drafts under a short window
        dict(name="window-8x8-f16", kind="attend", type="f16", seqs=8, M=8, ctx=5000, ragged=0.9,
             tree=0, window=1000, sinks=4, **LLAMA_1B),
        # a prompt's chunk under a window
        dict(name="window-2048-f16", kind="attend", type="f16", seqs=1, M=2048, ctx=6000, ragged=0.0,
             tree=0, window=1024, sinks=4, **LLAMA_8B),
    ]


def _log_int(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    kind = rng.choice(["store", "read", "attend", "attend", "attend", "window", "window"])
    c = dict(kind="attend" if kind == "window" else kind, type=rng.choice(["f16", "q8"]))
    ragged = round(rng.choice([0.0, rng.random()]), 2)
    if kind in ("store", "read"):
        seqs = _log_int(rng, 1, 32)
        c.update(seqs=seqs, M=0 if kind == "read" else max(1, _log_int(rng, 1, 2000) // seqs),
                 ctx=_log_int(rng, 1, 65536) // seqs + 1, ragged=ragged)
        return dict(c, **rng.choice([TINY, LLAMA_1B, LLAMA_8B]))
    shape = rng.choice([TINY, LLAMA_1B, LLAMA_8B, LLAMA_8B, LLAMA_70B])
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
    window = _log_int(rng, 1, 4096) if kind == "window" else 0
    sinks = rng.choice([0, 1, 4, 65]) if kind == "window" else 0
    return dict(c, seqs=seqs, M=M, ctx=ctx, ragged=ragged, tree=tree, window=window, sinks=sinks, **shape)


# ---------------------------------------------------------------- a case's sizes


def _spread(n, longest, ragged, start):
    """n lengths up to `longest`, spread over its last part `ragged` (the first is the longest)."""
    return [max(1, int(longest * (1.0 - ragged * ((start + s) * 0.6180339887 % 1.0)))) if longest else 0
            for s in range(n)]


def _sizes(case):
    """(committed, new) tokens of every sequence."""
    n = case["seqs"]
    past = _spread(n, case["ctx"], case["ragged"], 0)
    new = _spread(n, case["M"], 0.0 if case.get("tree") else case["ragged"], 0)
    return past, new


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


def prepare(case, seed):
    past, new = _sizes(case)
    S, kv, hd = case["seqs"], case["kv"], case["hd"]
    kc, vc, kn, vn, q = _inputs(case, seed)
    need = [(p + m + PAGE - 1) // PAGE for p, m in zip(past, new)]
    order = np.random.RandomState(seed % (1 << 31)).permutation(sum(need))
    ends = np.cumsum([0] + need)
    tables = [order[ends[s]:ends[s + 1]] for s in range(S)]
    par = _parents(case["M"], case["tree"]) if case.get("tree") else None
    window, sinks = case.get("window", 0), case.get("sinks", 0)
    attend = case["kind"] == "attend"
    st = dict(case=case, kn=kn, vn=vn, q=q)
    if own:
        from xwfes_amd import ftx

        ctx = _ctx()
        pool = ctx.pool(1, kv, hd, sum(need), {"f16": ftx.KV_F16, "q8": ftx.KV_Q8}[case["type"]])
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
    # the plain cache: pages of values and their scales
    vt = torch.float16 if case["type"] == "f16" else torch.int8
    shape = (sum(need), PAGE, kv)
    st.update(type=case["type"])
    for n in ("K", "V"):
        st[n] = torch.zeros(*shape, hd, dtype=vt, device=DEV)
        st[n + "s"] = torch.ones(shape, device=DEV)

    def places(first, count):
        got = [_slots(tables[s], first[s], count[s]) for s in range(S)]
        return tuple(torch.from_numpy(np.concatenate([g[i] for g in got])).to(DEV) for i in (0, 1))

    zero = [0] * S
    st["new"] = places(past, new)
    st["all"] = places(zero, [p + m for p, m in zip(past, new)])
    if case["kind"] != "store":
        _plain_store(st, places(zero, past), kc, vc)
    if attend:
        _plain_store(st, st["new"], kn, vn)
        st.update(_plain_plan(case, past, new, tables, par, window, sinks))
    return st


def _plain_plan(case, past, new, tables, par, window, sinks):
    """Padded index tensors of a batch: every sequence's pages that any of its new tokens
    sees, the slots' and tokens' positions, the rows of the packed queries."""
    S, Mm = case["seqs"], max(new)
    lo = [max(0, p - window + 1) // PAGE if window else 0 for p in past]
    vis = [sorted(set(range(0, min((sinks + PAGE - 1) // PAGE, len(t)))) | set(range(l, len(t))))
           for l, t in zip(lo, tables)]
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


def _quantise(x, kind):
    """Rows of hd values as (stored values, scales)."""
    a = x.abs().amax(-1, keepdim=True)
    if kind == "q8":
        # the rounding's border in 64 bits
        q = torch.round(x.double() * 127.0 / a.double().clamp_min(2.0 ** -100)).to(torch.int8)
        return q, (a / 127.0)[..., 0]
    e = torch.where((a >= 2.0 ** -8) & (a <= 65504.0) | (a == 0), torch.zeros_like(a),
                    torch.floor(torch.log2(a.double().clamp_min(2.0 ** -100))).float() - 14.0)
    return torch.ldexp(x, -e).to(torch.float16), torch.ldexp(torch.ones_like(a), e)[..., 0]


def _plain_store(st, places, k, v):
    for n, x in (("K", k), ("V", v)):
        st[n][places], st[n + "s"][places] = _quantise(x, st["type"])


def _plain_read(st, places):
    return [st[n][places].float() * st[n + "s"][places][..., None] for n in ("K", "V")]


def _plain_attend(st):
    c = st["case"]
    S, Mm = st["qi"].shape
    kv, hd, g = c["kv"], c["hd"], c["heads"] // c["kv"]
    k, v = [(st[n][st["page"]].float() * st[n + "s"][st["page"]][..., None]).reshape(S, -1, kv, hd).transpose(1, 2)
            for n in ("K", "V")]
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


def run(st):
    kind = st["case"]["kind"]
    if own:
        plan = st["plan"]
        if kind == "attend":
            plan.attend(0, st["q"].data_ptr(), st["out"].data_ptr())
            return st["out"]
        if kind == "store":
            plan.write(0, st["kn"].data_ptr(), st["vn"].data_ptr())
        plan.read(0, st["k"].data_ptr(), st["v"].data_ptr(), context=kind == "read")
        return st["k"], st["v"]
    if kind == "attend":
        return _plain_attend(st)
    if kind == "store":
        _plain_store(st, st["new"], st["kn"], st["vn"])
        return tuple(_plain_read(st, st["new"]))
    return tuple(_plain_read(st, st["all"]))


# ---------------------------------------------------------------- the least work, and 64 bits


def _row_bytes(case):
    return case["kv"] * (case["hd"] * (1 if case["type"] == "q8" else 2) + 4)


def work(case):
    past, new = _sizes(case)
    rb, wide = _row_bytes(case), 4 * case["kv"] * case["hd"]
    if case["kind"] != "attend":
        rows = sum(past) + sum(new) if case["kind"] == "read" else sum(new)
        passes = 2 if case["kind"] == "store" else 1
        return dict(bytes=float(passes * 2 * rows * (rb + wide)), flops=float(passes * 4 * rows * case["kv"] * case["hd"]))
    par = _parents(case["M"], case["tree"]) if case["tree"] else None
    nbytes = flops = 0.0
    for p, m in zip(past, new):
        see = _seen(p, m, par, case["window"], case["sinks"])
        nbytes += 2.0 * rb * int(see.any(0).sum()) + 8.0 * m * case["heads"] * case["hd"]
        flops += 4.0 * case["heads"] * case["hd"] * float(see.sum())
    return dict(bytes=nbytes, flops=flops)


def _held64(x, kind):
    """What a row stands for once it is stored, in 64 bits."""
    x = x.double()
    a = x.abs().max(dim=-1, keepdim=True).values
    if kind == "q8":
        return torch.where(a > 0, torch.round(x * 127.0 / a) * a / 127.0, torch.zeros_like(x))
    # (these inputs' rows lie where halves are kept as they are)
    return x.half().double()


def exact(case, seed):
    past, new = _sizes(case)
    kc, vc, kn, vn, q = _inputs(case, seed)
    kc, vc, kn, vn = (_held64(x, case["type"]) for x in (kc, vc, kn, vn))
    if case["kind"] == "store":
        return kn, vn
    pe, ne = np.cumsum([0] + past), np.cumsum([0] + new)
    ks = [torch.cat([kc[pe[s]:pe[s + 1]], kn[ne[s]:ne[s + 1]]]) for s in range(case["seqs"])]
    vs = [torch.cat([vc[pe[s]:pe[s + 1]], vn[ne[s]:ne[s + 1]]]) for s in range(case["seqs"])]
    if case["kind"] == "read":
        return torch.cat(ks), torch.cat(vs)
    par = _parents(case["M"], case["tree"]) if case["tree"] else None
    out = torch.empty(sum(new), case["heads"], case["hd"], dtype=torch.float64, device=DEV)
    g = case["heads"] // case["kv"]
    for s in range(case["seqs"]):
        see = torch.from_numpy(_seen(past[s], new[s], par, case["window"], case["sinks"])).to(DEV)
        for h in range(case["heads"]):
            z = q[ne[s]:ne[s + 1], h].double() @ ks[s][:, h // g].T.contiguous() / math.sqrt(case["hd"])
            z = torch.softmax(torch.where(see, z, torch.full_like(z, -math.inf)), dim=-1)
            out[ne[s]:ne[s + 1], h] = z @ vs[s][:, h // g].contiguous()
    return out
