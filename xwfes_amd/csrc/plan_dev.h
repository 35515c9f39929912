// plan_dev.h -- a step's tables from its lengths: what a sequence has to do, and
// the entries of the attention's work lists, each from its number alone, so that
// the threads that write them share nothing but running sums (device and host).
#pragma once

#include "paged.h"

// a / b, a >= 0, b > 0.  On the device by a reciprocal, off by at most one below
// 2^22 (8 instructions and not 40 one after the other: the build is their latency)
__host__ __device__ inline int idiv(int a, int b) {
#ifdef __HIP_DEVICE_COMPILE__
    if (a < 1 << 22) {
        int q = (int)((float)a * __builtin_amdgcn_rcpf((float)b));
        const int rem = a - q * b;
        q += rem >= b;
        q -= rem < 0;
        return q;
    }
#endif
    return a / b;
}

// What a sequence of p tokens and m new ones has to do, or an FTX_E_* code
struct SeqLoad {
    int code;
    int have, need, touch;  // pages before and after, pages that new tokens go to
    int many, tiles, n;     // its row tiles (PAGED_TR or PAGED_TR_MANY rows), at most n pages each
};
__host__ __device__ inline SeqLoad seq_load(const PagedRoom& r, int64_t ldt, int p, int m) {
    SeqLoad l{};
    const int64_t most = (int64_t)(ldt < r.n_pages ? ldt : r.n_pages) * FTX_PAGE;
    if (p < 0 || m < 0 || m > r.most || (int64_t)p + m > most) {
        l.code = FTX_E_RANGE;
        return l;
    }
    l.have = (p + FTX_PAGE - 1) / FTX_PAGE;
    l.need = (p + m + FTX_PAGE - 1) / FTX_PAGE;
    l.touch = m ? l.need - p / FTX_PAGE : 0;
    if (r.gqa && m) {
        const int R = m * r.gqa;
        l.many = R >= PAGED_MANY;
        const int tr = l.many ? PAGED_TR_MANY : PAGED_TR;
        l.tiles = (R + tr - 1) / tr;
        l.n = l.need;
        if (r.window) {
            // (a tile's positions, its tokens' and the window before them, end inside pages on both sides)
            const int64_t n = (int64_t)(r.sinks + FTX_PAGE - 1) / FTX_PAGE + ((int64_t)r.window + (tr - 1) / r.gqa + 1) / FTX_PAGE + 2;
            l.n = n < l.n ? (int)n : l.n;
        }
    }
    return l;
}
// Pages below have that have to be pages of the pool: [0, s) and [a, have).
// Under a window those between are not read, nor any of a sequence without new
// tokens (contexts are not read back then)
__host__ __device__ inline void seq_held(const PagedRoom& r, int p, int m, int have, int& s, int& a) {
    s = 0;
    a = 0;
    if (!r.window) return;
    if (m == 0) {
        a = have;
        return;
    }
    a = p - r.window + 1 > 0 ? (p - r.window + 1) / FTX_PAGE : 0;
    s = (int)(((int64_t)r.sinks + FTX_PAGE - 1) / FTX_PAGE);
    s = s < a ? s : a;
    s = s < have ? s : have;
    a = a < have ? a : have;
}

// The most pages of a part of lists of `total` pages in all: a launch then has
// some cut / n_kv workgroups more than it has lists
__host__ __device__ inline int seq_per(int total, int cut, int least) {
    if (cut <= 0) return INT32_MAX;
    const int per = total ? idiv(total - 1, cut) + 1 : 0;
    return per < least ? least : per;
}
// The most pages of a part where `lists` lists of few rows, `total` pages in all,
// share a chip that takes `slots` workgroups a kv head at once, two a CU.  One round
// is filled where that can be: parts of try_per pages, the first (finest) of FEW_TRIES
// that gives at most `slots` parts; else what is left of a round for each page, or
// half a round where that is less (long lists among many short ones).  16 sequences
// over 820 to 8192 slots of 4 bits 25.2 us, by four workgroups a CU, in rounds, 30.1;
// one over 131072 38.6 and 43.9; 64 over up to 2000, whole, 24.4, cut 32.  Lists of more
// rows, by this and by that rule: 16 sequences of 8 tokens, 32 rows a kv head, over 820 to
// 8192 49.4 / 55.0 (64 dims 32.8 / 34.0, under a window of 4096 28.3 / 27.5), one of 8 over
// 2048 11.4 / 11.4, over 16384 19.6 / 25.8, 4 of 16 29.1 / 39.0, 64 of 4 over up to 2000 29.2 /
// 37.4.  Of heads of 256 dims a CU takes one workgroup at a time (453 registers), so that
// this fills two rounds: this rule / slots for one a CU / that rule 16 of one token (16 query
// heads over 8) 64 / 64 / 98, 32 over up to 4000 60 / 72 / 87, 16 of 8 (32 over 8) 104 / 136 /
// 139, but one over 8192 26 / 20 / 26, 4 over 8192 43 / 32 / 64, one of 8 36 / 24 / 40
constexpr int FEW_TRIES = 3;
__host__ __device__ inline int try_per(int total, int slots, int lists, int k) {
    const int left = slots - (int)((int64_t)lists * (k + 1) / (FEW_TRIES + 1));
    return lists < slots ? seq_per(total, left, 4) : INT32_MAX;
}
__host__ __device__ inline int else_per(int total, int slots, int lists) {
    const int left = slots - lists;
    return seq_per(total, left > slots / 2 ? left : slots / 2, 4);
}
__host__ __device__ inline int seq_parts(int n, int per) { return per >= n ? 1 : idiv(n - 1, per) + 1; }
// Entries of a sequence: parts of a list, items, blocks of partials, joins
struct SeqCount {
    int np, items, parts, combs;
};
__host__ __device__ inline SeqCount seq_count(const SeqLoad& l, int per) {
    SeqCount c{};
    if (l.tiles == 0) return c;
    const int b = l.many ? PAGED_TR_MANY / PAGED_TR : 1;
    c.np = seq_parts(l.n, per);
    c.items = l.tiles * c.np;
    c.parts = c.np > 1 ? c.items * b : 0;
    c.combs = c.np > 1 ? l.tiles * b : 0;
    return c;
}

// The pages of the tile at row row0: [0, s) and then n - s from a on
__host__ __device__ inline void tile_pages(const PagedRoom& r, int p, int m, int row0, int tr, int& s, int& a, int& n) {
    const int R = m * r.gqa, t0 = idiv(row0, r.gqa), t1 = idiv((R < row0 + tr ? R : row0 + tr) - 1, r.gqa);
    const int lo = r.window && p + t0 - r.window + 1 > 0 ? p + t0 - r.window + 1 : 0;
    a = lo / FTX_PAGE;
    s = r.window ? (int)(((int64_t)r.sinks + FTX_PAGE - 1) / FTX_PAGE) : 0;
    s = s < a ? s : a;
    n = s + (p + t1) / FTX_PAGE + 1 - a;
}
// No item: what a workgroup reads before it looks at seq is the first row's
__host__ __device__ inline PagedItem seq_none() {
    PagedItem it{};
    it.seq = -1;
    it.q.M = 1;
    it.q.dep0 = -1;
    return it;
}
// Item e of sequence q (number s), its partials from part0 on; seq = -1: none (a
// tile whose list is shorter than the sequence's longest)
__host__ __device__ inline PagedItem seq_item(const PagedRoom& r, const PagedSeq& q, int s, int many, int np, int part0, int e) {
    const int tr = many ? PAGED_TR_MANY : PAGED_TR, tile = idiv(e, np), k = e - tile * np;
    PagedItem it{};
    int n;
    tile_pages(r, q.npast, q.M, tile * tr, tr, it.s, it.a, n);
    const int npt = np < n ? np : n;
    if (k >= npt) return seq_none();
    it.seq = s;
    it.row0 = tile * tr;
    // (the first n % npt parts are a page longer)
    const int len = idiv(n, npt), rem = n - len * npt;
    it.i0 = k * len + (k < rem ? k : rem);
    it.i1 = it.i0 + len + (k < rem);
    it.part = np > 1 ? part0 + e * (tr / PAGED_TR) : -1;
    // (one row tile a wave: the host's choice of 16, 128 or 256 rows follows from an estimate
    // over all lists.  Chunks of 64 tokens over 300, 4000, 8-bit, 32 query heads over 8: 18.5
    // and 48.2 us, by the host's plan 9.6 and 23.3; three of 1500 each over 1600 to 4000 686 and 644)
    it.nt = many;
    it.q = q;
    return it;
}
// Join c of it (M = 0: none)
__host__ __device__ inline PagedComb seq_comb(const PagedRoom& r, const PagedSeq& q, int s, int many, int np, int part0, int c) {
    const int tr = many ? PAGED_TR_MANY : PAGED_TR, b = tr / PAGED_TR, tile = c / b, row0 = c * PAGED_TR;
    PagedComb o{};
    if (row0 >= q.M * r.gqa) return o;
    int ps, pa, n;
    tile_pages(r, q.npast, q.M, tile * tr, tr, ps, pa, n);
    o.seq = s;
    o.row0 = row0;
    o.part0 = part0 + tile * np * b + c % b;
    o.n = np < n ? np : n;
    o.step = b;
    o.tok0 = q.tok0;
    o.M = q.M;
    return o;
}
