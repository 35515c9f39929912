// k_plan.hip -- a step's tables built on the GPU (ftx_plan_build).
#include <type_traits>

#include "plan_dev.h"

namespace {

// The entries of sequence s that have to be pages of the pool, by one wave: into
// the plan's own table; its code
__device__ __forceinline__ int check_seq(const PagedBuild& b, int s, int lane) {
    const int p = b.npast[s], m = b.M[s];
    const SeqLoad l = seq_load(b.r, b.ldt, p, m);
    if (l.code) return l.code;
    int hs, ha;
    seq_held(b.r, p, m, l.have, hs, ha);
    const int32_t* from = b.tables + s * b.ldt;
    int32_t* to = b.table + (int64_t)s * b.r.n_pages;
    bool bad = false;
    for (int i = lane; i < hs + l.have - ha; i += 64) {
        const int at = i < hs ? i : ha + i - hs, id = from[at];
        bad |= id < 0 || id >= b.r.pool_pages;
        to[at] = id;
    }
    return __builtin_amdgcn_ballot_w64(bad) ? FTX_E_INVALID : FTX_OK;
}

__global__ void __launch_bounds__(256) k_plan_check(PagedBuild b) {
    const int s = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (blockIdx.x == 0 && threadIdx.x == 0) b.codes[b.r.nseq] = b.used[0];
    if (s >= b.nseq) return;
    const int c = check_seq(b, s, lane);
    if (lane == 0) b.codes[s] = c;
}

// Threads of a workgroup: the only one has its entries to write as well (us a call for
// 16 sequences 256: 11.6, 512: 10.8, 1024: 12.4), of several each its share (512
// sequences of 48 new tokens, 128: 18.2, 256: 15.6, 512: 16.3)
template <bool CHECK>
constexpr int build_threads() {
    return CHECK ? 512 : 256;
}
// The most sequences, table entries and other entries of a build by one workgroup, which
// looks at the tables itself.  One / several and the launch before, us in a graph, heads 8 a pool
// if not said: sequences of some 100 pages 16 8.9 / 10.2, 32 9.5 / 10.4, 48 10.1 / 10.0, 64
// 10.3 / 9.6; of 63 64 9.3 / 9.4, 96 11.0 / 10.7, 128 11.8 / 10.7; of 16 192 14.5 / 11.7, 256 16.8 /
// 12.2; of 8 512 27.4 / 14.4; 16 sequences with 5008 table entries 9.6 / 10.0, 7504 10.4 / 10.3; with
// 1206 other entries 9.9 / 11.0, 2097 10.3 / 11.1, 3374 12.2 / 11.1, one with 1709 9.2 / 9.8, 2709
// 10.0 / 9.8 (one kv head, whose lists are cut finest, 16 with 1072 10.8 / 10.7, 64 with 1280 12.5 / 10.8)
constexpr int ONE_SEQS = 64, ONE_TABLE = 6144, ONE_ENTRIES = 2560;

// Between the waves' uses of LDS: what is on its way to global memory is not
// waited for (the stores, which no other wave reads)
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// The sequence that entry i belongs to: at[s] <= i < at[s + 1]
__device__ __forceinline__ int owner(const int* at, int n, int i) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (at[mid] <= i)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// Sums of non-negative numbers over the lanes up to this one, in registers, by
// DPP; SAT: they stop at 2^31 - 1
__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b) { return min(a + b, 0x7FFFFFFFu); }
template <bool SAT>
__device__ __forceinline__ int wave_upto(int v) {
    uint32_t x = (uint32_t)v;
    auto step = [&](auto ctrl, auto rows) {
        const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, decltype(rows)::value, 0xF, false);
        x = SAT ? sat_add(x, y) : x + y;
    };
    using std::integral_constant;
    constexpr integral_constant<int, 0xF> all{};
    step(integral_constant<int, 0x111>{}, all);  // from 1, 2, 4, 8 lanes before, in rows of 16
    step(integral_constant<int, 0x112>{}, all);
    step(integral_constant<int, 0x114>{}, all);
    step(integral_constant<int, 0x118>{}, all);
    step(integral_constant<int, 0x142>{}, integral_constant<int, 0xA>{});  // rows 1 and 3: the last lane of the row before
    step(integral_constant<int, 0x143>{}, integral_constant<int, 0xC>{});  // rows 2 and 3: lane 31
    return (int)x;
}
__device__ __forceinline__ int wave_total(int v) { return __builtin_amdgcn_readlane(wave_upto<true>(v), 63); }

enum { S_TOK, S_FRESH, S_TOUCH, S_FEW, S_MANY, S_PART, S_COMB, N_SUMS };

// Every workgroup forms all running sums itself (a sequence's lengths are eight
// bytes), then writes its share of the entries.  CHECK: the only workgroup, which
// looks at the tables too, where they are short: a launch less.  Bound by latency,
// lengths, tables, list and entries one after the other: two exchanges between
// the waves, the first of totals (how lists are cut follows from them), the second
// of running sums and what the list of pages holds.  16 sequences: 11.8 us of kernel
// for 370 bytes (10.7 a build in a graph), 730 vector instructions a wave; sums by one
// wave, with 40 instructions a division, 23.8.  512 sequences of 48 tokens: 4.0 and 13.3 us.
template <bool CHECK>
__global__ void __launch_bounds__(build_threads<CHECK>()) k_plan_build(PagedBuild b) {
    constexpr int NT = build_threads<CHECK>(), NW = NT / 64;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const PagedRoom& r = b.r;
    enum { T_FEW, T_MANY, T_LISTS, T_TOK, T_FRESH, T_CODE, N_TOT };  // (page lists' totals stay below 2^31: paged_room)
    __shared__ int parts_of[NW][FEW_TRIES];
    __shared__ int tot[NW][N_TOT], sum_of[NW][N_SUMS], rows_of[NW][2], bad_of[NW];
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, n = b.nseq, n1 = n + 1;
    int* const P = (int*)lds;  // [n] lengths
    int* const M = P + n;      // (in the end the parts of a list)
    int* const sums = M + n;   // [N_SUMS][n1] (CHECK: first have, s and a of seq_held)
    const int per = (n + NT - 1) / NT, s0 = min(tid * per, n), s1 = min(s0 + per, n);
    // waves that have sequences form their sums, the others wait: all would share the
    // SIMDs
    const bool busy = __builtin_amdgcn_readfirstlane(w) * 64 * per < n;
    // The first loads, none of which waits for another: the lengths, the first
    // table entries whether they are pages or not, and (next) the list from `used` on
    // (a wave takes a sequence's entries 64 at a time, every NW-th sequence, so that
    // all but the entry itself is the wave's)
    constexpr int U = CHECK ? 12 : 1;  // loads of a wave in flight
    const int chunks = (r.n_pages + 63) / 64, wv = __builtin_amdgcn_readfirstlane(w);
    const int loads = wv < n ? ((n - 1 - wv) / NW + 1) * chunks : 0;
    int id[U];
    // (a place past the row's end reads its last entry)
    const int row = (int)min((int64_t)r.n_pages, b.ldt);
    struct Walk {
        int s, c;  // sequence, chunk
    };
    auto next = [&](Walk& x) {
        if (++x.c == chunks) {
            x.c = 0;
            x.s += NW;
        }
    };
    Walk lw{wv, 0};
    const int32_t* from_row = b.tables + wv * b.ldt;
    auto load = [&](int e0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (e0 + u >= loads) break;
            id[u] = from_row[min(64 * lw.c + lane, row - 1)];
            next(lw);
            if (lw.c == 0) from_row += NW * b.ldt;
        }
    };
    if constexpr (CHECK) load(0);
    const int base = CHECK ? b.used[0] : b.codes[r.nseq];
    int code = FTX_OK;
    for (int s = s0; s < s1; ++s) {
        P[s] = b.npast[s];
        M[s] = b.M[s];
        if constexpr (CHECK) {
            const SeqLoad l = seq_load(r, b.ldt, P[s], M[s]);
            int hs = 0, ha = 0;
            if (!l.code) seq_held(r, P[s], M[s], l.have, hs, ha);
            sums[s] = l.have;  // (0 with a code: nothing to look at)
            sums[n1 + s] = hs;
            sums[2 * n1 + s] = ha;
        } else {
            code = min(code, b.codes[s]);
        }
    }
    const int mine_at = base >= 0 && base <= b.n_free && tid < b.n_free - base ? b.free_pages[base + tid] : 0;
    if constexpr (CHECK) {
        lds_barrier();
        Walk x{wv, 0};
        int have = 0, hs = 0, ha = 0;
        int32_t* to_row = b.table + (int64_t)wv * r.n_pages;
        for (int e0 = 0; e0 < loads;) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (e0 + u >= loads) break;
                if (x.c == 0) {
                    have = __builtin_amdgcn_readfirstlane(sums[x.s]);
                    hs = __builtin_amdgcn_readfirstlane(sums[n1 + x.s]);
                    ha = __builtin_amdgcn_readfirstlane(sums[2 * n1 + x.s]);
                }
                const int i = 64 * x.c + lane;
                if (i < have && (i < hs || i >= ha)) {
                    if ((uint32_t)id[u] >= (uint32_t)r.pool_pages) code = FTX_E_INVALID;
                    to_row[i] = id[u];
                }
                next(x);
                if (x.c == 0) to_row += (int64_t)NW * r.n_pages;
            }
            e0 += U;
            if (e0 < loads) load(e0);
        }
    }
    if (base < 0 || base > b.n_free) code = FTX_E_RANGE;
    uint32_t t[N_TOT] = {};
    for (int s = s0; s < s1; ++s) {
        const SeqLoad l = seq_load(r, b.ldt, P[s], M[s]);
        code = min(code, l.code);
        if (l.code) continue;
        const uint32_t pages = (uint32_t)(l.tiles * l.n);
        t[T_FEW] = sat_add(t[T_FEW], l.many ? 0 : pages);
        t[T_MANY] = sat_add(t[T_MANY], l.many ? pages : 0);
        t[T_LISTS] = sat_add(t[T_LISTS], l.many ? 0 : (uint32_t)l.tiles);
        t[T_TOK] = sat_add(t[T_TOK], (uint32_t)M[s]);
        t[T_FRESH] = sat_add(t[T_FRESH], (uint32_t)(l.need - l.have));
    }
#pragma unroll
    for (int x = 0; x < T_CODE; ++x) {
        const int v = busy ? wave_total((int)t[x]) : 0;
        if (lane == 0) tot[w][x] = v;
    }
    // (the lowest code: of 0, -1, -4, -5)
    const auto seen = [&](int c) { return __builtin_amdgcn_ballot_w64(code == c) != 0; };
    code = seen(FTX_E_RANGE) ? FTX_E_RANGE : seen(FTX_E_NOMEM) ? FTX_E_NOMEM : seen(FTX_E_INVALID) ? FTX_E_INVALID : FTX_OK;
    if (lane == 0) tot[w][T_CODE] = code;
    lds_barrier();
#pragma unroll
    for (int x = 0; x < T_CODE; ++x) t[x] = (uint32_t)tot[0][x];
#pragma unroll
    for (int i = 1; i < NW; ++i)
#pragma unroll
        for (int x = 0; x < T_CODE; ++x) t[x] = sat_add(t[x], (uint32_t)tot[i][x]);
#pragma unroll
    for (int i = 0; i < NW; ++i) code = min(code, tot[i][T_CODE]);
    if (t[T_TOK] > (uint32_t)r.tokens) code = FTX_E_RANGE;
    bool bad = false;
    if (base >= 0 && base <= b.n_free) {
        const int fresh = (int)t[T_FRESH];
        if (fresh > b.n_free - base)
            code = min(code, FTX_E_NOMEM);
        else
            for (int i = tid; i < fresh; i += NT) {
                const int pg = i < NT ? mine_at : b.free_pages[base + i];
                bad |= pg < 0 || pg >= r.pool_pages;
            }
    }
    int per_few = INT32_MAX;
    if (r.cut_few) {
        // (parts of each try, of all lists)
        uint32_t parts[FEW_TRIES] = {};
        int tries[FEW_TRIES];
#pragma unroll
        for (int k = 0; k < FEW_TRIES; ++k) tries[k] = try_per((int)t[T_FEW], r.slots, (int)t[T_LISTS], k);
        for (int s = s0; s < s1; ++s) {
            const SeqLoad l = seq_load(r, b.ldt, P[s], M[s]);
            if (l.many) continue;
#pragma unroll
            for (int k = 0; k < FEW_TRIES; ++k) parts[k] = sat_add(parts[k], (uint32_t)(l.tiles * seq_parts(l.n, tries[k])));
        }
#pragma unroll
        for (int k = 0; k < FEW_TRIES; ++k) {
            const int v = busy ? wave_total((int)parts[k]) : 0;
            if (lane == 0) parts_of[w][k] = v;
        }
        lds_barrier();
        per_few = else_per((int)t[T_FEW], r.slots, (int)t[T_LISTS]);
#pragma unroll
        for (int k = FEW_TRIES - 1; k >= 0; --k) {
            uint32_t v = (uint32_t)parts_of[0][k];
#pragma unroll
            for (int i = 1; i < NW; ++i) v = sat_add(v, (uint32_t)parts_of[i][k]);
            if (v <= (uint32_t)r.slots && (int)t[T_LISTS] < r.slots) per_few = tries[k];
        }
    }
    const int per_many = seq_per((int)t[T_MANY], r.cut_many, 2);
    int mine[N_SUMS] = {};
    int64_t rows = 0;
    auto add = [&](int s, int (&to)[N_SUMS], int64_t& to_rows) -> int {
        const SeqLoad l = seq_load(r, b.ldt, P[s], M[s]);
        const SeqCount c = seq_count(l, l.many ? per_many : per_few);
        const int v[N_SUMS] = {M[s], l.need - l.have, l.touch, l.many ? 0 : c.items, l.many ? c.items : 0, c.parts, c.combs};
#pragma unroll
        for (int x = 0; x < N_SUMS; ++x) to[x] += v[x];
        to_rows += (int64_t)P[s] + M[s];
        return c.np;
    };
    int np = 0;
    if (code == FTX_OK)
        for (int s = s0; s < s1; ++s) np = add(s, mine, rows);
    const int64_t own_rows = rows;
    int at[N_SUMS] = {}, low = 0, high = 0;
    if (busy) {
#pragma unroll
        for (int x = 0; x < N_SUMS; ++x) at[x] = wave_upto<false>(mine[x]);
        // (up to 2^30 positions a sequence: in two parts)
        low = wave_upto<false>((int)(rows & 0xFFFF));
        high = wave_upto<false>((int)(rows >> 16));
    }
    const bool any = __builtin_amdgcn_ballot_w64(bad);
    if (lane == 63) {
#pragma unroll
        for (int x = 0; x < N_SUMS; ++x) sum_of[w][x] = at[x];
        rows_of[w][0] = low;
        rows_of[w][1] = high;
        bad_of[w] = any;
    }
    lds_barrier();
    rows = low + ((int64_t)high << 16) - rows;
#pragma unroll
    for (int x = 0; x < N_SUMS; ++x) at[x] -= mine[x];
#pragma unroll
    for (int i = 0; i < NW; ++i)
        if (bad_of[i]) code = min(code, FTX_E_INVALID);
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        if (i >= w) continue;
        rows += rows_of[i][0] + ((int64_t)rows_of[i][1] << 16);
#pragma unroll
        for (int x = 0; x < N_SUMS; ++x) at[x] += sum_of[i][x];
    }
    const bool ok = code == FTX_OK;
    auto record = [&](int s, int m, int tok0, int64_t all0) {
        PagedSeq q{};
        q.npast = ok ? P[s] : 0;
        q.M = ok ? m : 0;
        q.tok0 = tok0;
        q.tab0 = s * r.n_pages;
        q.ntab = (q.npast + q.M + FTX_PAGE - 1) / FTX_PAGE;
        q.dep0 = -1;
        q.all0 = all0;
        return q;
    };
    for (int s = s0; s < s1; ++s) {
#pragma unroll
        for (int x = 0; x < N_SUMS; ++x) sums[x * n1 + s] = ok ? at[x] : 0;
        if (blockIdx.x == 0) b.seqs[s] = record(s, M[s], ok ? at[S_TOK] : 0, ok ? rows : 0);
        if (per == 1) {
#pragma unroll
            for (int x = 0; x < N_SUMS; ++x) at[x] += mine[x];
            rows += own_rows;
            M[s] = np;
        } else if (ok) {
            M[s] = add(s, at, rows);
        }
        if (s + 1 == n)
#pragma unroll
            for (int x = 0; x < N_SUMS; ++x) sums[x * n1 + n] = ok ? at[x] : 0;
    }
    lds_barrier();
    auto sum_at = [&](int x) { return sums + x * n1; };
    auto total = [&](int x) { return sums[x * n1 + n]; };
    auto of = [&](int s) { return record(s, sum_at(S_TOK)[s + 1] - sum_at(S_TOK)[s], sum_at(S_TOK)[s], 0); };
    // a page that new tokens go to
    auto page_of = [&](int s, int pg) {
        const int have = (P[s] + FTX_PAGE - 1) / FTX_PAGE;
        return pg < have ? b.tables[s * b.ldt + pg] : b.free_pages[base + sum_at(S_FRESH)[s] + pg - have];
    };
    const int g0 = blockIdx.x * NT + tid, gs = gridDim.x * NT;
    // (each kind's entries from another wave on, where they are few: side by side)
    auto from = [&](int wave) {
        const int o = 64 * wave % gs;
        return g0 >= o ? g0 - o : g0 - o + gs;  // in [0, gs)
    };
    if (g0 == 0) {
        b.used_after[0] = base + total(S_FRESH);
        b.status[0] = code;
    }
    for (int s = n + from(1); s < r.nseq; s += gs) {
        PagedSeq q{};
        q.dep0 = -1;
        b.seqs[s] = q;
    }
    if (b.starts)
        for (int s = from(2); s < n1; s += gs) b.starts[s] = sum_at(S_TOK)[s];
    for (int i = from(3); i < total(S_FRESH); i += gs) {
        const int s = owner(sum_at(S_FRESH), n, i), id = b.free_pages[base + i];
        const int64_t col = (P[s] + FTX_PAGE - 1) / FTX_PAGE + i - sum_at(S_FRESH)[s];
        b.tables[s * b.ldt + col] = id;
        b.table[(int64_t)s * r.n_pages + col] = id;
    }
    if (b.slots || b.positions)
        for (int i = from(4); i < r.tokens; i += gs) {
            int slot = -1, pos = -1;
            if (i < total(S_TOK)) {
                const int s = owner(sum_at(S_TOK), n, i);
                pos = P[s] + i - sum_at(S_TOK)[s];
                slot = page_of(s, pos / FTX_PAGE) * FTX_PAGE + pos % FTX_PAGE;
            }
            if (b.slots) b.slots[i] = slot;
            if (b.positions) b.positions[i] = pos;
        }
    for (int i = from(5); i < r.touch; i += gs) {
        PagedTouch to{-1, 0, 0, 0, 0, 0};
        if (i < total(S_TOUCH)) {
            const int s = owner(sum_at(S_TOUCH), n, i), p = P[s], pg = p / FTX_PAGE + i - sum_at(S_TOUCH)[s];
            const int tok0 = sum_at(S_TOK)[s], m = sum_at(S_TOK)[s + 1] - tok0;
            to.page = page_of(s, pg);
            to.s0 = max(p - pg * FTX_PAGE, 0);
            to.s1 = min(p + m - pg * FTX_PAGE, FTX_PAGE);
            to.row = (int64_t)tok0 - p + (int64_t)pg * FTX_PAGE;
        }
        b.touch[i] = to;
    }
    for (int i = from(6); i < r.few + r.many; i += gs) {
        const int mn = i >= r.few, e = mn ? i - r.few : i, x = mn ? S_MANY : S_FEW;
        if (e >= total(x)) {
            b.items[i] = seq_none();
            continue;
        }
        const int s = owner(sum_at(x), n, e);
        b.items[i] = seq_item(r, of(s), s, mn, M[s], sum_at(S_PART)[s], e - sum_at(x)[s]);
    }
    for (int i = from(7); i < r.combs; i += gs) {
        PagedComb o{};
        if (i < total(S_COMB)) {
            const int s = owner(sum_at(S_COMB), n, i);
            const PagedSeq q = of(s);
            o = seq_comb(r, q, s, q.M * r.gqa >= PAGED_MANY, M[s], sum_at(S_PART)[s], i - sum_at(S_COMB)[s]);
        }
        b.combs[i] = o;
    }
}

}  // namespace

hipError_t paged_build_limits() {
    // (k_plan_build<true>, of ONE_SEQS sequences, needs no limit set)
    static std::atomic<uint64_t> set{0};
    return lds_limit((const void*)k_plan_build<false>, (size_t)(PAGED_ROOM_SEQS + 1) * (8 + 4 * N_SUMS), set);
}

hipError_t launch_paged_build(hipStream_t st, const PagedBuild& b) {
    const PagedRoom& r = b.r;
    const int64_t entries = (int64_t)r.tokens + r.nseq + r.touch + r.few + r.many + r.combs;
    const bool one = b.nseq <= ONE_SEQS && (int64_t)b.nseq * r.n_pages <= ONE_TABLE && entries <= ONE_ENTRIES;
    const size_t bytes = (size_t)(b.nseq + 1) * (8 + 4 * N_SUMS);
    if (one) {
        hipLaunchKernelGGL(k_plan_build<true>, dim3(1), dim3(build_threads<true>()), bytes, st, b);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(k_plan_check, dim3((unsigned)(b.nseq + 3) / 4), dim3(256), 0, st, b);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    constexpr int NT = build_threads<false>();
    const unsigned wgs = (unsigned)std::min<int64_t>(128, (entries + NT - 1) / NT);
    hipLaunchKernelGGL(k_plan_build<false>, dim3(wgs), dim3(NT), bytes, st, b);
    return hipGetLastError();
}
