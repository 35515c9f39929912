// k_plan.hip -- a step's tables built on the GPU (ftx_plan_build).
#include "plan_dev.h"

namespace {

// The entries of sequence s that have to be pages of the pool, by one wave: into
// the plan's own table; its code
__device__ __forceinline__ int check_seq(const PagedBuild& b, int s, int lane) {
    const int p = b.npast[s], m = b.M[s];
    const SeqLoad l = seq_load(b.r, b.ldt, p, m);
    if (l.code) return l.code;
    int hs, ha;
    seq_held(b.r, p, l.have, hs, ha);
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

constexpr int NT = 1024, NW = NT / 64;

// sums over the workgroup, in all threads
template <typename T>
__device__ __forceinline__ T group_sum(T v, T* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();  // (red may still be read)
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    T t = red[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) t += red[w];
    return t;
}
// the sum over the threads before this one
template <typename T>
__device__ __forceinline__ T group_before(T v, T* red) {
    T x = v;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const T y = __shfl_up(x, o, 64);
        x += lane >= o ? y : T(0);
    }
    __syncthreads();
    if (lane == 63) red[w] = x;
    __syncthreads();
    T t = x - v;
    for (int i = 0; i < w; ++i) t += red[i];
    return t;
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

enum { S_TOK, S_FRESH, S_TOUCH, S_FEW, S_MANY, S_PART, S_COMB, N_SUMS };

// Every workgroup forms all running sums itself (a sequence's lengths are eight
// bytes), then writes its share of the entries.  CHECK: the only workgroup, which
// looks at the tables too, where they are short.
template <bool CHECK>
__global__ void __launch_bounds__(NT) k_plan_build(PagedBuild b) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const PagedRoom& r = b.r;
    __shared__ int64_t red[NW];
    const int tid = threadIdx.x, n1 = b.nseq + 1;
    int64_t* const rows_at = (int64_t*)lds;            // [n1]
    int* const sums = (int*)(lds + 8 * (size_t)n1);    // [N_SUMS][n1]
    int* const codes = CHECK ? sums + N_SUMS * n1 : b.codes;
    const int per = (b.nseq + NT - 1) / NT, s0 = min(tid * per, b.nseq), s1 = min(s0 + per, b.nseq);
    const int base = CHECK ? b.used[0] : b.codes[r.nseq];
    if constexpr (CHECK) {
        for (int s = tid >> 6; s < b.nseq; s += NW) {
            const int c = check_seq(b, s, tid & 63);
            if ((tid & 63) == 0) codes[s] = c;
        }
        __syncthreads();
    }
    int64_t few = 0, many = 0, tok = 0, fresh = 0;
    int code = base < 0 || base > b.n_free ? FTX_E_RANGE : FTX_OK;
    for (int s = s0; s < s1; ++s) {
        const SeqLoad l = seq_load(r, b.ldt, b.npast[s], b.M[s]);
        code = min(code, codes[s]);
        if (l.code) continue;
        (l.many ? many : few) += (int64_t)l.tiles * l.n;
        tok += b.M[s];
        fresh += l.need - l.have;
    }
    few = group_sum(few, red);
    many = group_sum(many, red);
    tok = group_sum(tok, red);
    fresh = group_sum(fresh, red);
    if (tok > r.tokens) code = FTX_E_RANGE;
    if (code == FTX_OK && fresh > b.n_free - base) code = FTX_E_NOMEM;
    // (before the list is read past its end)
    const bool fits = base >= 0 && base <= b.n_free && fresh <= b.n_free - base;
    if (fits)
        for (int64_t i = tid; i < fresh; i += NT) {
            const int id = b.free_pages[base + i];
            if (id < 0 || id >= r.pool_pages) code = min(code, FTX_E_INVALID);
        }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) code = min(code, __shfl_xor(code, o, 64));
    __syncthreads();
    if ((tid & 63) == 0) red[tid >> 6] = code;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) code = min(code, (int)red[w]);
    const bool ok = code == FTX_OK;
    const int per_few = r.wide ? INT32_MAX : seq_per(few, r.cut_few, 4), per_many = seq_per(many, r.cut_many, 2);
    int mine[N_SUMS] = {};
    int64_t rows = 0;
    auto add = [&](int s, auto&& each) {
        const int m = b.M[s], p = b.npast[s];
        const SeqLoad l = seq_load(r, b.ldt, p, m);
        const SeqCount c = seq_count(l, l.many ? per_many : per_few);
        const int v[N_SUMS] = {m, l.need - l.have, l.touch, l.many ? 0 : c.items, l.many ? c.items : 0, c.parts, c.combs};
        each(v, (int64_t)p + m);
    };
    if (ok)
        for (int s = s0; s < s1; ++s)
            add(s, [&](const int (&v)[N_SUMS], int64_t n) {
#pragma unroll
                for (int x = 0; x < N_SUMS; ++x) mine[x] += v[x];
                rows += n;
            });
    int at[N_SUMS];
#pragma unroll
    for (int x = 0; x < N_SUMS; ++x) at[x] = (int)group_before<int64_t>(mine[x], red);
    rows = group_before(rows, red);
    for (int s = s0; s < s1; ++s) {
#pragma unroll
        for (int x = 0; x < N_SUMS; ++x) sums[x * n1 + s] = at[x];
        rows_at[s] = rows;
        if (ok)
            add(s, [&](const int (&v)[N_SUMS], int64_t n) {
#pragma unroll
                for (int x = 0; x < N_SUMS; ++x) at[x] += v[x];
                rows += n;
            });
        if (s + 1 == b.nseq) {
#pragma unroll
            for (int x = 0; x < N_SUMS; ++x) sums[x * n1 + b.nseq] = at[x];
            rows_at[b.nseq] = rows;
        }
    }
    __syncthreads();
    auto sum_at = [&](int x) { return sums + x * n1; };
    auto total = [&](int x) { return sums[x * n1 + b.nseq]; };
    auto record = [&](int s) {
        PagedSeq q{};
        q.npast = ok ? b.npast[s] : 0;
        q.M = ok ? b.M[s] : 0;
        q.tok0 = sum_at(S_TOK)[s];
        q.tab0 = s * r.n_pages;
        q.ntab = (q.npast + q.M + FTX_PAGE - 1) / FTX_PAGE;
        q.dep0 = -1;
        q.all0 = rows_at[s];
        return q;
    };
    const int g0 = blockIdx.x * NT + tid, gs = gridDim.x * NT;
    if (g0 == 0) {
        b.used_after[0] = base + total(S_FRESH);
        b.status[0] = code;
    }
    for (int s = g0; s < r.nseq; s += gs) {
        PagedSeq q{};
        q.dep0 = -1;
        if (s < b.nseq) q = record(s);
        b.seqs[s] = q;
    }
    if (b.starts)
        for (int s = g0; s < n1; s += gs) b.starts[s] = sum_at(S_TOK)[s];
    for (int i = g0; i < total(S_FRESH); i += gs) {
        const int s = owner(sum_at(S_FRESH), b.nseq, i), id = b.free_pages[base + i];
        const int64_t col = (b.npast[s] + FTX_PAGE - 1) / FTX_PAGE + i - sum_at(S_FRESH)[s];
        b.tables[s * b.ldt + col] = id;
        b.table[(int64_t)s * r.n_pages + col] = id;
    }
    if (b.slots || b.positions)
        for (int i = g0; i < r.tokens; i += gs) {
            int slot = -1, pos = -1;
            if (i < total(S_TOK)) {
                const int s = owner(sum_at(S_TOK), b.nseq, i), p = b.npast[s], have = (p + FTX_PAGE - 1) / FTX_PAGE;
                pos = p + i - sum_at(S_TOK)[s];
                const int pg = pos / FTX_PAGE;
                const int id = pg < have ? b.tables[s * b.ldt + pg] : b.free_pages[base + sum_at(S_FRESH)[s] + pg - have];
                slot = id * FTX_PAGE + pos % FTX_PAGE;
            }
            if (b.slots) b.slots[i] = slot;
            if (b.positions) b.positions[i] = pos;
        }
    for (int i = g0; i < r.touch; i += gs) {
        int2 t{-1, 0};
        if (i < total(S_TOUCH)) {
            t.x = owner(sum_at(S_TOUCH), b.nseq, i);
            t.y = b.npast[t.x] / FTX_PAGE + i - sum_at(S_TOUCH)[t.x];
        }
        b.touch[i] = t;
    }
    for (int i = g0; i < r.few + r.many; i += gs) {
        const int mn = i >= r.few, e = mn ? i - r.few : i, x = mn ? S_MANY : S_FEW;
        if (e >= total(x)) {
            b.items[i].seq = -1;
            continue;
        }
        const int s = owner(sum_at(x), b.nseq, e);
        const PagedSeq q = record(s);
        const SeqCount c = seq_count(seq_load(r, b.ldt, q.npast, q.M), mn ? per_many : per_few);
        b.items[i] = seq_item(r, q, s, mn, c.np, sum_at(S_PART)[s], e - sum_at(x)[s]);
    }
    for (int i = g0; i < r.combs; i += gs) {
        PagedComb o{};
        if (i < total(S_COMB)) {
            const int s = owner(sum_at(S_COMB), b.nseq, i);
            const PagedSeq q = record(s);
            const SeqLoad l = seq_load(r, b.ldt, q.npast, q.M);
            const SeqCount c = seq_count(l, l.many ? per_many : per_few);
            o = seq_comb(r, q, s, l.many, c.np, sum_at(S_PART)[s], i - sum_at(S_COMB)[s]);
        }
        b.combs[i] = o;
    }
}

}  // namespace

hipError_t launch_paged_build(hipStream_t st, const PagedBuild& b) {
    const PagedRoom& r = b.r;
    const int64_t entries = (int64_t)r.tokens + r.nseq + r.touch + r.few + r.many + r.combs;
    const bool one = (int64_t)b.nseq * r.n_pages <= 8192 && entries <= 8192;
    const size_t bytes = (size_t)(b.nseq + 1) * (8 + 4 * N_SUMS + (one ? 4 : 0));
    static std::atomic<uint64_t> set_one{0}, set_many{0};
    const size_t most = (size_t)(PAGED_ROOM_SEQS + 1) * (8 + 4 * N_SUMS);
    hipError_t e = lds_limit(one ? (const void*)k_plan_build<true> : (const void*)k_plan_build<false>, most,
                             one ? set_one : set_many);
    if (e != hipSuccess) return e;
    if (one) {
        hipLaunchKernelGGL(k_plan_build<true>, dim3(1), dim3(NT), bytes, st, b);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(k_plan_check, dim3((unsigned)(b.nseq + 3) / 4), dim3(256), 0, st, b);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    const unsigned wgs = (unsigned)std::min<int64_t>(64, (entries + NT - 1) / NT);
    hipLaunchKernelGGL(k_plan_build<false>, dim3(wgs), dim3(NT), bytes, st, b);
    return hipGetLastError();
}
