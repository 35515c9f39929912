// k_paged.hip -- kernels of the paged KV caches: rows quantised into their
// pages and read back, and the attention of new tokens over pages.
#include "mm_dev.h"
#include "paged.h"

namespace {

constexpr float FLT_BIG = 3.402823466e38f;
// rows below this are stored as zeros
constexpr float ROW_TINY = 7.888609052210118e-31f;  // 2^-100

__device__ __forceinline__ uint8_t* page_block(const PagedView& p, int page, int kvh) {
    return p.data + ((int64_t)page * p.n_kv + kvh) * p.block;
}

// four consecutive floats; vec: 16-byte aligned
__device__ __forceinline__ v4f ld4(const float* p, bool vec) {
    if (vec) return *(const v4f*)p;
    return v4f{p[0], p[1], p[2], p[3]};
}
__device__ __forceinline__ void st4(float* p, v4f v, bool vec) {
    if (vec) {
        *(v4f*)p = v;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = v[i];
}

// 127 x / a rounded to the nearest integer, ties to even.  The fp32 quotient
// is off by less than 2e-5; where that could matter the quotient is formed in
// 64 bits, whose rounding cannot cross a half: |254 x - (2 n + 1) a| is 0 or
// at least 2^-31 of its terms.
__device__ __forceinline__ int q8_round(float x, float a, float inv) {
    const float f = x * inv;
    float n = rintf(f);
    if (fabsf(f - n) > 0.4999f) n = (float)rint((double)x * 127.0 / (double)a);
    return (int)n;
}

// The power of two that a row of halves is stored under
__device__ __forceinline__ int f16_exp(float a) {
    return a >= 0.00390625f && a <= 65504.f ? 0 : (int)((__builtin_bit_cast(uint32_t, a) >> 23) & 255) - 127 - 14;
}

// ---------------------------------------------------------------- write
// Workgroup (page x of sequence y's new tokens, kv head z); a wave per row.
template <int HD, bool Q8>
__global__ void __launch_bounds__(256) k_paged_write(PagedView p, const float* __restrict__ k, int64_t ldk,
                                                     const float* __restrict__ v, int64_t ldv) {
    constexpr int E = HD / 64;  // values a lane
    const PagedSeq sq = p.seqs[blockIdx.y];
    const int first = sq.npast / FTX_PAGE + blockIdx.x;  // the page's place in the table
    const int s0 = max(first * FTX_PAGE, sq.npast), s1 = min(first * FTX_PAGE + FTX_PAGE, sq.npast + sq.M);
    if (s0 >= s1) return;
    const int kvh = blockIdx.z, w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    uint8_t* blk = page_block(p, p.table[sq.tab0 + first], kvh);
    const int64_t vb = paged_values_bytes(HD, Q8);
    float* scale = (float*)(blk + 2 * vb);
    for (int i = w; i < 2 * (s1 - s0); i += 4) {
        const bool isv = i & 1;
        const int pos = s0 + (i >> 1), slot = pos % FTX_PAGE;
        const int64_t row = sq.tok0 + (pos - sq.npast);
        const float* src = (isv ? v + row * ldv : k + row * ldk) + (int64_t)kvh * HD + E * lane;
        float x[E], a = 0.f;
        bool fin = true;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            x[e] = src[e];
            fin = fin && fabsf(x[e]) <= FLT_BIG;
            a = fmaxf(a, fabsf(x[e]));
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor(a, o, 64));
        const bool ok = !__builtin_amdgcn_ballot_w64(!fin), zero = !ok || a < ROW_TINY;
        uint8_t* dst = blk + (isv ? vb : 0);
        float sc;
        if constexpr (Q8) {
            const float inv = 127.f / a;
            sc = zero ? 0.f : a / 127.f;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int q = zero ? 0 : q8_round(x[e], a, inv);
                const int d = E * lane + e;
                dst[isv ? paged_v_at(slot, d, 1) : paged_k_at(slot, d, 1)] = (uint8_t)(q + 128);
            }
        } else {
            const int ex = zero ? 0 : f16_exp(a);
            sc = ldexpf(1.f, ex);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int d = E * lane + e;
                *(_Float16*)(dst + (isv ? paged_v_at(slot, d, 0) : paged_k_at(slot, d, 0))) =
                    zero ? (_Float16)0.f : (_Float16)ldexpf(x[e], -ex);
            }
        }
        if (lane == 0) scale[(isv ? FTX_PAGE : 0) + slot] = ok ? sc : __builtin_nanf("");
    }
}

// ---------------------------------------------------------------- read back
template <int HD, bool Q8>
__global__ void __launch_bounds__(256) k_paged_read(PagedView p, int context, float* __restrict__ k, int64_t ldk,
                                                    float* __restrict__ v, int64_t ldv) {
    constexpr int E = HD / 64;
    const PagedSeq sq = p.seqs[blockIdx.y];
    const int from = context ? 0 : sq.npast;
    const int first = from / FTX_PAGE + blockIdx.x;
    const int s0 = max(first * FTX_PAGE, from), s1 = min(first * FTX_PAGE + FTX_PAGE, sq.npast + sq.M);
    if (s0 >= s1) return;
    const int kvh = blockIdx.z, w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const uint8_t* blk = page_block(p, p.table[sq.tab0 + first], kvh);
    const int64_t vb = paged_values_bytes(HD, Q8);
    const float* scale = (const float*)(blk + 2 * vb);
    for (int i = w; i < 2 * (s1 - s0); i += 4) {
        const bool isv = i & 1;
        const int pos = s0 + (i >> 1), slot = pos % FTX_PAGE;
        const int64_t row = context ? sq.all0 + pos : (int64_t)sq.tok0 + (pos - sq.npast);
        float* dst = (isv ? v + row * ldv : k + row * ldk) + (int64_t)kvh * HD + E * lane;
        const uint8_t* src = blk + (isv ? vb : 0);
        const float sc = scale[(isv ? FTX_PAGE : 0) + slot];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int d = E * lane + e;
            const int at = isv ? paged_v_at(slot, d, Q8) : paged_k_at(slot, d, Q8);
            const float q = Q8 ? (float)((int)src[at] - 128) : (float)*(const _Float16*)(src + at);
            dst[e] = q * sc;
        }
    }
}

// ---------------------------------------------------------------- moves
// Thread = one dim of a kv head of a layer; it walks the path in increasing i
// (dst[i] is never a later source).
__global__ void __launch_bounds__(256) k_paged_move(PagedMove m) {
    const int d = threadIdx.x;
    if (d >= m.hd) return;
    uint8_t* base = m.data + ((int64_t)blockIdx.y * m.n_pages * m.n_kv + blockIdx.x) * m.block;
    const int64_t vb = paged_values_bytes(m.hd, m.q8), step = m.block * m.n_kv;
    for (int i = 0; i < m.n; ++i) {
        const int ss = m.src[i] % FTX_PAGE, ds = m.dst[i] % FTX_PAGE;
        const uint8_t* s = base + (m.src[i] / FTX_PAGE) * step;
        uint8_t* t = base + (m.dst[i] / FTX_PAGE) * step;
        if (m.src[i] == m.dst[i]) continue;
        if (m.q8) {
            t[paged_k_at(ds, d, 1)] = s[paged_k_at(ss, d, 1)];
            t[vb + paged_v_at(ds, d, 1)] = s[vb + paged_v_at(ss, d, 1)];
        } else {
            *(uint16_t*)(t + paged_k_at(ds, d, 0)) = *(const uint16_t*)(s + paged_k_at(ss, d, 0));
            *(uint16_t*)(t + vb + paged_v_at(ds, d, 0)) = *(const uint16_t*)(s + vb + paged_v_at(ss, d, 0));
        }
        if (d < 2) ((float*)(t + 2 * vb))[d * FTX_PAGE + ds] = ((const float*)(s + 2 * vb))[d * FTX_PAGE + ss];
    }
}

// ---------------------------------------------------------------- attention
// 8 biased bytes -> fp16 q (exact): the byte under 0x64 is 1024 + q + 128
__device__ __forceinline__ v8h u8x8(uint32_t a, uint32_t b) {
    const v2h o = {(_Float16)(-1152.f), (_Float16)(-1152.f)};
    const v2h h0 = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(a, 0x64646464u, 0x00050004u)) + o;
    const v2h h1 = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(a, 0x64646464u, 0x00070006u)) + o;
    const v2h h2 = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(b, 0x64646464u, 0x00050004u)) + o;
    const v2h h3 = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(b, 0x64646464u, 0x00070006u)) + o;
    return v8h{h0[0], h0[1], h1[0], h1[1], h2[0], h2[1], h3[0], h3[1]};
}

__device__ __forceinline__ int f_exp(float x) {  // floor(log2 x) of a normal x
    return (int)((__builtin_bit_cast(uint32_t, x) >> 23) & 255) - 127;
}

// The lowest exponent that V scales are taken relative to: 2^(14 - ev) is
// finite.  (The smallest scale is 2^-114.)
constexpr int EV_MIN = -113;

// One wave's online softmax over pages for a tile of 16 query rows.  Lane
// (col, kq) holds the scores of row col at slots 16 st + 4 kq + r and the
// outputs of row col at dims 16 dt + 4 kq + r.
// Scores in units of log2: s2 = ((q 2^eq) . k) (2^-eq log2 e / sqrt(hd)) ks.
// P.V: p vs 2^(14 - ev) is split in two halves, ev the exponent of the largest
// V scale that the row has seen, so the outputs stand 2^(14 - ev) over.
template <int HD, bool Q8>
struct WaveAttn {
    static constexpr int NDC = HD / 32, NDT = HD / 16;
    v8h qh[NDC], ql[NDC];
    v4f o[NDT];
    float m = -INFINITY, l = 0.f;  // (l: this lane's slots only)
    float c2;
    int ev = EV_MIN;

    // the query row at q, this lane's dims
    __device__ __forceinline__ void query(const float* q, int kq, bool vec) {
        v4f x[NDC][2];
        float a = 0.f;
#pragma unroll
        for (int dc = 0; dc < NDC; ++dc) {
            const int d0 = Q8 ? 64 * (dc >> 1) + 16 * kq + 8 * (dc & 1) : 32 * dc + 8 * kq;
            x[dc][0] = ld4(q + d0, vec);
            x[dc][1] = ld4(q + d0 + 4, vec);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float b = fabsf(x[dc][i >> 2][i & 3]);
                a = b <= FLT_BIG ? fmaxf(a, b) : a;
            }
        }
        a = fmaxf(a, __shfl_xor(a, 16, 64));
        a = fmaxf(a, __shfl_xor(a, 32, 64));
        // the largest to [2^6, 2^7): the halves of the smaller ones keep 2^-31 of it
        const int e = a > 0.f ? min(max(6 - f_exp(a), -121), 126) : 0;
        const float qs = ldexpf(1.f, e);
        c2 = ldexpf(1.4426950408889634f / sqrtf((float)HD), -e);
#pragma unroll
        for (int dc = 0; dc < NDC; ++dc)
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                v2h h, lo;
                split_hl2(x[dc][i >> 2][i & 3] * qs, x[dc][i >> 2][(i & 3) + 1] * qs, h, lo);
                qh[dc][i] = h[0];
                qh[dc][i + 1] = h[1];
                ql[dc][i] = lo[0];
                ql[dc][i + 1] = lo[1];
            }
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) o[dt] = v4f{0.f, 0.f, 0.f, 0.f};
    }

    __device__ __forceinline__ v8h k_frag(const uint8_t* blk, int st, int dc, int lane) const {
        if constexpr (Q8) {
            const uint4 u = *(const uint4*)(blk + (((dc >> 1) * 4 + st) * 64 + lane) * 16);
            return dc & 1 ? u8x8(u.z, u.w) : u8x8(u.x, u.y);
        } else {
            return *(const v8h*)(blk + ((dc * 4 + st) * 64 + lane) * 16);
        }
    }
    __device__ __forceinline__ v8h v_frag(const uint8_t* vals, int dt, int sp, int lane) const {
        if constexpr (Q8) {
            const uint4 u = *(const uint4*)(vals + (dt * 64 + lane) * 16);
            return sp ? u8x8(u.z, u.w) : u8x8(u.x, u.y);
        } else {
            return *(const v8h*)(vals + ((dt * 2 + sp) * 64 + lane) * 16);
        }
    }

    // one page; seen(st, r): whether the row sees the slot (whole: it sees all)
    template <typename Seen>
    __device__ __forceinline__ void page(const uint8_t* blk, int lane, bool whole, Seen seen) {
        const int kq = lane >> 4;
        const uint8_t* vals = blk + paged_values_bytes(HD, Q8);
        const float* scale = (const float*)(blk + 2 * paged_values_bytes(HD, Q8));
        v4f s[4], ks[4], vs[4];
#pragma unroll
        for (int st = 0; st < 4; ++st) {
            ks[st] = *(const v4f*)(scale + 16 * st + 4 * kq);
            vs[st] = *(const v4f*)(scale + FTX_PAGE + 16 * st + 4 * kq);
        }
#pragma unroll
        for (int st = 0; st < 4; ++st) {
            s[st] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int dc = 0; dc < NDC; ++dc) {
                const v8h kf = k_frag(blk, st, dc, lane);
                s[st] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[dc], s[st], 0, 0, 0);
                s[st] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qh[dc], s[st], 0, 0, 0);
            }
        }
        float mx = -INFINITY, vm = 0.f;
#pragma unroll
        for (int st = 0; st < 4; ++st)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const bool ok = whole || seen(st, r);
                s[st][r] = ok ? (s[st][r] * c2) * ks[st][r] : -INFINITY;
                vs[st][r] = ok ? vs[st][r] : 0.f;
                mx = fmaxf(mx, s[st][r]);
                vm = fmaxf(vm, vs[st][r]);
            }
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        vm = fmaxf(vm, __shfl_xor(vm, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        vm = fmaxf(vm, __shfl_xor(vm, 32, 64));
        const float mn = fmaxf(m, mx);
        const float mr = mn == -INFINITY ? 0.f : mn;  // (nothing seen yet: every p is 0)
        const float al = __builtin_amdgcn_exp2f(m - mr);
        const int en = max(ev, f_exp(vm));  // (vm = 0: -127)
        const float vscale = ldexpf(1.f, 14 - min(en, 127));
        const float oal = ldexpf(al, ev - en);
        m = mn;
        ev = en;
        l *= al;
        v8h ph[2], pl[2];
#pragma unroll
        for (int st = 0; st < 4; ++st)
#pragma unroll
            for (int r = 0; r < 4; r += 2) {
                const float p0 = __builtin_amdgcn_exp2f(s[st][r] - mr);
                const float p1 = __builtin_amdgcn_exp2f(s[st][r + 1] - mr);
                l += p0 + p1;
                // (split_hl2: a high half formed twice, once from the product
                // unrounded, would not fit its low half)
                v2h h, lo;
                split_hl2(p0 * (vs[st][r] * vscale), p1 * (vs[st][r + 1] * vscale), h, lo);
                const int i = 4 * (st & 1) + r;
                ph[st >> 1][i] = h[0];
                ph[st >> 1][i + 1] = h[1];
                pl[st >> 1][i] = lo[0];
                pl[st >> 1][i + 1] = lo[1];
            }
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
            o[dt] *= oal;
#pragma unroll
            for (int sp = 0; sp < 2; ++sp) {
                const v8h vf = v_frag(vals, dt, sp, lane);
                o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl[sp], o[dt], 0, 0, 0);
                o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph[sp], o[dt], 0, 0, 0);
            }
        }
    }
};

// What a lane's row (token t of the sequence) may see.
struct RowSight {
    int hi;   // context positions (a chain: all positions) up to hi
    int lo;   // from lo on, or below sinks
    int node0, M;  // a tree: slot node0 + j is node j, by its mask word
    const uint32_t* anc;  // null: a chain
    int sinks;
    __device__ __forceinline__ RowSight(const PagedAttn& a, const PagedSeq& sq, int t) {
        const bool tree = sq.dep0 >= 0;
        const int pos = sq.npast + (tree ? a.depth[sq.dep0 + t] : t);
        hi = tree ? sq.npast - 1 : pos;
        lo = a.window ? max(0, pos - a.window + 1) : 0;
        node0 = sq.npast;
        M = sq.M;
        anc = tree ? a.anc + sq.anc0 + (int64_t)t * sq.aw : nullptr;
        sinks = a.sinks;
    }
    __device__ __forceinline__ bool sees(int p) const {
        if (p <= hi) return p >= lo || p < sinks;
        const int j = p - node0;
        return anc && j < M && ((anc[j >> 5] >> (j & 31)) & 1u);
    }
};

// Workgroup = (item, kv head), neighbours on one XCD's L2 sharing a head where
// there are 8; the item's pages dealt to its four waves, whose softmaxes meet
// in LDS.
template <int HD, bool Q8>
__global__ void __launch_bounds__(256) k_paged_attn(PagedAttn a) {
    using W = WaveAttn<HD, Q8>;
    __shared__ float so[3][4 * W::NDT][64], sm[4][64], sl[4][64];
    __shared__ int se[4][64];
    const int kvh = blockIdx.x % a.p.n_kv;
    const PagedItem it = a.items[blockIdx.x / a.p.n_kv];
    const PagedSeq sq = a.p.seqs[it.seq];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, col = lane & 15, kq = lane >> 4;
    const int R = sq.M * a.gqa, rr = it.row0 + col, r = min(rr, R - 1), t = r / a.gqa;
    const int64_t tok = sq.tok0 + t;
    const int head = kvh * a.gqa + r % a.gqa;
    const bool vecq = !(((uintptr_t)a.q | (uintptr_t)(a.ldq * 4)) & 15);
    W wa;
    wa.query(a.q + tok * a.ldq + (int64_t)head * HD, kq, vecq);
    const RowSight sight(a, sq, t);
    // the pages that every row of the tile sees whole
    int hi = sight.hi, lo = sight.lo;
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) {
        hi = min(hi, __shfl_xor(hi, x, 64));
        lo = max(lo, __shfl_xor(lo, x, 64));
    }
    for (int i = it.i0 + w; i < it.i1; i += 4) {
        const int pg = i < it.s ? i : it.a + (i - it.s), p0 = pg * FTX_PAGE;
        const bool whole = p0 + FTX_PAGE - 1 <= hi && (p0 >= lo || p0 + FTX_PAGE <= sight.sinks);
        const uint8_t* blk = page_block(a.p, a.p.table[sq.tab0 + pg], kvh);
        wa.page(blk, lane, whole, [&](int st, int x) { return sight.sees(p0 + 16 * st + 4 * kq + x); });
    }
    wa.l += __shfl_xor(wa.l, 16, 64);
    wa.l += __shfl_xor(wa.l, 32, 64);
    sm[w][lane] = wa.m;
    sl[w][lane] = wa.l;
    se[w][lane] = wa.ev;
    if (w)
#pragma unroll
        for (int dt = 0; dt < W::NDT; ++dt)
#pragma unroll
            for (int x = 0; x < 4; ++x) so[w - 1][4 * dt + x][lane] = wa.o[dt][x];
    __syncthreads();
    if (w) return;
    float M = wa.m, f[4], L = 0.f;
    int EV = wa.ev;
#pragma unroll
    for (int x = 1; x < 4; ++x) {
        M = fmaxf(M, sm[x][lane]);
        EV = max(EV, se[x][lane]);
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        const float mx = sm[x][lane];
        f[x] = mx == M ? 1.f : __builtin_amdgcn_exp2f(mx - M);
        L += f[x] * sl[x][lane];
        f[x] = ldexpf(f[x], se[x][lane] - EV);
    }
    if (rr >= R) return;
    const bool part = it.part >= 0;
    const int64_t prow = ((int64_t)it.part * a.p.n_kv + kvh) * PAGED_TR + col;
    float* dst = part ? a.part + prow * HD : a.out + tok * a.ldo + (int64_t)head * HD;
    const bool vec = part || !(((uintptr_t)a.out | (uintptr_t)(a.ldo * 4)) & 15);
    const bool none = L == 0.f;  // no page of this part is seen by the row
#pragma unroll
    for (int dt = 0; dt < W::NDT; ++dt) {
        v4f y;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            float n = wa.o[dt][x] * f[0];
#pragma unroll
            for (int u = 1; u < 4; ++u) n += so[u - 1][4 * dt + x][lane] * f[u];
            y[x] = none ? 0.f : ldexpf(n / L, EV - 14);
        }
        st4(dst + 16 * dt + 4 * kq, y, vec);
    }
    if (part && kq == 0) {
        a.pml[2 * prow] = M;
        a.pml[2 * prow + 1] = L;
    }
}

// Workgroup (row tile with several partials, kv head):
// out = sum_i 2^(m_i - M) l_i o_i / sum_i 2^(m_i - M) l_i
template <int HD>
__global__ void __launch_bounds__(256) k_paged_combine(PagedAttn a) {
    const int kvh = blockIdx.x % a.p.n_kv;
    const PagedComb c = a.combs[blockIdx.x / a.p.n_kv];
    const PagedSeq sq = a.p.seqs[c.seq];
    const int R = sq.M * a.gqa;
    const bool vec = !(((uintptr_t)a.out | (uintptr_t)(a.ldo * 4)) & 15);
    for (int e = threadIdx.x; e < PAGED_TR * HD / 4; e += 256) {
        const int col = e / (HD / 4), d = e % (HD / 4) * 4, rr = c.row0 + col;
        if (rr >= R) continue;
        const int64_t step = (int64_t)a.p.n_kv * PAGED_TR;
        const int64_t p0 = ((int64_t)c.part0 * a.p.n_kv + kvh) * PAGED_TR + col;
        float M = -INFINITY;
        for (int i = 0; i < c.n; ++i) M = fmaxf(M, a.pml[2 * (p0 + i * step)]);
        float den = 0.f;
        v4f num = {0.f, 0.f, 0.f, 0.f};
        for (int i = 0; i < c.n; ++i) {
            const float mi = a.pml[2 * (p0 + i * step)];
            const float f = (mi == M ? 1.f : __builtin_amdgcn_exp2f(mi - M)) * a.pml[2 * (p0 + i * step) + 1];
            den += f;
        }
        for (int i = 0; i < c.n; ++i) {
            const float mi = a.pml[2 * (p0 + i * step)];
            const float f = (mi == M ? 1.f : __builtin_amdgcn_exp2f(mi - M)) * a.pml[2 * (p0 + i * step) + 1] / den;
            const v4f o = *(const v4f*)(a.part + (p0 + i * step) * HD + d);
#pragma unroll
            for (int x = 0; x < 4; ++x) num[x] += f * o[x];
        }
        const int64_t tok = sq.tok0 + rr / a.gqa;
        st4(a.out + tok * a.ldo + (int64_t)(kvh * a.gqa + rr % a.gqa) * HD + d, num, vec);
    }
}

}  // namespace

// f<HD, Q8>() of the pool's head size and type
#define PAGED_CASE(f, hd, q8)                                             \
    ((hd) == 64 ? ((q8) ? f<64, true> : f<64, false>)                     \
                : (hd) == 128 ? ((q8) ? f<128, true> : f<128, false>)     \
                              : ((q8) ? f<256, true> : f<256, false>))

hipError_t launch_paged_write(hipStream_t st, const PagedView& p, int64_t max_new_pages, const float* k, int64_t ldk,
                              const float* v, int64_t ldv) {
    if (max_new_pages == 0) return hipSuccess;
    const dim3 grid((unsigned)max_new_pages, (unsigned)p.nseq, (unsigned)p.n_kv);
    ktimed_launch(PAGED_CASE(k_paged_write, p.hd, p.q8), grid, dim3(256), 0, st, p, k, ldk, v, ldv);
    return hipGetLastError();
}

hipError_t launch_paged_read(hipStream_t st, const PagedView& p, int64_t max_pages, int context, float* k, int64_t ldk,
                             float* v, int64_t ldv) {
    if (max_pages == 0) return hipSuccess;
    const dim3 grid((unsigned)max_pages, (unsigned)p.nseq, (unsigned)p.n_kv);
    ktimed_launch(PAGED_CASE(k_paged_read, p.hd, p.q8), grid, dim3(256), 0, st, p, context, k, ldk, v, ldv);
    return hipGetLastError();
}

hipError_t launch_paged_attention(hipStream_t st, const PagedAttn& a) {
    if (a.n_items == 0) return hipSuccess;
    const dim3 grid((unsigned)a.n_items * (unsigned)a.p.n_kv);
    ktimed_launch(PAGED_CASE(k_paged_attn, a.p.hd, a.p.q8), grid, dim3(256), 0, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.n_combs == 0) return e;
    const dim3 cg((unsigned)a.n_combs * (unsigned)a.p.n_kv);
    auto* comb = a.p.hd == 64 ? k_paged_combine<64> : a.p.hd == 128 ? k_paged_combine<128> : k_paged_combine<256>;
    hipLaunchKernelGGL(comb, cg, dim3(256), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_paged_move(hipStream_t st, const PagedMove& m) {
    hipLaunchKernelGGL(k_paged_move, dim3((unsigned)m.n_kv, (unsigned)m.n_layer), dim3(256), 0, st, m);
    return hipGetLastError();
}
