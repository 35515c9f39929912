// k_paged.hip -- kernels of the paged KV caches: rows quantised into their
// pages and read back, and the attention of new tokens over pages.
#include <algorithm>
#include <type_traits>

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

// The largest of v over aligned groups of W lanes (16, 32 or 64), in all of
// them: within 16 lanes by DPP, whose moves cost no LDS round trip
template <int W>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
    auto step = [&](auto ctrl) {
        const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, 0xF, 0xF, false);
        v = v > o ? v : o;
    };
    step(std::integral_constant<int, 0xB1>{});   // quad_perm [1, 0, 3, 2]
    step(std::integral_constant<int, 0x4E>{});   // quad_perm [2, 3, 0, 1]
    step(std::integral_constant<int, 0x141>{});  // mirrored in 8 lanes
    step(std::integral_constant<int, 0x140>{});  // mirrored in 16
#pragma unroll
    for (int o = 16; o < W; o <<= 1) {
        const uint32_t t = (uint32_t)__shfl_xor((int)v, o, 64);
        v = v > t ? v : t;
    }
    return v;
}

// 127 x / a + 128 rounded to the nearest integer, ties to even, in the low byte
// of b; inv is 127 / a to 2^-22, so the product is off by less than 4e-5.
// Nearer than 1e-4 to a half the quotient is formed in 64 bits, whose rounding
// cannot cross a half: |254 x - (2 n + 1) a| is 0 or at least 2^-31 of its
// terms.  big: so large a row that its reciprocal is not to be had.
template <int N>
__device__ __forceinline__ void q8_bits(const float (&x)[N], float a, float inv, bool big, uint32_t (&b)[N]) {
    constexpr float MAGIC = 12582912.f + 128.f;  // 1.5 2^23: units in the last place
    float off = big ? 1.f : 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float t = __builtin_fmaf(x[i], inv, MAGIC);
        b[i] = __builtin_bit_cast(uint32_t, t);
        off = fmaxf(off, fabsf(__builtin_fmaf(x[i], inv, MAGIC - t)));
    }
    if (off > 0.4999f)
#pragma unroll
        for (int i = 0; i < N; ++i) b[i] = (uint32_t)((int)rint((double)x[i] * 127.0 / (double)a) + 128);
}

// The power of two that a row of halves is stored under
__device__ __forceinline__ int f16_exp(float a) {
    return a >= 0.00390625f && a <= 65504.f ? 0 : (int)((__builtin_bit_cast(uint32_t, a) >> 23) & 255) - 127 - 14;
}

// A workgroup of the store and of the read-back takes K or V of one page and kv
// head (its x: page, then head, then K or V: the heads' pieces of a token's row
// are written at about the same time, or the pieces of one head, a row apart,
// meet in a few memory channels: 162 us instead of 121 to read back 57138
// tokens of 8 heads of 128): slots s0 .. s1 - 1 of it, row by row where
// they are few, else the page's values as they lie in memory through LDS, so
// that both sides of the copy are whole runs (32 lanes a row of 128 floats;
// 16 bytes a thread of the page).
struct PageRows {
    uint8_t* vals;  // the page's K or V values
    float* scale;
    int s0, s1;
    int64_t row;  // of slot 0 in the matrix (it may lie before its start)
    int col;      // the kv head's first float
    bool isv;
};
template <int HD, bool Q8>
__device__ __forceinline__ PageRows page_rows(const PagedView& p, int context) {
    const PagedSeq sq = p.seqs[blockIdx.y];
    const int from = context ? 0 : sq.npast;
    const int z = blockIdx.x % (2 * p.n_kv);
    const int first = from / FTX_PAGE + blockIdx.x / (2 * p.n_kv);  // the page's place in the table
    PageRows r{};
    r.s0 = max(from - first * FTX_PAGE, 0);
    r.s1 = min(FTX_PAGE, sq.npast + sq.M - first * FTX_PAGE);
    if (r.s0 >= r.s1) return r;
    const int kvh = z >> 1;
    r.isv = z & 1;
    uint8_t* blk = page_block(p, p.table[sq.tab0 + first], kvh);
    r.vals = blk + (r.isv ? paged_values_bytes(HD, Q8) : 0);
    r.scale = (float*)(blk + 2 * paged_values_bytes(HD, Q8)) + (r.isv ? FTX_PAGE : 0);
    r.row = (int64_t)first * FTX_PAGE + (context ? sq.all0 : (int64_t)sq.tok0 - sq.npast);
    r.col = kvh * HD;
    return r;
}
constexpr int ROWS_FEW = 16;  // up to here a wave a row is no slower

// |x| as an integer: ordered as the magnitudes are, infinity and NaN above all
__device__ __forceinline__ uint32_t mag(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu; }

// How a row of largest magnitude `amax` (mag) is stored
template <bool Q8>
struct RowForm {
    float a, by;
    bool ok, zero;
    __device__ __forceinline__ explicit RowForm(uint32_t amax) {
        a = __builtin_bit_cast(float, amax);
        ok = a <= FLT_BIG;
        zero = !ok || a < ROW_TINY;
        if constexpr (Q8)
            by = zero ? 0.f : 127.f * __builtin_amdgcn_rcpf(a);
        else
            by = zero ? 0.f : ldexpf(1.f, -f16_exp(a));
    }
    __device__ __forceinline__ float scale() const {
        if (!ok) return __builtin_nanf("");
        if constexpr (Q8) return zero ? 0.f : a / 127.f;
        return zero ? 1.f : ldexpf(1.f, f16_exp(a));
    }
    // the values' bits in the page, in the low byte (half) of b; finite
    // whatever the row holds
    template <int N>
    __device__ __forceinline__ void bits(const float (&x)[N], uint32_t (&b)[N]) const {
        if constexpr (Q8) {
            q8_bits(x, a, by, !zero && a > 1e36f, b);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                b[i] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)(ok ? x[i] * by : 0.f));
        }
    }
};

// The page's image in LDS: 16-byte unit u at u ^ (4 bits of what lies above
// it), so that the units of one slot's dims (or one slot group's) lie in
// different banks: 8- to 16-way conflicts without it
__device__ __forceinline__ int image_unit(int u) { return u ^ (((u >> 4) ^ (u >> 6)) & 15); }
__device__ __forceinline__ int image_at(int byte) { return image_unit(byte >> 4) * 16 + (byte & 15); }

// ---------------------------------------------------------------- write
template <int HD, bool Q8>
__global__ void __launch_bounds__(256) k_paged_write(PagedView p, const float* __restrict__ k, int64_t ldk,
                                                     const float* __restrict__ v, int64_t ldv) {
    constexpr int E = HD / 64, D4 = HD / 4, EB = Q8 ? 1 : 2;
    __shared__ uint4 img[HD * FTX_PAGE * EB / 16];
    __shared__ uint32_t amax[FTX_PAGE];
    const PageRows pr = page_rows<HD, Q8>(p, 0);
    if (pr.s0 >= pr.s1) return;
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
    const int64_t ld = pr.isv ? ldv : ldk;
    const float* src = (pr.isv ? v : k) + pr.row * ld + pr.col;
    if (pr.s1 - pr.s0 < ROWS_FEW) {
        for (int slot = pr.s0 + w; slot < pr.s1; slot += 4) {
            float x[E];
            uint32_t a = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                x[e] = src[slot * ld + E * lane + e];
                a = max(a, mag(x[e]));
            }
            const RowForm<Q8> f(group_max<64>(a));
            uint32_t b[E];
            f.bits(x, b);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int d = E * lane + e;
                uint8_t* t = pr.vals + (pr.isv ? paged_v_at(slot, d, Q8) : paged_k_at(slot, d, Q8));
                if constexpr (Q8)
                    *t = (uint8_t)b[e];
                else
                    *(uint16_t*)t = (uint16_t)b[e];
            }
            if (lane == 0) pr.scale[slot] = f.scale();
        }
        return;
    }
    const bool vec = !(((uintptr_t)src | (uintptr_t)(ld * 4)) & 15);
    uint8_t* im = (uint8_t*)img;
    // four dims of four consecutive slots a thread: K's run along the dims, V's
    // along the slots
#pragma unroll
    for (int i0 = 0; i0 < FTX_PAGE / 4 * D4; i0 += 256) {
        const int i = i0 + tid, g = i / D4, d = i % D4 * 4;
        v4f x[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int slot = 4 * g + r;
            x[r] = slot >= pr.s0 && slot < pr.s1 ? ld4(src + slot * ld + d, vec) : v4f{0.f, 0.f, 0.f, 0.f};
        }
        uint32_t bits[4][4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint32_t a =
                group_max<D4>(max(max(mag(x[r][0]), mag(x[r][1])), max(mag(x[r][2]), mag(x[r][3]))));
            const RowForm<Q8> f(a);
            const float xr[4] = {x[r][0], x[r][1], x[r][2], x[r][3]};
            f.bits(xr, bits[r]);
            if (d == 0) amax[4 * g + r] = a;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            // K: slot 4 g + r, dims d ..+3; V: dim d + r, slots 4 g ..+3
            uint32_t b[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) b[e] = pr.isv ? bits[e][r] : bits[r][e];
            uint8_t* t = im + image_at(pr.isv ? paged_v_at(4 * g, d + r, Q8) : paged_k_at(4 * g + r, d, Q8));
            if constexpr (Q8)
                *(uint32_t*)t = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0C0C0400u),
                                                      __builtin_amdgcn_perm(b[1], b[0], 0x0C0C0400u), 0x05040100u);
            else
                *(uint2*)t = uint2{b[0] | b[1] << 16, b[2] | b[3] << 16};
        }
    }
    __syncthreads();
    if (tid >= pr.s0 && tid < pr.s1) pr.scale[tid] = RowForm<Q8>(amax[tid]).scale();
    const bool full = pr.s0 == 0 && pr.s1 == FTX_PAGE;
    for (int u = tid; u < HD * FTX_PAGE * EB / 16; u += 256) {
        if (full) {
            ((uint4*)pr.vals)[u] = img[image_unit(u)];
        } else if (!pr.isv) {
            const int slot = 16 * ((u >> 6) & 3) + (u & 15);
            if (slot >= pr.s0 && slot < pr.s1) ((uint4*)pr.vals)[u] = img[image_unit(u)];
        } else {
            // a unit holds 16 (8) slots: those of other tokens stay
#pragma unroll
            for (int x = 0; x < 16 / EB; ++x) {
                const int st = Q8 ? x >> 2 : 2 * ((u >> 6) & 1) + (x >> 2);
                const int slot = 16 * st + 4 * ((u >> 4) & 3) + (x & 3);
                if (slot < pr.s0 || slot >= pr.s1) continue;
                if constexpr (Q8)
                    pr.vals[u * 16 + x] = im[image_unit(u) * 16 + x];
                else
                    ((uint16_t*)pr.vals)[u * 8 + x] = ((const uint16_t*)im)[image_unit(u) * 8 + x];
            }
        }
    }
}

// ---------------------------------------------------------------- read back
template <int HD, bool Q8>
__global__ void __launch_bounds__(256) k_paged_read(PagedView p, int context, float* __restrict__ k, int64_t ldk,
                                                    float* __restrict__ v, int64_t ldv) {
    constexpr int E = HD / 64, D4 = HD / 4, EB = Q8 ? 1 : 2;
    __shared__ uint4 img[HD * FTX_PAGE * EB / 16];
    const PageRows pr = page_rows<HD, Q8>(p, context);
    if (pr.s0 >= pr.s1) return;
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
    const int64_t ld = pr.isv ? ldv : ldk;
    float* dst = (pr.isv ? v : k) + pr.row * ld + pr.col;
    if (pr.s1 - pr.s0 < ROWS_FEW) {
        for (int slot = pr.s0 + w; slot < pr.s1; slot += 4) {
            const float sc = pr.scale[slot];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int d = E * lane + e;
                const uint8_t* t = pr.vals + (pr.isv ? paged_v_at(slot, d, Q8) : paged_k_at(slot, d, Q8));
                dst[slot * ld + d] = (Q8 ? (float)((int)*t - 128) : (float)*(const _Float16*)t) * sc;
            }
        }
        return;
    }
#pragma unroll
    for (int u = tid; u < HD * FTX_PAGE * EB / 16; u += 256) img[image_unit(u)] = ((const uint4*)pr.vals)[u];
    __syncthreads();
    const bool vec = !(((uintptr_t)dst | (uintptr_t)(ld * 4)) & 15);
    const uint8_t* im = (const uint8_t*)img;
#pragma unroll
    for (int i0 = 0; i0 < FTX_PAGE / 4 * D4; i0 += 256) {
        const int i = i0 + tid, g = i / D4, d = i % D4 * 4;
        float q[4][4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint8_t* t = im + image_at(pr.isv ? paged_v_at(4 * g, d + r, Q8) : paged_k_at(4 * g + r, d, Q8));
#pragma unroll
            for (int e = 0; e < 4; ++e)
                q[r][e] = Q8 ? (float)((*(const uint32_t*)t >> (8 * e)) & 255) : (float)((const _Float16*)t)[e];
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int slot = 4 * g + r;
            if (slot < pr.s0 || slot >= pr.s1) continue;
            const float sc = pr.scale[slot];
            v4f y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = ((pr.isv ? q[e][r] : q[r][e]) - (Q8 ? 128.f : 0.f)) * sc;
            st4(dst + slot * ld + d, y, vec);
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

// A product rounded once, in a register: converted to halves in two places, it
// could otherwise be rounded from its exact value in one of them, and a low
// half would not fit its high half (seen: one weight in some 2^13 off by 2^-11).
__device__ __forceinline__ float rounded(float x) {
    asm("" : "+v"(x));
    return x;
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
                split_hl2(rounded(x[dc][i >> 2][i & 3] * qs), rounded(x[dc][i >> 2][(i & 3) + 1] * qs), h, lo);
                qh[dc][i] = h[0];
                qh[dc][i + 1] = h[1];
                ql[dc][i] = lo[0];
                ql[dc][i + 1] = lo[1];
            }
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) o[dt] = v4f{0.f, 0.f, 0.f, 0.f};
    }

    // A page's loads, issued together: the values of K (or V) as this lane's
    // operands, 16 bytes each, and the lane's 16 K and V scales
    static constexpr int NL = HD / (Q8 ? 16 : 8);  // 16-byte loads of K or of V
    struct Vals {
        uint4 u[NL];
    };
    struct Scales {
        v4f k[4], v[4];
    };
    static __device__ __forceinline__ void load_vals(Vals& x, const uint8_t* vals, int lane) {
#pragma unroll
        for (int i = 0; i < NL; ++i) x.u[i] = *(const uint4*)(vals + (i * 64 + lane) * 16);
    }
    static __device__ __forceinline__ void load_scales(Scales& x, const uint8_t* blk, int kq) {
        const float* scale = (const float*)(blk + 2 * paged_values_bytes(HD, Q8));
#pragma unroll
        for (int st = 0; st < 4; ++st) {
            x.k[st] = *(const v4f*)(scale + 16 * st + 4 * kq);
            x.v[st] = *(const v4f*)(scale + FTX_PAGE + 16 * st + 4 * kq);
        }
    }
    static __device__ __forceinline__ v8h k_frag(const Vals& x, int st, int dc) {
        if constexpr (Q8) {
            const uint4 u = x.u[(dc >> 1) * 4 + st];
            return dc & 1 ? u8x8(u.z, u.w) : u8x8(u.x, u.y);
        } else {
            return __builtin_bit_cast(v8h, x.u[dc * 4 + st]);
        }
    }
    static __device__ __forceinline__ v8h v_frag(const Vals& x, int dt, int sp) {
        if constexpr (Q8) {
            const uint4 u = x.u[dt];
            return sp ? u8x8(u.z, u.w) : u8x8(u.x, u.y);
        } else {
            return __builtin_bit_cast(v8h, x.u[dt * 2 + sp]);
        }
    }

    __device__ __forceinline__ void scores(v4f (&s)[4], const Vals& k) const {
#pragma unroll
        for (int st = 0; st < 4; ++st) {
            s[st] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int dc = 0; dc < NDC; ++dc) {
                const v8h kf = k_frag(k, st, dc);
                s[st] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[dc], s[st], 0, 0, 0);
                s[st] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qh[dc], s[st], 0, 0, 0);
            }
        }
    }

    // The page's weights from its scores; the sums so far brought to the new
    // maximum and V exponent.  seen(st, r): whether the row sees the slot
    // (whole: it sees all)
    template <typename Seen>
    __device__ __forceinline__ void soften(v4f (&s)[4], const Scales& sc, bool whole, Seen seen, v8h (&ph)[2],
                                           v8h (&pl)[2]) {
        v4f vs[4];
        float mx = -INFINITY, vm = 0.f;
#pragma unroll
        for (int st = 0; st < 4; ++st)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[st][r] = (s[st][r] * c2) * sc.k[st][r];
                vs[st][r] = sc.v[st][r];
            }
        if (!whole)
#pragma unroll
            for (int st = 0; st < 4; ++st)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool ok = seen(st, r);
                    s[st][r] = ok ? s[st][r] : -INFINITY;
                    vs[st][r] = ok ? vs[st][r] : 0.f;
                }
#pragma unroll
        for (int st = 0; st < 4; ++st)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
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
        const float vscale = ldexpf(1.f, 14 - en);
        const float oal = ldexpf(al, ev - en);
        m = mn;
        ev = en;
        l *= al;
#pragma unroll
        for (int st = 0; st < 4; ++st)
#pragma unroll
            for (int r = 0; r < 4; r += 2) {
                const float p0 = __builtin_amdgcn_exp2f(s[st][r] - mr);
                const float p1 = __builtin_amdgcn_exp2f(s[st][r + 1] - mr);
                l += p0 + p1;
                v2h h, lo;
                split_hl2(rounded(p0 * (vs[st][r] * vscale)), rounded(p1 * (vs[st][r + 1] * vscale)), h, lo);
                const int i = 4 * (st & 1) + r;
                ph[st >> 1][i] = h[0];
                ph[st >> 1][i + 1] = h[1];
                pl[st >> 1][i] = lo[0];
                pl[st >> 1][i + 1] = lo[1];
            }
        if (__builtin_amdgcn_ballot_w64(oal != 1.f))  // (wave-uniform)
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) o[dt] *= oal;
    }

    __device__ __forceinline__ void outputs(const Vals& v, const v8h (&ph)[2], const v8h (&pl)[2]) {
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int sp = 0; sp < 2; ++sp) {
                const v8h vf = v_frag(v, dt, sp);
                o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl[sp], o[dt], 0, 0, 0);
                o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph[sp], o[dt], 0, 0, 0);
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
__global__ void __launch_bounds__(256, HD <= 128 ? 2 : 1) k_paged_attn(PagedAttn a) {
    using W = WaveAttn<HD, Q8>;
    constexpr bool PRE = HD * (Q8 ? 1 : 2) <= 128, EARLY = PRE;  // as far as two waves a SIMD have the registers
    __shared__ float so[3][4 * W::NDT][64], sm[4][64], sl[4][64];
    __shared__ int se[4][64];
    const int kvh = blockIdx.x % a.p.n_kv;
    const PagedItem it = a.items[blockIdx.x / a.p.n_kv];
    const PagedSeq sq = it.q;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, col = lane & 15, kq = lane >> 4;
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
    // the wave's pages: entries i0 + w, + 4, ..; their ids 64 at a time in the
    // lanes.  A page's V loads are issued before its scores are formed, the
    // next page's K loads and scales (PRE) before its softmax, so that each
    // wait leaves the later loads in flight.
    const int n = max(0, (it.i1 - it.i0 - w + 3) >> 2);
    auto place = [&](int j) {  // in the table
        const int i = it.i0 + w + 4 * j;
        return i < it.s ? i : it.a + (i - it.s);
    };
    int ids = lane < n ? a.p.table[sq.tab0 + place(lane)] : 0;
    auto block_of = [&](int j) {
        if ((j & 63) == 0 && j) ids = j + lane < n ? a.p.table[sq.tab0 + place(j + lane)] : 0;
        return page_block(a.p, __builtin_amdgcn_readlane(ids, j & 63), kvh);
    };
    typename W::Vals kv, vv;
    typename W::Scales sc;
    const uint8_t* blk = nullptr;
    if (n) {
        blk = block_of(0);
        if (PRE) W::load_vals(kv, blk, lane);
    }
    for (int j = 0; j < n; ++j) {
        if (!PRE) W::load_vals(kv, blk, lane);
        W::load_scales(sc, blk, kq);
        if (EARLY) W::load_vals(vv, blk + paged_values_bytes(HD, Q8), lane);
        __builtin_amdgcn_sched_barrier(0);
        v4f s[4];
        wa.scores(s, kv);
        __builtin_amdgcn_sched_barrier(0);
        if (!EARLY) W::load_vals(vv, blk + paged_values_bytes(HD, Q8), lane);
        if (j + 1 < n) {
            blk = block_of(j + 1);
            if (PRE) W::load_vals(kv, blk, lane);
        }
        __builtin_amdgcn_sched_barrier(0);
        const int p0 = place(j) * FTX_PAGE;
        const bool whole = p0 + FTX_PAGE - 1 <= hi && (p0 >= lo || p0 + FTX_PAGE <= sight.sinks);
        v8h ph[2], pl[2];
        wa.soften(s, sc, whole, [&](int st, int x) { return sight.sees(p0 + 16 * st + 4 * kq + x); }, ph, pl);
        wa.outputs(vv, ph, pl);
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

// Workgroup (row of a tile with several partials, kv head):
// out = sum_i 2^(m_i - M) l_i o_i / sum_i 2^(m_i - M) l_i.  Every wave forms M
// and the sum itself; thread (g, d) adds the partials g, g + G, .. of dims
// 4 d .. 4 d + 3, the G sums meet in LDS.
template <int HD>
__global__ void __launch_bounds__(256) k_paged_combine(PagedAttn a) {
    constexpr int D4 = HD / 4, G = 256 / D4;
    __shared__ v4f red[G][D4];
    const int kvh = blockIdx.x % a.p.n_kv, col = blockIdx.y;
    const PagedComb c = a.combs[blockIdx.x / a.p.n_kv];
    const PagedSeq sq = a.p.seqs[c.seq];
    const int rr = c.row0 + col, lane = threadIdx.x & 63;
    if (rr >= sq.M * a.gqa) return;
    const int64_t step = (int64_t)a.p.n_kv * PAGED_TR;
    const int64_t p0 = ((int64_t)c.part0 * a.p.n_kv + kvh) * PAGED_TR + col;
    const float2* ml = (const float2*)a.pml + p0;
    float M = -INFINITY, den = 0.f;
    for (int i = lane; i < c.n; i += 64) M = fmaxf(M, ml[i * step].x);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    auto weight = [&](int i) {
        const float2 t = ml[i * step];
        return (t.x == M ? 1.f : __builtin_amdgcn_exp2f(t.x - M)) * t.y;
    };
    for (int i = lane; i < c.n; i += 64) den += weight(i);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) den += __shfl_xor(den, o, 64);
    const int g = threadIdx.x / D4, d = threadIdx.x % D4;
    v4f num = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = g; i < c.n; i += G) {
        const float f = weight(i) / den;
        const v4f o = *(const v4f*)(a.part + (p0 + i * step) * HD + 4 * d);
#pragma unroll
        for (int x = 0; x < 4; ++x) num[x] += f * o[x];
    }
    red[g][d] = num;
    __syncthreads();
    if (g) return;
#pragma unroll
    for (int x = 1; x < G; ++x) num += red[x][d];
    const int64_t tok = sq.tok0 + rr / a.gqa;
    const bool vec = !(((uintptr_t)a.out | (uintptr_t)(a.ldo * 4)) & 15);
    st4(a.out + tok * a.ldo + (int64_t)(kvh * a.gqa + rr % a.gqa) * HD + 4 * d, num, vec);
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
    const dim3 grid((unsigned)(max_new_pages * 2 * p.n_kv), (unsigned)p.nseq);
    ktimed_launch(PAGED_CASE(k_paged_write, p.hd, p.q8), grid, dim3(256), 0, st, p, k, ldk, v, ldv);
    return hipGetLastError();
}

hipError_t launch_paged_read(hipStream_t st, const PagedView& p, int64_t max_pages, int context, float* k, int64_t ldk,
                             float* v, int64_t ldv) {
    if (max_pages == 0) return hipSuccess;
    const dim3 grid((unsigned)(max_pages * 2 * p.n_kv), (unsigned)p.nseq);
    ktimed_launch(PAGED_CASE(k_paged_read, p.hd, p.q8), grid, dim3(256), 0, st, p, context, k, ldk, v, ldv);
    return hipGetLastError();
}

hipError_t launch_paged_attention(hipStream_t st, const PagedAttn& a) {
    if (a.n_items == 0) return hipSuccess;
    const dim3 grid((unsigned)a.n_items * (unsigned)a.p.n_kv);
    ktimed_launch(PAGED_CASE(k_paged_attn, a.p.hd, a.p.q8), grid, dim3(256), 0, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.n_combs == 0) return e;
    const dim3 cg((unsigned)a.n_combs * (unsigned)a.p.n_kv, (unsigned)std::min(PAGED_TR, a.rows_max));
    auto* comb = a.p.hd == 64 ? k_paged_combine<64> : a.p.hd == 128 ? k_paged_combine<128> : k_paged_combine<256>;
    hipLaunchKernelGGL(comb, cg, dim3(256), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_paged_move(hipStream_t st, const PagedMove& m) {
    hipLaunchKernelGGL(k_paged_move, dim3((unsigned)m.n_kv, (unsigned)m.n_layer), dim3(256), 0, st, m);
    return hipGetLastError();
}
