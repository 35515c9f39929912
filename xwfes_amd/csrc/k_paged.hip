// k_paged.hip -- kernels of the paged KV caches: rows quantised into their
// pages and read back, and the attention of new tokens over pages.
#include <algorithm>
#include <type_traits>

#include "mm_dev.h"
#include "paged_dev.h"

namespace {

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

// A workgroup of the store and of the read-back takes K or V of one page and kv
// head (its x: page, then head, then K or V: the heads' pieces of a token's row
// are written at about the same time, or the pieces of one head, a row apart,
// meet in a few memory channels: 162 us instead of 121 to read back 57138
// tokens of 8 heads of 128): slots s0 .. s1 - 1 of it, row by row where
// they are few, else the page's values as they lie in memory through LDS, so
// that both sides of the copy are whole runs (32 lanes a row of 128 floats;
// 16 bytes a thread of the page).
struct PageRows {
    uint8_t* blk;
    uint8_t* vals;  // the page's K or V values
    float* scale;
    uint8_t* mult;  // (of 4-bit rows)
    int s0, s1;
    int64_t row;  // of slot 0 in the matrix (it may lie before its start)
    int col;      // the kv head's first float
    bool isv;
};
template <int HD, int KT>
__device__ __forceinline__ PageRows page_rows(const PagedView& p, int context) {
    const int z = blockIdx.x % (2 * p.n_kv);
    PageRows r{};
    int page;
    if (p.touch && !context) {
        const PagedTouch to = p.touch[blockIdx.x / (2 * p.n_kv)];
        if (to.page < 0) return r;
        r.s0 = to.s0;
        r.s1 = to.s1;
        r.row = to.row;
        page = to.page;
    } else {
        const PagedSeq sq = p.seqs[blockIdx.y];
        const int from = context ? 0 : sq.npast;
        const int first = from / FTX_PAGE + blockIdx.x / (2 * p.n_kv);  // the page's place in the table
        r.s0 = max(from - first * FTX_PAGE, 0);
        r.s1 = min(FTX_PAGE, sq.npast + sq.M - first * FTX_PAGE);
        if (r.s0 >= r.s1) return r;
        r.row = (int64_t)first * FTX_PAGE + (context ? sq.all0 : (int64_t)sq.tok0 - sq.npast);
        page = p.table[sq.tab0 + first];
    }
    const int kvh = z >> 1;
    r.isv = z & 1;
    r.blk = page_block(p, page, kvh);
    r.vals = r.blk + (r.isv ? paged_values_bytes(HD, KT) : 0);
    r.scale = (float*)(r.blk + 2 * paged_values_bytes(HD, KT)) + (r.isv ? FTX_PAGE : 0);
    r.mult = r.blk + 2 * paged_values_bytes(HD, KT) + 2 * FTX_PAGE * 4 + (r.isv ? paged_mult_bytes(HD, KT) : 0);
    r.col = kvh * HD;
    return r;
}
constexpr int ROWS_FEW = PAGED_ROWS_FEW + 1;  // below it a wave a row is no slower

// The page's image in LDS: 16-byte unit u at u ^ (4 bits of what lies above
// it), so that the units of one slot's dims (or one slot group's) lie in
// different banks: 8- to 16-way conflicts without it
__device__ __forceinline__ int image_unit(int u) { return u ^ (((u >> 4) ^ (u >> 6)) & 15); }
__device__ __forceinline__ int image_at(int byte) { return image_unit(byte >> 4) * 16 + (byte & 15); }

// ---------------------------------------------------------------- write
// q = round(127 x / a) + 128 with scale a / 127, or half(x 2^-e) with scale 2^e,
// a the row's largest magnitude.  4 bytes read for one or two written; 2000
// tokens of 8 heads of 128, 8-bit: 8.0 us, where the bytes take 4.2 at a copy's
// rate and a launch that does nothing 2: bound by the latency of a workgroup's
// one pass, load, maximum, LDS, barrier and store.  A kernel without the image
// in LDS, its values written a row apart, took 24.  4 bits (q4_store_row's, paged_dev.h):
// 9.2 of 3.9.
template <int HD, int KT>
__global__ void __launch_bounds__(256) k_paged_write(PagedView p, const float* __restrict__ k, int64_t ldk,
                                                     const float* __restrict__ v, int64_t ldv) {
    constexpr bool Q8 = KT == PT_Q8, Q4 = KT == PT_Q4;
    constexpr int E = HD / 64, D4 = HD / 4, EB = Q8 ? 1 : 2, UNITS = paged_values_bytes(HD, KT) / 16;
    __shared__ uint4 img[UNITS];
    __shared__ uint32_t amax[FTX_PAGE];
    __shared__ uint8_t mult[Q4 ? FTX_PAGE * HD / 32 : 1];
    const PageRows pr = page_rows<HD, KT>(p, 0);
    if (pr.s0 >= pr.s1) return;
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
    const int64_t ld = pr.isv ? ldv : ldk;
    const float* src = (pr.isv ? v : k) + pr.row * ld + pr.col;
    if (pr.s1 - pr.s0 < ROWS_FEW) {
        for (int slot = pr.s0 + w; slot < pr.s1; slot += 4) {
            if constexpr (Q4) {
                q4_store_row(pr.blk, HD, slot, pr.isv, lane, [&](int d) { return src[slot * ld + d]; });
                continue;
            }
            float x[E];
            uint32_t a = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                x[e] = src[slot * ld + E * lane + e];
                a = max(a, mag(x[e]));
            }
            const RowForm<KT> f(group_max<64>(a));
            uint32_t b[E];
            f.bits(x, b);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int d = E * lane + e;
                uint8_t* t = pr.vals + (pr.isv ? paged_v_at(slot, d, KT) : paged_k_at(slot, d, KT));
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
        if constexpr (Q4) {
            // (a block of 32 dims: eight threads)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                uint32_t t = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) t = max(t, mag(q4_need(x[r][e])));
                const uint32_t top = group_max<D4>(t);
                const Q4Row f(top);
                float by;
                const int c = f.mult(group_max<8>(t), by);
#pragma unroll
                for (int e = 0; e < 4; ++e) bits[r][e] = f.bits(x[r][e], by);
                if ((d & 31) == 0) mult[paged_c_at(4 * g + r, d >> 5)] = (uint8_t)c;
                if (d == 0) amax[4 * g + r] = top;
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                // K: slot 4 g + r's eight dims about d, half of them the neighbour's;
                // V: slots 4 g ..+3 of dim d + r and, from four threads on, d + r + 16
                uint32_t word;
                if (pr.isv) {
                    word = (bits[0][r] | bits[1][r] << 16 | bits[2][r] << 8 | bits[3][r] << 24) << (d & 16 ? 4 : 0);
                    word |= (uint32_t)__shfl_xor((int)word, 4, 64);
                } else {
                    word = (bits[r][0] | bits[r][1] << 16 | bits[r][2] << 4 | bits[r][3] << 20) << (d & 4 ? 8 : 0);
                    word |= (uint32_t)__shfl_xor((int)word, 1, 64);
                }
                // (both threads of a word have it: each stores half of them)
                if (pr.isv ? (r >> 1) == ((d >> 4) & 1) : (r >> 1) == ((d >> 2) & 1))
                    *(uint32_t*)(im + (image_at(pr.isv ? paged_v_at(4 * g, d + r, KT) : paged_k_at(4 * g + r, d, KT)) &
                                       ~3)) = word;
            }
            continue;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint32_t a =
                group_max<D4>(max(max(mag(x[r][0]), mag(x[r][1])), max(mag(x[r][2]), mag(x[r][3]))));
            const RowForm<Q4 ? PT_Q8 : KT> f(a);
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
            uint8_t* t = im + image_at(pr.isv ? paged_v_at(4 * g, d + r, KT) : paged_k_at(4 * g + r, d, KT));
            if constexpr (Q8)
                *(uint32_t*)t = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0C0C0400u),
                                                      __builtin_amdgcn_perm(b[1], b[0], 0x0C0C0400u), 0x05040100u);
            else
                *(uint2*)t = uint2{b[0] | b[1] << 16, b[2] | b[3] << 16};
        }
    }
    __syncthreads();
    if constexpr (Q4) {
        if (tid >= pr.s0 && tid < pr.s1) pr.scale[tid] = Q4Row(amax[tid]).scale();
        for (int i = tid; i < FTX_PAGE * HD / 32; i += 256) {
            const int slot = 16 * ((i >> 2) & 3) + 4 * ((i >> 4) & 3) + (i & 3);
            if (slot >= pr.s0 && slot < pr.s1) pr.mult[i] = mult[i];
        }
    } else {
        if (tid >= pr.s0 && tid < pr.s1) pr.scale[tid] = RowForm<KT>(amax[tid]).scale();
    }
    const bool full = pr.s0 == 0 && pr.s1 == FTX_PAGE;
    for (int u = tid; u < UNITS; u += 256) {
        if (full) {
            ((uint4*)pr.vals)[u] = img[image_unit(u)];
        } else if (Q4 && !pr.isv) {
            // a unit holds two slots, 8 bytes each
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int slot = 16 * (2 * ((u >> 6) & 1) + x) + (u & 15);
                if (slot >= pr.s0 && slot < pr.s1) ((uint2*)pr.vals)[2 * u + x] = ((const uint2*)img)[2 * image_unit(u) + x];
            }
        } else if (Q4) {
            // 16: those of other tokens stay
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                const int slot = 16 * (x >> 2) + 4 * ((u >> 4) & 3) + ((x >> 1) & 1) + 2 * (x & 1);
                if (slot >= pr.s0 && slot < pr.s1) pr.vals[u * 16 + x] = im[image_unit(u) * 16 + x];
            }
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
// x = (byte - 128) scale, or half scale.  Bound by HBM, mostly its writes: four
// contexts of up to 16384 (57138 tokens in all, 8 heads of 128, 8-bit) 120 us,
// 4.9 TB/s, a large copy's rate; 4 bits 109 us, the same.
template <int HD, int KT>
__global__ void __launch_bounds__(256) k_paged_read(PagedView p, int context, float* __restrict__ k, int64_t ldk,
                                                    float* __restrict__ v, int64_t ldv) {
    constexpr bool Q8 = KT == PT_Q8, Q4 = KT == PT_Q4;
    constexpr int E = HD / 64, D4 = HD / 4, UNITS = paged_values_bytes(HD, KT) / 16;
    __shared__ uint4 img[UNITS];
    const PageRows pr = page_rows<HD, KT>(p, context);
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
                const uint8_t* t = pr.vals + (pr.isv ? paged_v_at(slot, d, KT) : paged_k_at(slot, d, KT));
                if constexpr (Q4) {
                    const int n = (*t >> (d & (pr.isv ? 16 : 2) ? 4 : 0) & 15) - 8;
                    dst[slot * ld + d] = (float)(n * (int)pr.mult[paged_c_at(slot, d >> 5)]) * sc;
                    continue;
                }
                dst[slot * ld + d] = (Q8 ? (float)((int)*t - 128) : (float)*(const _Float16*)t) * sc;
            }
        }
        return;
    }
#pragma unroll
    for (int u = tid; u < UNITS; u += 256) img[image_unit(u)] = ((const uint4*)pr.vals)[u];
    __syncthreads();
    const bool vec = !(((uintptr_t)dst | (uintptr_t)(ld * 4)) & 15);
    const uint8_t* im = (const uint8_t*)img;
#pragma unroll
    for (int i0 = 0; i0 < FTX_PAGE / 4 * D4; i0 += 256) {
        const int i = i0 + tid, g = i / D4, d = i % D4 * 4;
        float q[4][4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint8_t* t = im + image_at(pr.isv ? paged_v_at(4 * g, d + r, KT) : paged_k_at(4 * g + r, d, KT));
            if constexpr (Q4) {
                // (the thread's first byte in the word: K's second four dims are the bytes above)
                const uint32_t word = *(const uint32_t*)((uintptr_t)t & ~(uintptr_t)3) >>
                                      (pr.isv ? d & 16 ? 4 : 0 : d & 4 ? 8 : 0);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int at = pr.isv ? (e & 1) * 16 + (e >> 1) * 8 : (e & 1) * 16 + (e >> 1) * 4;
                    q[r][e] = (float)((int)((word >> at) & 15) - 8);
                }
                continue;
            }
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
            for (int e = 0; e < 4; ++e) {
                const float z = pr.isv ? q[e][r] : q[r][e];
                y[e] = Q4 ? z * (float)pr.mult[paged_c_at(slot, d >> 5)] * sc : (z - (Q8 ? 128.f : 0.f)) * sc;
            }
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
    const int64_t vb = paged_values_bytes(m.hd, m.kt), step = m.block * m.n_kv;
    const int64_t mb = paged_mult_bytes(m.hd, m.kt);
    for (int i = 0; i < m.n; ++i) {
        const int ss = m.src[i] % FTX_PAGE, ds = m.dst[i] % FTX_PAGE;
        const uint8_t* s = base + (m.src[i] / FTX_PAGE) * step;
        uint8_t* t = base + (m.dst[i] / FTX_PAGE) * step;
        if (m.src[i] == m.dst[i]) continue;
        if (m.kt == PT_Q4) {
            if (d < m.hd / 2) {
                const int kd = paged_k_dim(d), vd = paged_v_dim(d);
                t[paged_k_at(ds, kd, PT_Q4)] = s[paged_k_at(ss, kd, PT_Q4)];
                t[vb + paged_v_at(ds, vd, PT_Q4)] = s[vb + paged_v_at(ss, vd, PT_Q4)];
            }
            if (d < 2 * (m.hd / 32)) {
                const int64_t at = 2 * vb + 2 * FTX_PAGE * 4 + (d & 1) * mb;
                t[at + paged_c_at(ds, d >> 1)] = s[at + paged_c_at(ss, d >> 1)];
            }
        } else if (m.kt == PT_Q8) {
            t[paged_k_at(ds, d, PT_Q8)] = s[paged_k_at(ss, d, PT_Q8)];
            t[vb + paged_v_at(ds, d, PT_Q8)] = s[vb + paged_v_at(ss, d, PT_Q8)];
        } else {
            *(uint16_t*)(t + paged_k_at(ds, d, PT_F16)) = *(const uint16_t*)(s + paged_k_at(ss, d, PT_F16));
            *(uint16_t*)(t + vb + paged_v_at(ds, d, PT_F16)) = *(const uint16_t*)(s + vb + paged_v_at(ss, d, PT_F16));
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

// 4-bit values under their multipliers as halves (exact: |q c| <= 2040).  A nibble
// n = q + 8 under 0x64 is 1024 + n, four bits up under 0x54 it is 64 + n.
// (the constants in registers, so that `and` and `or` are one instruction)
__device__ __forceinline__ uint32_t in_sgpr(uint32_t x) {
    asm("" : "+s"(x));
    return x;
}
__device__ __forceinline__ uint32_t in_vgpr(uint32_t x) {
    asm("" : "+v"(x));
    return x;
}
__device__ __forceinline__ v2h q4_low(uint32_t x) {
    return __builtin_bit_cast(v2h, (x & in_sgpr(0x000F000Fu)) | in_vgpr(0x64006400u)) +
           v2h{(_Float16)(-1032.f), (_Float16)(-1032.f)};
}
__device__ __forceinline__ v2h q4_high(uint32_t x) {
    return __builtin_bit_cast(v2h, (x & in_sgpr(0x00F000F0u)) | in_vgpr(0x54005400u)) +
           v2h{(_Float16)(-72.f), (_Float16)(-72.f)};
}
__device__ __forceinline__ v8h join(v2h a, v2h b, v2h c, v2h d) {
    return v8h{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// a K word: eight dims of a slot
__device__ __forceinline__ v8h q4x8(uint32_t x, v8h c) {
    return join(q4_low(x), q4_high(x), q4_low(x >> 8), q4_high(x >> 8)) * c;
}
// two V words: four slots each of a dim's low nibbles or of another's high ones;
// c0, c1: the slots' multipliers, a byte each
__device__ __forceinline__ v8h q4x4x2(uint32_t x, uint32_t y, bool high, uint32_t c0, uint32_t c1) {
    const v2h o = {(_Float16)(-1024.f), (_Float16)(-1024.f)};
    const v2h a = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(c0, 0x64646464u, 0x00050004u)) + o;
    const v2h b = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(c0, 0x64646464u, 0x00070006u)) + o;
    const v2h c = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(c1, 0x64646464u, 0x00050004u)) + o;
    const v2h d = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(c1, 0x64646464u, 0x00070006u)) + o;
    if (high) return join(q4_high(x) * a, q4_high(x >> 8) * b, q4_high(y) * c, q4_high(y >> 8) * d);
    return join(q4_low(x) * a, q4_low(x >> 8) * b, q4_low(y) * c, q4_low(y >> 8) * d);
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

// The largest of x over the four lanes of a column (l, l ^ 16, l ^ 32, l ^ 48),
// by exchanging rows of 16 and halves of the wave in registers
__device__ __forceinline__ float col_max(float x) {
    auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false,
                                              false);
    x = fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
    r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false,
                                         false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}

// Levels that V scales are taken relative to: powers of 2^4.  The lowest: 2^-ev
// is finite; the smallest scale is 2^-114.
constexpr int EV_MIN = -112;
// Halves come in two kinds: rows kept as they are (scale 1) or larger (2 and up),
// and small ones, of scales 2^-23 and less whose values reach 2^15 all the same.
// Under level 0, which a row of scale 1 sets whatever its size from 2^-8 up, a
// small row's weights would lose their low bits, and more than those: a page of
// both kinds is taken in two visits, large slots then small ones, and the small
// ones' level of a row at level 0 is this (the highest that they have).
constexpr int EV_SMALL = -20;
enum Kind { ALL, LARGE, SMALL };
// whether a page of halves with slot lane's V scale v holds rows of both kinds
// (rows of zeros and slots never written have scale 0 and are neither)
__device__ __forceinline__ bool both_kinds(float v) {
    return __builtin_amdgcn_ballot_w64(v >= 1.f) && __builtin_amdgcn_ballot_w64((v > 0.f) & (v < 1.f));
}
// the lowest level with 2^level >= vm (1: 0, so that pages with and without a
// scale other than 1 weigh alike)
__device__ __forceinline__ int ev_level(float vm) {
    const uint32_t below = __builtin_bit_cast(uint32_t, fmaxf(vm, 1e-37f)) - 1u;
    return max(EV_MIN, (((int)(below >> 23) - 127 + 4) >> 2) * 4);
}

// One wave's online softmax over pages for a tile of 16 query rows.  Lane
// (col, kq) holds the scores of row col at slots 16 st + 4 kq + r and the
// outputs of row col at dims 16 dt + 4 kq + r.
// The query row is taken times log2 e / sqrt(hd) and a power of two, 2^e, that
// brings it to [2^6, 2^7); a score in units of log2 is 2^-e s ks exactly as
// s ks is, so one fma gives the weight's exponent: p = 2^(s ks 2^-e - off).
// off, as it was rounded, is the running maximum less 12 when it was last taken:
// it is taken anew where a page's maximum would bring a weight above 2^15 (p is at
// most that, also where a score's last place is worth more; the
// products of the sums so far, a third of a page's arithmetic, then fall to one
// page in ten).  l = sum p, and P.V of p vs 2^-ev in two halves, ev the level
// of the largest V scale that the row has seen.  out = 2^ev o / l.
template <int HD, int KT>
struct WaveAttn {
    // values that are integers under a scale of any size (8 and 4 bits), or halves
    static constexpr bool Q8 = KT != PT_F16;
    static constexpr int NDC = HD / 32, NDT = HD / 16;
    v8h qh[NDC], ql[NDC];
    v4f o[NDT];
    float off = -INFINITY;  // the weights' offset, -inf: nothing seen
    float l = 0.f, lp = 0.f;  // (this lane's slots only; lp: of the last page)
    float c2;               // 2^-e
    int ev = EV_MIN;

    // the query row at q, this lane's dims
    __device__ __forceinline__ void query(const float* q, int kq, bool vec) {
        v4f x[NDC][2];
        float a = 0.f;
#pragma unroll
        for (int dc = 0; dc < NDC; ++dc) {
            const int d0 = KT == PT_Q8 ? 64 * (dc >> 1) + 16 * kq + 8 * (dc & 1) : 32 * dc + 8 * kq;
            x[dc][0] = ld4(q + d0, vec);
            x[dc][1] = ld4(q + d0 + 4, vec);
        }
        const float by = 1.4426950408889634f / sqrtf((float)HD);
#pragma unroll
        for (int dc = 0; dc < NDC; ++dc)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = rounded(x[dc][i >> 2][i & 3] * by);
                x[dc][i >> 2][i & 3] = y;
                a = fabsf(y) <= FLT_BIG ? fmaxf(a, fabsf(y)) : a;
            }
        a = col_max(a);
        const int e = a > 0.f ? min(max(6 - f_exp(a), -121), 126) : 0;
        const float qs = ldexpf(1.f, e);
        c2 = ldexpf(1.f, -e);
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
    static constexpr int NL = HD / (KT == PT_F16 ? 8 : KT == PT_Q8 ? 16 : 32);  // 16-byte loads of K or of V
    struct Vals {
        uint4 u[NL];
        uint4 c[KT == PT_Q4 ? NDC : 1];  // 4 bits: the multipliers of each 32 dims
    };
    struct Scales {
        v4f k[4], v[4];
    };
    static __device__ __forceinline__ void load_vals(Vals& x, const uint8_t* vals, int lane) {
#pragma unroll
        for (int i = 0; i < NL; ++i) x.u[i] = *(const uint4*)(vals + (i * 64 + lane) * 16);
    }
    // 4 bits: the multipliers of a page for the lane's K (kq: of slots 16 st + m) or V operands
    static __device__ __forceinline__ void load_mults(Vals& x, const uint8_t* mult, int kq) {
#pragma unroll
        for (int g = 0; g < NDC; ++g) x.c[g] = *(const uint4*)(mult + 64 * g + 16 * kq);
    }
    static __device__ __forceinline__ void load_four(v4f (&x)[4], const float* at, int kq) {
#pragma unroll
        for (int st = 0; st < 4; ++st) x[st] = *(const v4f*)(at + 16 * st + 4 * kq);
    }
    static __device__ __forceinline__ void load_scales(Scales& x, const float* k, const float* v, int kq) {
        load_four(x.k, k, kq);
        load_four(x.v, v, kq);
    }
    static __device__ __forceinline__ uint32_t word(const uint4& u, int i) {
        return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w;
    }
    // lane: of the wave
    static __device__ __forceinline__ v8h k_frag(const Vals& x, int st, int dc, int lane) {
        if constexpr (KT == PT_Q4) {
            const uint32_t c = (word(x.c[dc], st) >> (8 * (lane & 3))) & 255;
            const _Float16 h = (_Float16)(float)c;
            return q4x8(word(x.u[(dc >> 1) * 2 + (st >> 1)], (st & 1) * 2 + (dc & 1)), v8h{h, h, h, h, h, h, h, h});
        } else if constexpr (Q8) {
            const uint4 u = x.u[(dc >> 1) * 4 + st];
            return dc & 1 ? u8x8(u.z, u.w) : u8x8(u.x, u.y);
        } else {
            return __builtin_bit_cast(v8h, x.u[dc * 4 + st]);
        }
    }
    static __device__ __forceinline__ v8h v_frag(const Vals& x, int dt, int sp) {
        if constexpr (KT == PT_Q4) {
            const uint32_t c0 = word(x.c[dt >> 1], 2 * sp), c1 = word(x.c[dt >> 1], 2 * sp + 1);
            return q4x4x2(word(x.u[dt >> 1], 2 * sp), word(x.u[dt >> 1], 2 * sp + 1), dt & 1, c0, c1);
        } else if constexpr (Q8) {
            const uint4 u = x.u[dt];
            return sp ? u8x8(u.z, u.w) : u8x8(u.x, u.y);
        } else {
            return __builtin_bit_cast(v8h, x.u[dt * 2 + sp]);
        }
    }

    // scores of a page, k(st, dc) its operands, of the query halves hi(dc), lo(dc)
    template <typename K, typename L, typename H>
    static __device__ __forceinline__ void scores_of(v4f (&s)[4], K k, L lo, H hi) {
#pragma unroll
        for (int st = 0; st < 4; ++st) s[st] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int dc = 0; dc < NDC; ++dc) {
            const v8h l8 = lo(dc), h8 = hi(dc);
#pragma unroll
            for (int st = 0; st < 4; ++st) {
                const v8h kf = k(st, dc);
                s[st] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, l8, s[st], 0, 0, 0);
                s[st] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, h8, s[st], 0, 0, 0);
            }
        }
    }

    // outputs to another V level
    __device__ __forceinline__ void raise(int en) {
        const float f = ldexpf(1.f, max(ev - en, -126));
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) o[dt] *= f;
        ev = en;
    }

    // scores by the K scales
    static __device__ __forceinline__ void by_scale(v4f (&s)[4], const Scales& sc) {
#pragma unroll
        for (int st = 0; st < 4; ++st) s[st] *= sc.k[st];
    }

    // the scores' largest of the row (`maximum`, which hands NaN on: fmaxf, from
    // products of another basic block, makes every score quiet first.  By the
    // compiler's own instructions, so that it keeps the products' wait)
    static __device__ __forceinline__ float row_max(const v4f (&s)[4]) {
        auto max3 = [](float x, float y, float z) {
            return __builtin_elementwise_maximum(__builtin_elementwise_maximum(x, y), z);
        };
        const float a = max3(s[0][0], s[0][1], s[0][2]), b = max3(s[0][3], s[1][0], s[1][1]);
        const float c = max3(s[1][2], s[1][3], s[2][0]), d = max3(s[2][1], s[2][2], s[2][3]);
        const float e = max3(s[3][0], s[3][1], s[3][2]);
        return col_max(max3(max3(a, b, c), max3(d, e, s[3][3]), s[3][3]));
    }

    // The page's weights from its scores (by_scale's); the sums so far brought to a new
    // offset or V level where one is needed.  ones: every scale of the page is 1
    // (sc is not read).  whole: the row sees every slot, else slot x by bit x of
    // sight.  pe: sc.v stands 2^-pe over, pe the level of the page's largest
    // V scale (whole pages of one kind only: what a row does not see must not set its
    // level), or NO_LEVEL.  kind: the page's slots, or its large or its small ones.
    static constexpr int NO_LEVEL = 1 << 20;
    __device__ __forceinline__ void soften(v4f (&s)[4], Scales& sc, bool ones, bool whole, int pe, Kind kind,
                                           uint64_t sight, int kq, v8h (&ph)[2], v8h (&pl)[2]) {
        if (!Q8 && kind != ALL) {
#pragma unroll
            for (int st = 0; st < 4; ++st)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if ((sc.v[st][r] < 1.f) == (kind == LARGE)) {
                        s[st][r] = -INFINITY;
                        sc.v[st][r] = 0.f;
                    }
        }
        if (!whole) {
            const uint64_t seen = sight >> (4 * kq);
#pragma unroll
            for (int st = 0; st < 4; ++st)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    // all ones or zeros
                    const uint32_t ok = __builtin_amdgcn_sbfe((int)(seen >> (st >= 2 ? 32 : 0)), 16 * (st & 1) + r, 1);
                    // (copies: a bit cast of a vector's element takes element 0)
                    const float x = s[st][r], y = sc.v[st][r];
                    s[st][r] = __builtin_bit_cast(
                        float, (__builtin_bit_cast(uint32_t, x) & ok) | (0xFF800000u & ~ok));  // -inf
                    if (!ones) sc.v[st][r] = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, y) & ok);
                }
        }
        l += lp;
        const float mx = row_max(s);
        // (rows that need none keep theirs: a row's bits are its own, not its tile's)
        const bool over = __builtin_fmaf(mx, c2, -off) > 15.f;
        if (__builtin_amdgcn_ballot_w64(over)) {
            float cand = __builtin_fmaf(mx, c2, -12.f);
            // (from 2^26 on the 12 may round to 16, then to nothing: the score itself)
            if (__builtin_fmaf(mx, c2, -cand) > 15.f) cand = mx * c2;
            if (cand > FLT_BIG) cand = __builtin_nanf("");  // (a score past fp32)
            const float on = over ? cand : off;
            const float al = off == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(off - on);
            off = on;
            l *= al;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) o[dt] *= al;
        }
        const float on = off == -INFINITY ? 0.f : off;  // (nothing seen yet: every weight is 0)
        float vf = 1.f;
        bool flat = true;
        if (ones) {
            // (a row that sees nothing here keeps its level: its weights are 0)
            const uint64_t any = whole ? ~0ull : __builtin_amdgcn_ballot_w64(sight != 0);
            if (__builtin_amdgcn_ballot_w64(ev < 0) & any) raise(whole || sight ? max(ev, 0) : ev);
            flat = !(__builtin_amdgcn_ballot_w64(ev != 0) & any);
            if (!flat) vf = ldexpf(1.f, -ev);
        } else if (pe != NO_LEVEL) {
            const int en = !Q8 && pe < 0 && ev == 0 ? EV_SMALL : max(ev, pe);
            if (__builtin_amdgcn_ballot_w64(ev != en)) raise(en);
            if (__builtin_amdgcn_ballot_w64(ev != pe)) {
                const float f = ldexpf(1.f, pe - ev);
#pragma unroll
                for (int st = 0; st < 4; ++st) sc.v[st] *= f;
            }
        } else {
            const float top = fmaxf(fmaxf(fmaxf(fmaxf(sc.v[0][0], sc.v[0][1]), fmaxf(sc.v[0][2], sc.v[0][3])),
                                          fmaxf(fmaxf(sc.v[1][0], sc.v[1][1]), fmaxf(sc.v[1][2], sc.v[1][3]))),
                                    fmaxf(fmaxf(fmaxf(sc.v[2][0], sc.v[2][1]), fmaxf(sc.v[2][2], sc.v[2][3])),
                                          fmaxf(fmaxf(sc.v[3][0], sc.v[3][1]), fmaxf(sc.v[3][2], sc.v[3][3]))));
            // (halves: the scales left are of one kind)
            const bool down = !Q8 && ev == 0 && __builtin_amdgcn_ballot_w64((top > 0.f) & (top < 1.f));
            if (__builtin_amdgcn_ballot_w64(down | (top > ldexpf(1.f, ev)))) {
                const int lev = ev_level(col_max(fmaxf(top, 0.f)));
                raise(down ? EV_SMALL : max(ev, lev));
            }
            const float f = ldexpf(1.f, -ev);
#pragma unroll
            for (int st = 0; st < 4; ++st) sc.v[st] *= f;
        }
        // (one loop for each form: tests inside it would part the exponentials.
        // A page's weights are added up by themselves, lp, so that a long sum
        // takes one rounding a page where the outputs take four; joined to l at
        // the next page: here it costs copies of the outputs, 480 -> 495 us for
        // three chunks of 1500 tokens, there none, 478)
        auto weigh = [&](auto by) {
            lp = 0.f;
#pragma unroll
            for (int st = 0; st < 4; ++st)
#pragma unroll
                for (int r = 0; r < 4; r += 2) {
                    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[st][r], c2, -on));
                    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[st][r + 1], c2, -on));
                    lp += p0;
                    lp += p1;
                    v2h h, lo;
                    split_hl2(by(p0, st, r), by(p1, st, r + 1), h, lo);
                    const int i = 4 * (st & 1) + r;
                    ph[st >> 1][i] = h[0];
                    ph[st >> 1][i + 1] = h[1];
                    pl[st >> 1][i] = lo[0];
                    pl[st >> 1][i + 1] = lo[1];
                }
        };
        if (!ones)
            weigh([&](float p, int st, int r) { return rounded(p * sc.v[st][r]); });
        else if (flat)
            weigh([&](float p, int, int) { return p; });
        else
            weigh([&](float p, int, int) { return rounded(p * vf); });
    }

    // v(dt, sp): the page's V operands
    template <typename V>
    __device__ __forceinline__ void outputs(V v, const v8h (&ph)[2], const v8h (&pl)[2]) {
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int sp = 0; sp < 2; ++sp) {
                const v8h vf = v(dt, sp);
                o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl[sp], o[dt], 0, 0, 0);
                o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph[sp], o[dt], 0, 0, 0);
            }
    }
};

// Scores of a page for NT tiles of 16 rows from operands in LDS, k(st, dc) K's,
// lo(x, dc) and hi(x, dc) tile x's query halves: the operands of four slot tiles
// are read while the products of the four before them run, on accumulators that
// do not wait for each other (left to itself the compiler reads one operand,
// waits and multiplies: three chunks of 1500 tokens of 8-bit 128 took 733 us,
// in this way 657).
template <int NDC, int NT, typename K, typename L, typename H>
__device__ __forceinline__ void staged_scores(v4f (&s)[NT][4], K k, L lo, H hi) {
    v8h f[2][4], l[2][NT];
    auto read = [&](int dc) {
#pragma unroll
        for (int st = 0; st < 4; ++st) f[dc & 1][st] = k(st, dc);
#pragma unroll
        for (int x = 0; x < NT; ++x) l[dc & 1][x] = lo(x, dc);
    };
    read(0);
#pragma unroll
    for (int dc = 0; dc < NDC; ++dc) {
        if (dc + 1 < NDC) read(dc + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int st = 0; st < 4; ++st)
#pragma unroll
            for (int x = 0; x < NT; ++x)
                s[x][st] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[dc & 1][st], l[dc & 1][x],
                                                                  dc ? s[x][st] : v4f{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
        for (int st = 0; st < 4; ++st)
#pragma unroll
            for (int x = 0; x < NT; ++x)
                s[x][st] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[dc & 1][st], hi(x, dc), s[x][st], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    }
}
// Outputs of a page, v(dt, sp) its V operands, read in the same way
template <int NT, typename W, typename V>
__device__ __forceinline__ void staged_outputs(W* wa, V v, const v8h (&ph)[NT][2], const v8h (&pl)[NT][2]) {
    v8h f[2][4];
#pragma unroll
    for (int x = 0; x < 4; ++x) f[0][x] = v(x, 0);
    constexpr int NG = W::NDT / 2;  // groups: four dim tiles, one half of the slots
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        if (g + 1 < NG)
#pragma unroll
            for (int x = 0; x < 4; ++x) f[(g + 1) & 1][x] = v((g + 1) / 2 * 4 + x, (g + 1) & 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int y = 0; y < NT; ++y)
                wa[y].o[g / 2 * 4 + x] =
                    __builtin_amdgcn_mfma_f32_16x16x32_f16(f[g & 1][x], pl[y][g & 1], wa[y].o[g / 2 * 4 + x], 0, 0, 0);
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int y = 0; y < NT; ++y)
                wa[y].o[g / 2 * 4 + x] =
                    __builtin_amdgcn_mfma_f32_16x16x32_f16(f[g & 1][x], ph[y][g & 1], wa[y].o[g / 2 * 4 + x], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// What a lane's row (token t of the sequence) may see: slots lo .. hi and those
// below sinks (a chain: up to its own; a tree: of the context), and of a tree's
// nodes those of its mask words.
struct RowSight {
    int hi, lo, sinks;
    int node0, aw;
    const uint32_t* anc;  // null: a chain
    __device__ __forceinline__ RowSight(const PagedAttn& a, const PagedSeq& sq, int t) {
        const bool tree = sq.dep0 >= 0;
        const int pos = sq.npast + (tree ? a.depth[sq.dep0 + t] : t);
        hi = tree ? sq.npast - 1 : pos;
        lo = a.window ? max(0, pos - a.window + 1) : 0;
        sinks = min(a.sinks, hi + 1);
        node0 = sq.npast;
        aw = sq.aw;
        anc = tree ? a.anc + sq.anc0 + (int64_t)t * sq.aw : nullptr;
    }
    static __device__ __forceinline__ uint64_t below(int n) {  // bits 0 .. n - 1
        return n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1;
    }
    // bit x: whether slot p0 + x is seen
    __device__ __forceinline__ uint64_t page(int p0) const {
        uint64_t v = (below(hi + 1 - p0) & ~below(lo - p0)) | below(sinks - p0);
        const int j0 = p0 - node0;
        if (anc && j0 > -FTX_PAGE && j0 < 32 * aw) {
            const int w = max(j0, 0) >> 5;
            const uint64_t x = anc[w] | (uint64_t)(w + 1 < aw ? anc[w + 1] : 0u) << 32;
            if (j0 < 0) {
                v |= x << -j0;
            } else {
                const uint64_t y = w + 2 < aw ? anc[w + 2] : 0u;
                v |= x >> (j0 & 31) | (j0 & 31 ? y << (64 - (j0 & 31)) : 0);
            }
        }
        return v;
    }
};

// Few rows: workgroup = (item, kv head), neighbours on one XCD's L2 sharing a
// head where there are 8; the item's pages dealt to its NW waves, whose
// softmaxes meet in LDS (of eight, the last four with the first four before).
// Four waves take a part of a list, eight a whole one where that is faster.  For one token a sequence bound by HBM, the pages
// straight to registers: 16 sequences of 820 to 8192 slots (8-bit, 8 kv heads
// of 128) 35 us, where a kernel of the loads alone takes 31.4 (5.3 TB/s); one
// of 131072 (halves) 104 us, the loads alone 104.  Of 4 bits, rows that do not fit
// FoldAttn's columns: 16 sequences of 8 tokens under a window of 4096 (64 dims, 32
// rows a kv head) 28.3 us a call with the join, 507 vector instructions a page and tile,
// the vector units busy for 65% of the cycles, the rest the start and the end of short
// lists; two tiles a wave that share their operands: 64 dims 28.3 ->
// 26.8, 128 dims 34.3 -> 38.2 (28 registers spilled) and one sequence of 8 tokens 10.8
// -> 16.1, so not; nibbles as FoldAttn takes them 28.0 -> 27.7 and, with 67 spilled,
// 33.9 -> 50.4.  (Joining the partials in the
// last workgroup of a list instead of a launch of their own: the same for
// short lists, 14 us slower for one of 131072; by fences 60 us slower.)
template <int HD, int KT, int NW>
__global__ void __launch_bounds__(64 * NW, HD <= 128 ? 2 : 1) k_paged_attn(PagedAttn a) {
    using W = WaveAttn<HD, KT>;
    constexpr bool Q8 = W::Q8;
    constexpr bool PRE = paged_values_bytes(HD, KT) <= 8192, EARLY = PRE;  // as far as two waves a SIMD have the registers
    // the query's halves, of which the waves have the same: in LDS where
    // they would leave too few registers for the values in flight (halves of
    // 128 dims: 37 spilled, 129 us for one token over 131072; so 104)
    constexpr bool QLDS = !Q8 && HD >= 128;
    __shared__ v8h qs[QLDS ? 2 : 1][W::NDC][64];
    __shared__ float so[NW == 4 ? 3 : 4][4 * W::NDT][64], sm[NW][64], sl[NW][64];
    __shared__ int se[NW][64];
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
    if constexpr (QLDS) {
        if (w == 0)
#pragma unroll
            for (int dc = 0; dc < W::NDC; ++dc) {
                qs[0][dc][lane] = wa.qh[dc];
                qs[1][dc][lane] = wa.ql[dc];
            }
        __syncthreads();
    }
    const RowSight sight(a, sq, t);
    // the pages that every row of the tile sees whole
    int hi = sight.hi, lo = sight.lo;
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) {
        hi = min(hi, __shfl_xor(hi, x, 64));
        lo = max(lo, __shfl_xor(lo, x, 64));
    }
    hi = __builtin_amdgcn_readfirstlane(hi);
    lo = __builtin_amdgcn_readfirstlane(lo);
    // the wave's pages: entries i0 + w, + NW, ..; their ids 64 at a time in the
    // lanes.  A page's V loads are issued before its scores are formed, the
    // next page's K loads and scales (PRE) before its softmax, so that each
    // wait leaves the later loads in flight.
    // (none, of tables built on the GPU: looked at here, where the item's other parts
    // have been waited for; at the start it takes 0.3 us)
    if (it.seq < 0) return;
    const int n = max(0, (it.i1 - it.i0 - w + NW - 1) / NW);
    auto place = [&](int j) {  // in the table
        const int i = it.i0 + w + NW * j;
        return i < it.s ? i : it.a + (i - it.s);
    };
    int ids = lane < n ? a.p.table[sq.tab0 + place(lane)] : 0;
    auto block_of = [&](int j) {
        if ((j & 63) == 0 && j) ids = j + lane < n ? a.p.table[sq.tab0 + place(j + lane)] : 0;
        return page_block(a.p, __builtin_amdgcn_readlane(ids, j & 63), kvh);
    };
    constexpr int64_t VB = paged_values_bytes(HD, KT), MB = paged_mult_bytes(HD, KT), MULT = 2 * VB + 2 * FTX_PAGE * 4;
    auto load_k = [&](typename W::Vals& x, const uint8_t* b) {
        W::load_vals(x, b, lane);
        if constexpr (KT == PT_Q4) W::load_mults(x, b + MULT, col >> 2);
    };
    auto load_v = [&](typename W::Vals& x, const uint8_t* b) {
        W::load_vals(x, b + VB, lane);
        if constexpr (KT == PT_Q4) W::load_mults(x, b + MULT + MB, kq);
    };
    typename W::Vals kv, vv;
    typename W::Scales sc;
    const uint8_t* blk = nullptr;
    if (n) {
        blk = block_of(0);
        if (PRE) load_k(kv, blk);
    }
    bool second = false;  // a page of large and small rows of halves: its small ones
    for (int j = 0; j < n;) {
        if (!PRE) load_k(kv, blk);
        const float* scale = (const float*)(blk + 2 * VB);
        float k1 = 0.f, v1 = 0.f;
        if constexpr (Q8) {
            W::load_scales(sc, scale, scale + FTX_PAGE, kq);
        } else {
            // (a page of halves has scales other than 1 where rows are very
            // large or small: they are loaded then)
            k1 = scale[lane];
            v1 = scale[FTX_PAGE + lane];
        }
        if (EARLY) load_v(vv, blk);
        __builtin_amdgcn_sched_barrier(0);
        v4f s[4];
        auto kf = [&](int st, int dc) { return W::k_frag(kv, st, dc, lane); };
        if constexpr (QLDS) {
            asm volatile("" ::: "memory");  // (read again for every page)
            W::scores_of(s, kf, [&](int dc) { return qs[1][dc][lane]; }, [&](int dc) { return qs[0][dc][lane]; });
        } else {
            W::scores_of(s, kf, [&](int dc) { return wa.ql[dc]; }, [&](int dc) { return wa.qh[dc]; });
        }
        __builtin_amdgcn_sched_barrier(0);
        const bool ones = !Q8 && !__builtin_amdgcn_ballot_w64((k1 != 1.f) | (v1 != 1.f));
        if (!Q8 && !ones) W::load_scales(sc, scale, scale + FTX_PAGE, kq);
        if (!EARLY) load_v(vv, blk);
        const int p0 = place(j) * FTX_PAGE;
        const bool both = !Q8 && !ones && both_kinds(v1), again = both && !second;
        if (again) {
            if (PRE) load_k(kv, blk);
        } else if (++j < n) {
            blk = block_of(j);
            if (PRE) load_k(kv, blk);
        }
        __builtin_amdgcn_sched_barrier(0);
        const bool whole = p0 + FTX_PAGE - 1 <= hi && (p0 >= lo || p0 + FTX_PAGE <= a.sinks);
        v8h ph[2], pl[2];
        if (!ones) W::by_scale(s, sc);
        wa.soften(s, sc, ones, whole, W::NO_LEVEL, !both ? ALL : second ? SMALL : LARGE, whole ? 0 : sight.page(p0), kq, ph,
                  pl);
        wa.outputs([&](int dt, int sp) { return W::v_frag(vv, dt, sp); }, ph, pl);
        second = again;
    }
    wa.l += wa.lp;
    wa.l += __shfl_xor(wa.l, 16, 64);
    wa.l += __shfl_xor(wa.l, 32, 64);
    if constexpr (NW == 8) {
        // waves 4 to 7 into 0 to 3
        if (w >= 4) {
            sm[w][lane] = wa.off;
            sl[w][lane] = wa.l;
            se[w][lane] = wa.ev;
#pragma unroll
            for (int dt = 0; dt < W::NDT; ++dt)
#pragma unroll
                for (int x = 0; x < 4; ++x) so[w - 4][4 * dt + x][lane] = wa.o[dt][x];
        }
        __syncthreads();
        if (w < 4) {
            const float mo = sm[w + 4][lane], M = fmaxf(wa.off, mo);
            const int eo = se[w + 4][lane], EV = max(wa.ev, eo);
            const float f0 = wa.off == M ? 1.f : __builtin_amdgcn_exp2f(wa.off - M);
            const float f1 = mo == M ? 1.f : __builtin_amdgcn_exp2f(mo - M);
            const float g0 = ldexpf(f0, wa.ev - EV), g1 = ldexpf(f1, eo - EV);
            wa.l = wa.l * f0 + sl[w + 4][lane] * f1;
            wa.off = M;
            wa.ev = EV;
#pragma unroll
            for (int dt = 0; dt < W::NDT; ++dt)
#pragma unroll
                for (int x = 0; x < 4; ++x) wa.o[dt][x] = wa.o[dt][x] * g0 + so[w][4 * dt + x][lane] * g1;
        }
        __syncthreads();
    }
    sm[w][lane] = wa.off;
    sl[w][lane] = wa.l;
    se[w][lane] = wa.ev;
    if (w && w < 4)
#pragma unroll
        for (int dt = 0; dt < W::NDT; ++dt)
#pragma unroll
            for (int x = 0; x < 4; ++x) so[w - 1][4 * dt + x][lane] = wa.o[dt][x];
    __syncthreads();
    if (w) return;
    float M = wa.off, f[4], L = 0.f;
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
    // (0: no page of this part is seen by the row; of a whole list, every score is below fp32: NaN)
    const float inv = part && L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int dt = 0; dt < W::NDT; ++dt) {
        v4f y;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            float n = wa.o[dt][x] * f[0];
#pragma unroll
            for (int u = 1; u < 4; ++u) n += so[u - 1][4 * dt + x][lane] * f[u];
            y[x] = ldexpf(n * inv, EV);
        }
        st4(dst + 16 * dt + 4 * kq, y, vec);
    }
    if (part && kq == 0) {
        a.pml[2 * prow] = M;
        a.pml[2 * prow + 1] = L;
    }
}

// ---------------------------------------------------------------- few rows of 4 bits
// A lane's value from lane `st` of its group of U (2 or 4), or from the lane across
template <int U, int ST>
__device__ __forceinline__ float of_lane(float x) {
    constexpr int b = ST % U, ctrl = U == 4 ? b * 0x55 : b | b << 2 | (2 + b) << 4 | (2 + b) << 6;
    return __builtin_bit_cast(
        float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), ctrl, 0xF, 0xF, false));
}
template <int X>  // 1 or 2
__device__ __forceinline__ float across(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), X == 1 ? 0xB1 : 0x4E,
                                                                 0xF, 0xF, false));
}

// One wave's online softmax over pages of 4-bit rows for at most 16 / U query
// rows: a product's 16 columns are U for each row, column U r + u of row r.
//   Scores: slot tile st goes to column u = st % U (the others' query is zeros), so
// that the tiles share their sums' registers and each lane keeps the scores of one
// tile (two of U = 2): the softmax of a page is 4 (8) weights a lane and not 16.
// K's operand is the nibbles n = q + 8, bits 4 to 7 of halves (n 2^-20), and the sums
// start at -8 sum q of the block; a slot's multiplier of a block is applied once, to
// the block's sum.  A product's sum keeps some 24 bits below the largest that its
// operands' exponents allow, so a nibble needs its place near the top of a half's bits:
// as the low bits, 2^-24, with two shifts less for eight dims, outputs are off by
// 6.8e-6 of their size and not 5.6e-7 (in bits 6 to 9, a shift more, 4.8e-7; 131072
// slots 35.5, 36.3 and 36.5 us).
//   Outputs: column u takes the weights times the slots' multipliers of block U j + u
// and so holds the output dims of its blocks (the others' are not used).  V's
// operand is signed: a sum over unsigned values less 8 times the weights' would leave
// a dim whose values are all zero with the rounding of that sum.
// Bound by the SIMDs' vector instructions (82% of the cycles of long lists by 16-row
// tiles; products run beside them) and, with lists long enough, by HBM: 64
// sequences of 16384 slots (8 kv heads of 128, 4 query heads each) 223 us, 5.4 TB/s, which is what loads
// alone take.  In 16-row tiles, 950 vector instructions a page, one token of 16 sequences over
// 820 to 8192 slots takes 41.6 us; folded with signed K operands and the multipliers
// on partial sums, 600 a page, 23.7; as here, 530, 23.5, and longer lists 4 to 8% less.
// Sums, offsets and V levels as in WaveAttn; weights are taken times c / 256, rounded
// with the scale and again with the multiplier (WaveAttn's once: its operands are the
// integers q c): 2^-24 more beside the 2^-22 of their two halves.
template <int HD, int U>
struct FoldAttn {
    static constexpr int NB = HD / 32, J = NB > U ? NB / U : 1, NDT = HD / 16, S = 4 / U, NL = HD / 32, OWN = 2 * J;
    static constexpr int64_t VB = paged_values_bytes(HD, PT_Q4), MB = paged_mult_bytes(HD, PT_Q4);
    static constexpr float NIBBLE = 0x1p-20f;  // what a nibble of K's operand counts
    float bias[NB];  // -8 sum q of the blocks
    v4f o[NDT];
    float off = -INFINITY, l = 0.f, lp = 0.f, c2;
    int ev = EV_MIN;
    // the query's halves in LDS, [block][high, low][kq][row], and as many zeros behind
    // them, which the lanes of the other slot tiles read
    // (in the banks beside those of the same lanes' halves)
    static constexpr int QROWS = 16 / U, QN = NB * 2 * 4 * QROWS, QZ = QN + QROWS;
    typedef v8h Query[QN + QZ];

    // the largest of a row's lanes
    static __device__ __forceinline__ float row_top(float x) {
        x = fmaxf(x, across<1>(x));
        if constexpr (U == 4) x = fmaxf(x, across<2>(x));
        return col_max(x);
    }

    // The query row at q, to LDS if `store`
    __device__ __forceinline__ void query(const float* q, int u, int r, int kq, bool vec, bool store, v8h* qs) {
        // (each lane the blocks U j + u; heads of 64 dims have two)
        v4f x[J][2];
        float a = 0.f;
        const bool any = u < NB;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int d0 = 32 * (U * j + (any ? u : 0)) + 8 * kq;
            x[j][0] = ld4(q + d0, vec);
            x[j][1] = ld4(q + d0 + 4, vec);
        }
        const float by = 1.4426950408889634f / sqrtf((float)HD);
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = rounded(x[j][i >> 2][i & 3] * by);
                x[j][i >> 2][i & 3] = y;
                a = fabsf(y) <= FLT_BIG ? fmaxf(a, fabsf(y)) : a;
            }
        a = row_top(a);
        const int e = a > 0.f ? min(max(6 - f_exp(a), -121), 126) : 0;
        const float qs1 = ldexpf(1.f, e);
        c2 = ldexpf(1.f, -e);
        float own[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
            v8h h, lo;
            double sum = 0.0;
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                v2h hh, ll;
                split_hl2(rounded(x[j][i >> 2][i & 3] * qs1), rounded(x[j][i >> 2][(i & 3) + 1] * qs1), hh, ll);
                h[i] = hh[0];
                h[i + 1] = hh[1];
                lo[i] = ll[0];
                lo[i + 1] = ll[1];
                // (a half and its rest add up exactly)
                sum += (double)((float)hh[0] + (float)ll[0]) + (double)((float)hh[1] + (float)ll[1]);
            }
            sum += __shfl_xor(sum, 16, 64);
            sum += __shfl_xor(sum, 32, 64);
            own[j] = (float)(sum * (-8.0 * NIBBLE));
            if (store && any) {
                const int dc = U * j + u;
                qs[((dc * 2 + 0) * 4 + kq) * QROWS + r] = h;
                qs[((dc * 2 + 1) * 4 + kq) * QROWS + r] = lo;
            }
        }
        auto share = [&](auto u_) {
            constexpr int x = decltype(u_)::value;
#pragma unroll
            for (int j = 0; j < J; ++j)
                if (U * j + x < NB) bias[U * j + x] = of_lane<U, x>(own[j]);
        };
        share(std::integral_constant<int, 0>{});
        share(std::integral_constant<int, 1>{});
        if constexpr (U == 4) {
            share(std::integral_constant<int, 2>{});
            share(std::integral_constant<int, 3>{});
        }
        if (store)
            for (int i = threadIdx.x & 63; i < QZ; i += 64) qs[QN + i] = v8h{};
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) o[dt] = v4f{0.f, 0.f, 0.f, 0.f};
    }

    // A page's loads of K or V: values, the lane's blocks' multipliers of its 16
    // slots, the scales of the slots that it keeps
    struct Keys {
        uint4 u[NL];
        uint32_t c[NB][S];  // the multipliers of the lane's slots
        v4f s[S];
    };
    struct Vals {
        uint4 u[NL], c[J];  // the lane's blocks' multipliers of its 16 slots
        v4f s[S];
    };
    static __device__ __forceinline__ void load_scales(v4f (&s)[S], const float* scale, int u, int kq) {
#pragma unroll
        for (int a = 0; a < S; ++a) s[a] = *(const v4f*)(scale + 16 * (U * a + u) + 4 * kq);
    }
    static __device__ __forceinline__ void load(Keys& x, const uint8_t* blk, int u, int kq, int lane) {
#pragma unroll
        for (int i = 0; i < NL; ++i) x.u[i] = *(const uint4*)(blk + (i * 64 + lane) * 16);
        const uint8_t* mult = blk + 2 * VB + 2 * FTX_PAGE * 4;
#pragma unroll
        for (int g = 0; g < NB; ++g)
#pragma unroll
            for (int a = 0; a < S; ++a) x.c[g][a] = *(const uint32_t*)(mult + 64 * g + 16 * kq + 4 * (U * a + u));
        load_scales(x.s, (const float*)(blk + 2 * VB), u, kq);
    }
    static __device__ __forceinline__ void load(Vals& x, const uint8_t* blk, int u, int kq, int lane) {
#pragma unroll
        for (int i = 0; i < NL; ++i) x.u[i] = *(const uint4*)(blk + VB + (i * 64 + lane) * 16);
        const uint8_t* mult = blk + 2 * VB + 2 * FTX_PAGE * 4 + MB;
#pragma unroll
        for (int j = 0; j < J; ++j) x.c[j] = *(const uint4*)(mult + 64 * (U * j + u % NB) + 16 * kq);
        load_scales(x.s, (const float*)(blk + 2 * VB) + FTX_PAGE, u, kq);
    }
    static __device__ __forceinline__ uint32_t word(const uint4& x, int i) {
        return i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w;
    }
    // multiplier of slot 16 st + 4 kq + i
    static __device__ __forceinline__ float mult(const uint4& c, int st, int i) {
        return (float)((word(c, st) >> (8 * i)) & 255);
    }

    // Eight products, between each two of which go four or five of the vector
    // instructions that make the next eight's operands
    static __device__ __forceinline__ void beside() {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, 5, 0);
        }
    }

    // the scores, by the K scales, of the lane's slots: tile st's products take the
    // query in the lanes that keep it and zeros in the others, so that a block's sums
    // of all tiles share one accumulator (two of U = 2) and each lane has its own
    // slots' alone
    __device__ __forceinline__ void scores(v4f (&s)[S], const Keys& x, const v8h* qs, const int (&at)[U]) const {
        v8h k[2][4];
        auto make = [&](int dc) {
#pragma unroll
            for (int st = 0; st < 4; ++st) {
                const uint32_t w = word(x.u[(dc >> 1) * 2 + (st >> 1)], (st & 1) * 2 + (dc & 1));
                const uint32_t bits = in_sgpr(0x00F000F0u);
                k[dc & 1][st] = __builtin_bit_cast(v8h, uint4{w << 4 & bits, w & bits, w >> 4 & bits, w >> 8 & bits});
            }
        };
        make(0);
#pragma unroll
        for (int dc = 0; dc < NB; ++dc) {
            if (dc + 1 < NB) make(dc + 1);
            v4f acc[S];
#pragma unroll
            for (int a = 0; a < S; ++a) acc[a] = v4f{bias[dc], bias[dc], bias[dc], bias[dc]};
#pragma unroll
            for (int hl = 1; hl >= 0; --hl)
#pragma unroll
                for (int st = 0; st < 4; ++st)
                    acc[st / U] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                        k[dc & 1][st], qs[(dc * 2 + hl) * 4 * QROWS + at[st % U]], acc[st / U], 0, 0, 0);
#pragma unroll
            for (int a = 0; a < S; ++a)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float c = (float)((x.c[dc][a] >> (8 * i)) & 255);
                    s[a][i] = dc ? __builtin_fmaf(acc[a][i], c, s[a][i]) : acc[a][i] * c;
                }
        }
#pragma unroll
        for (int a = 0; a < S; ++a) s[a] = s[a] * (1.f / NIBBLE) * x.s[a];
    }

    __device__ __forceinline__ void raise(int en) {
        const float f = ldexpf(1.f, max(ev - en, -126));
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) o[dt] *= f;
        ev = en;
    }

    // the page's weights (as WaveAttn's soften) and their outputs
    __device__ __forceinline__ void take(v4f (&s)[S], Vals& x, bool whole, uint64_t sight, int u, int kq) {
        if (!whole) {
            const uint64_t seen = sight >> (4 * kq);
#pragma unroll
            for (int a = 0; a < S; ++a)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (!((seen >> (16 * (U * a + u) + i)) & 1)) {
                        s[a][i] = -INFINITY;
                        x.s[a][i] = 0.f;
                    }
        }
        l += lp;
        // (`maximum`, which hands NaN on, as in WaveAttn)
        float mx = __builtin_elementwise_maximum(__builtin_elementwise_maximum(s[0][0], s[0][1]),
                                                 __builtin_elementwise_maximum(s[0][2], s[0][3]));
        float top = fmaxf(fmaxf(x.s[0][0], x.s[0][1]), fmaxf(x.s[0][2], x.s[0][3]));
        if constexpr (S == 2) {
            mx = __builtin_elementwise_maximum(
                mx, __builtin_elementwise_maximum(__builtin_elementwise_maximum(s[1][0], s[1][1]),
                                                  __builtin_elementwise_maximum(s[1][2], s[1][3])));
            top = fmaxf(top, fmaxf(fmaxf(x.s[1][0], x.s[1][1]), fmaxf(x.s[1][2], x.s[1][3])));
        }
        mx = row_top(mx);
        const bool over = __builtin_fmaf(mx, c2, -off) > 15.f;
        if (__builtin_amdgcn_ballot_w64(over)) {
            float cand = __builtin_fmaf(mx, c2, -12.f);
            if (__builtin_fmaf(mx, c2, -cand) > 15.f) cand = mx * c2;
            if (cand > FLT_BIG) cand = __builtin_nanf("");
            const float on = over ? cand : off;
            const float al = off == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(off - on);
            off = on;
            l *= al;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) o[dt] *= al;
        }
        const float on = off == -INFINITY ? 0.f : off;
        if (__builtin_amdgcn_ballot_w64(top > ldexpf(1.f, ev))) raise(max(ev, ev_level(row_top(fmaxf(top, 0.f)))));
        const float f = ldexpf(1.f, -ev - 8);
        lp = 0.f;
        v4f w[S];
#pragma unroll
        for (int a = 0; a < S; ++a)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[a][i], c2, -on));
                lp += p;
                w[a][i] = p * (x.s[a][i] * f);
            }
#pragma unroll
        for (int j = 0; j < J; ++j) {
            v8h ph[2], pl[2];
            auto tile = [&](auto st_) {
                constexpr int st = decltype(st_)::value;
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    v2h h, lo;
                    split_hl2(rounded(of_lane<U, st>(w[st / U][i]) * mult(x.c[j], st, i)),
                              rounded(of_lane<U, st>(w[st / U][i + 1]) * mult(x.c[j], st, i + 1)), h, lo);
                    const int at = 4 * (st & 1) + i;
                    ph[st >> 1][at] = h[0];
                    ph[st >> 1][at + 1] = h[1];
                    pl[st >> 1][at] = lo[0];
                    pl[st >> 1][at + 1] = lo[1];
                }
            };
            tile(std::integral_constant<int, 0>{});
            tile(std::integral_constant<int, 1>{});
            tile(std::integral_constant<int, 2>{});
            tile(std::integral_constant<int, 3>{});
            // the dims of blocks U j .. U j + U - 1, two dim tiles each
            constexpr int N = NB < U ? NB : U;
            v8h v[2][2][2];  // [block's parity][dim tile][slots' half]
            auto make = [&](int g) {
#pragma unroll
                for (int sp = 0; sp < 2; ++sp) {
                    const uint32_t y = word(x.u[U * j + g], 2 * sp), z = word(x.u[U * j + g], 2 * sp + 1);
                    const uint32_t y8 = y >> 8, z8 = z >> 8;
                    v[g & 1][0][sp] = join(q4_low(y), q4_low(y8), q4_low(z), q4_low(z8));
                    v[g & 1][1][sp] = join(q4_high(y), q4_high(y8), q4_high(z), q4_high(z8));
                }
            };
            make(0);
#pragma unroll
            for (int g = 0; g < N; ++g) {
                if (g + 1 < N) make(g + 1);
                v4f* const d = o + 2 * (U * j + g);
#pragma unroll
                for (int sp = 0; sp < 2; ++sp) {
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        d[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[g & 1][e][sp], pl[sp], d[e], 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        d[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[g & 1][e][sp], ph[sp], d[e], 0, 0, 0);
                }
                if (g + 1 < N) beside();
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }

    // the lane's own outputs: own[2 j + e], dim tile 2 (U j + u) + e
    __device__ __forceinline__ void pick(v4f (&own)[OWN], int u) const {
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                own[2 * j + e] = o[2 * U * j + e];
#pragma unroll
                for (int x = 1; x < U && U * j + x < NB; ++x)
                    if (u == x) own[2 * j + e] = o[2 * (U * j + x) + e];
            }
    }
};

// As k_paged_attn, at most 16 / U query rows a sequence
template <int HD, int U, int NW>
__global__ void __launch_bounds__(64 * NW, 2) k_paged_fold(PagedAttn a) {
    using W = FoldAttn<HD, U>;
    __shared__ v4f so[NW - 1][W::OWN][64];
    __shared__ float sm[NW][64], sl[NW][64];
    __shared__ int se[NW][64];
    __shared__ typename W::Query qs;
    const int kvh = blockIdx.x % a.p.n_kv;
    const PagedItem it = a.items[blockIdx.x / a.p.n_kv];
    const PagedSeq sq = it.q;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, u = lane & (U - 1), rr = (lane & 15) / U, kq = lane >> 4;
    const int R = sq.M * a.gqa, r = min(rr, R - 1), t = r / a.gqa;
    const int64_t tok = sq.tok0 + t;
    const int head = kvh * a.gqa + r % a.gqa;
    // the pages of the wave, as in k_paged_attn
    const int n = max(0, (it.i1 - it.i0 - w + NW - 1) / NW);
    auto place = [&](int j) {
        const int i = it.i0 + w + NW * j;
        return i < it.s ? i : it.a + (i - it.s);
    };
    int ids = lane < n ? a.p.table[sq.tab0 + place(lane)] : 0;
    auto block_of = [&](int j) {
        if ((j & 63) == 0 && j) ids = j + lane < n ? a.p.table[sq.tab0 + place(j + lane)] : 0;
        return page_block(a.p, __builtin_amdgcn_readlane(ids, j & 63), kvh);
    };
    if (it.seq < 0) return;
    W wa;
    wa.query(a.q + tok * a.ldq + (int64_t)head * HD, u, rr, kq, !(((uintptr_t)a.q | (uintptr_t)(a.ldq * 4)) & 15), w == 0, qs);
    int at[U];  // slot tile st's query: the lane's row, or zeros
#pragma unroll
    for (int x = 0; x < U; ++x) at[x] = kq * W::QROWS + rr + (x == u ? 0 : W::QZ);
    __syncthreads();
    const RowSight sight(a, sq, t);
    int hi = sight.hi, lo = sight.lo;
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) {
        hi = min(hi, __shfl_xor(hi, x, 64));
        lo = max(lo, __shfl_xor(lo, x, 64));
    }
    hi = __builtin_amdgcn_readfirstlane(hi);
    lo = __builtin_amdgcn_readfirstlane(lo);
    typename W::Keys kv;
    typename W::Vals vv;
    const uint8_t* blk = nullptr;
    if (n) {
        blk = block_of(0);
        W::load(kv, blk, u, kq, lane);
    }
    for (int j = 0; j < n; ++j) {
        W::load(vv, blk, u, kq, lane);
        __builtin_amdgcn_sched_barrier(0);
        v4f s[W::S];
        asm volatile("" ::: "memory");  // (the query is read again for every page)
        wa.scores(s, kv, qs, at);
        __builtin_amdgcn_sched_barrier(0);
        const int p0 = place(j) * FTX_PAGE;
        if (j + 1 < n) {
            blk = block_of(j + 1);
            W::load(kv, blk, u, kq, lane);
        }
        __builtin_amdgcn_sched_barrier(0);
        const bool whole = p0 + FTX_PAGE - 1 <= hi && (p0 >= lo || p0 + FTX_PAGE <= a.sinks);
        wa.take(s, vv, whole, whole ? 0 : sight.page(p0), u, kq);
    }
    wa.l += wa.lp;
    wa.l += across<1>(wa.l);
    if constexpr (U == 4) wa.l += across<2>(wa.l);
    wa.l += __shfl_xor(wa.l, 16, 64);
    wa.l += __shfl_xor(wa.l, 32, 64);
    v4f own[W::OWN];
    wa.pick(own, u);
    sm[w][lane] = wa.off;
    sl[w][lane] = wa.l;
    se[w][lane] = wa.ev;
    if (w)
#pragma unroll
        for (int x = 0; x < W::OWN; ++x) so[w - 1][x][lane] = own[x];
    __syncthreads();
    if (w) return;
    float M = wa.off, f[NW], L = 0.f;
    int EV = wa.ev;
#pragma unroll
    for (int x = 1; x < NW; ++x) {
        M = fmaxf(M, sm[x][lane]);
        EV = max(EV, se[x][lane]);
    }
#pragma unroll
    for (int x = 0; x < NW; ++x) {
        const float mx = sm[x][lane];
        f[x] = mx == M ? 1.f : __builtin_amdgcn_exp2f(mx - M);
        L += f[x] * sl[x][lane];
        f[x] = ldexpf(f[x], se[x][lane] - EV);
    }
    if (rr >= R || u >= W::NB) return;
    const bool part = it.part >= 0;
    const int64_t prow = ((int64_t)it.part * a.p.n_kv + kvh) * PAGED_TR + rr;
    float* dst = part ? a.part + prow * HD : a.out + tok * a.ldo + (int64_t)head * HD;
    const bool vec = part || !(((uintptr_t)a.out | (uintptr_t)(a.ldo * 4)) & 15);
    const float inv = part && L == 0.f ? 0.f : 1.f / L;  // (as in k_paged_attn)
#pragma unroll
    for (int x = 0; x < W::OWN; ++x) {
        v4f y = own[x] * f[0];
#pragma unroll
        for (int z = 1; z < NW; ++z) y += so[z - 1][x][lane] * f[z];
#pragma unroll
        for (int z = 0; z < 4; ++z) y[z] = ldexpf(y[z] * inv, EV + 8);
        st4(dst + 32 * (U * (x >> 1) + u) + 16 * (x & 1) + 4 * kq, y, vec);
    }
    if (part && kq == 0 && u == 0) {
        a.pml[2 * prow] = M;
        a.pml[2 * prow + 1] = L;
    }
}

typedef __attribute__((address_space(3))) void lds_void;

// Many rows: workgroup = (item of 128 or 256 rows, kv head), eight waves of one
// or two tiles of 16 rows, the low halves of the queries in LDS (but for heads
// of 256 dims, where LDS holds the pages alone and a wave has one tile).
// Each page goes to LDS as the halves that the operands are (8- and 4-bit values
// converted once, by all waves, these under their multipliers), one page ahead in the
// other buffer: halves by direct copies, the others through registers, their loads
// issued before the current page's work and written after it.
// Bound by the SIMDs' issue: queries and weights in two halves make it two
// products of 16x16x32 for each of the formula's, 16 cycles each; three chunks
// of 1500 tokens after 1600 to 4000 (8-bit, 128 dims) take 467 us call after
// call, the CUs busy for 88% of it, in that time products for 48% and other
// vector instructions for 45% of the SIMDs' cycles (a wave's products run beside
// another's vector instructions in part); 4 bits 513, for whose conversion it issues
// 7% more vector instructions and twice the loads.  On the lower clock of a trace, where
// the kernel takes 539 and took 557: one tile a wave reads twice the
// LDS for a product: 656 us, LDS as busy as the products.  Tried and slower:
// both tiles' low halves in registers (73 spilled, 680), the waves' halves kept
// in antiphase, scores beside softmax (690), 64 rows a workgroup (686).
template <int HD>
constexpr int many_buf_bytes() {
    return 2 * FTX_PAGE * HD * 2 + 3 * FTX_PAGE * 4 + 16;  // values, scales of K, V, V by level, its level
}
constexpr int NW_MANY = PAGED_TR_MANY / PAGED_TR;
template <int HD>
constexpr int many_tiles() {
    return HD <= 128 ? 2 : 1;
}
template <int HD>
constexpr int many_lo_bytes() {
    return HD <= 128 ? many_tiles<HD>() * PAGED_TR_MANY * HD * 2 : 0;
}
template <int HD, int KT>
__global__ void __launch_bounds__(64 * NW_MANY) k_paged_many(PagedAttn a) {
    constexpr int NW = NW_MANY, NT = many_tiles<HD>();
    constexpr bool QLO = many_lo_bytes<HD>() > 0;
    using W = WaveAttn<HD, KT>;
    constexpr bool Q8 = W::Q8;
    constexpr int VB = FTX_PAGE * HD * 2;  // bytes of K's (V's) halves in LDS
    constexpr int BUF = many_buf_bytes<HD>();
    constexpr int NC = 2 * VB / 1024;  // KB of both
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int kvh = blockIdx.x % a.p.n_kv;
    const PagedItem it = a.items[a.n_few + blockIdx.x / a.p.n_kv];
    const PagedSeq sq = it.q;
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63, col = lane & 15, kq = lane >> 4;
    const int R = sq.M * a.gqa;
    const int nt = NT == 1 ? 1 : it.nt;  // the wave's tiles
    auto tile_of = [&](int x) { return w * nt + x; };
    auto row_of = [&](int x) { return it.row0 + 16 * tile_of(x) + col; };
    const bool live = it.row0 + 16 * tile_of(0) < R;  // (wave-uniform)
    const bool vecq = !(((uintptr_t)a.q | (uintptr_t)(a.ldq * 4)) & 15);
    const int n = it.i1 - it.i0;
    auto place = [&](int j) {
        const int i = it.i0 + j;
        return i < it.s ? i : it.a + (i - it.s);
    };
    int ids = lane < n ? a.p.table[sq.tab0 + place(lane)] : 0;
    auto block_of = [&](int j) {
        if ((j & 63) == 0 && j) ids = j + lane < n ? a.p.table[sq.tab0 + place(j + lane)] : 0;
        return page_block(a.p, __builtin_amdgcn_readlane(ids, j & 63), kvh);
    };
    // the thread's share of the next page
    constexpr int64_t PB = 2 * paged_values_bytes(HD, KT);  // bytes of K's and V's values in the page
    constexpr int NQ = Q8 ? (PB / 16 + 64 * NW - 1) / (64 * NW) : 1;  // 16-byte units of 8- or 4-bit values
    constexpr int UK = PB / 32;                                       // of K
    uint4 u[NQ], um[KT == PT_Q4 ? NQ : 1];
    float sc1 = 0.f;
    auto stage = [&](int j) {
        const uint8_t* blk = block_of(j);
        uint8_t* dst = lds + (j & 1) * BUF;
        if (tid < 2 * FTX_PAGE) sc1 = ((const float*)(blk + PB))[tid];
        if constexpr (KT == PT_Q4) {
#pragma unroll
            for (int i = 0; i < NQ; ++i) {
                const int x = i * 64 * NW + tid;
                if (x >= 2 * UK) break;  // (heads of 64 dims: half of the threads)
                u[i] = ((const uint4*)blk)[x];
                const uint8_t* mult = blk + PB + 2 * FTX_PAGE * 4;
                // K: the lane's four multipliers of two slots and blocks; V: those of its 16 slots
                if (x < UK) {
                    const uint8_t* t = mult + (x >> 7) * 128 + ((x >> 2) & 3) * 16 + (x >> 6 & 1) * 8 + (x & 3);
                    um[i] = uint4{t[0], t[64], t[4], t[68]};
                } else {
                    um[i] = *(const uint4*)(mult + paged_mult_bytes(HD, KT) + ((x - UK) >> 6) * 64 + ((x >> 4) & 3) * 16);
                }
            }
        } else if constexpr (Q8) {
#pragma unroll
            for (int i = 0; i < NQ; ++i) u[i] = ((const uint4*)blk)[i * 64 * NW + tid];
        } else {
#pragma unroll
            for (int i = 0; i < NC / NW; ++i)
                __builtin_amdgcn_global_load_lds((const void*)(blk + ((i * NW + w) * 64 + lane) * 16),
                                                 (lds_void*)(dst + (i * NW + w) * 1024), 16, 0, 0);
        }
    };
    auto commit = [&](int j) {
        uint8_t* dst = lds + (j & 1) * BUF;
        if (tid < 2 * FTX_PAGE) ((float*)(dst + 2 * VB))[tid] = sc1;
        if (w == 1) {
            // the page's V level (or that it has none: rows of both kinds) and its V scales by it
            const int pe = ev_level(__builtin_bit_cast(float, group_max<64>(mag(sc1 <= FLT_BIG ? sc1 : 0.f))));
            ((float*)(dst + 2 * VB))[FTX_PAGE + tid] = ldexpf(sc1, -pe);
            const bool both = !Q8 && both_kinds(sc1);
            if (lane == 0) *(int*)(dst + 2 * VB + 3 * FTX_PAGE * 4) = both ? W::NO_LEVEL : pe;
        }
        if constexpr (KT == PT_Q4) {
#pragma unroll
            for (int i = 0; i < NQ; ++i) {
                const int x = i * 64 * NW + tid, l = x & 63;
                if (x >= 2 * UK) break;
                if (x < UK) {
                    // words: slot tile 2 sh + (w >> 1), dims 32 (2 dh + (w & 1)) ..
                    const int sh = (x >> 6) & 1, dh = x >> 7;
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const _Float16 h = (_Float16)(float)W::word(um[i], y);
                        ((v8h*)dst)[((2 * dh + (y & 1)) * 4 + 2 * sh + (y >> 1)) * 64 + l] =
                            q4x8(W::word(u[i], y), v8h{h, h, h, h, h, h, h, h});
                    }
                } else {
                    v8h* t = (v8h*)(dst + VB) + ((x - UK) >> 6) * 256 + l;
#pragma unroll
                    for (int y = 0; y < 4; ++y)  // dim tile 2 g + (y >> 1), slots' half y & 1
                        t[y * 64] = q4x4x2(W::word(u[i], 2 * (y & 1)), W::word(u[i], 2 * (y & 1) + 1), y >> 1,
                                           W::word(um[i], 2 * (y & 1)), W::word(um[i], 2 * (y & 1) + 1));
                }
            }
        } else if constexpr (Q8) {
#pragma unroll
            for (int i = 0; i < NQ; ++i) {
                // unit x of K: dims' half (dc) and slot tile; of V: dim tile
                const int x = i * 64 * NW + tid, g = x >> 6;
                v8h* t;
                int step;
                if (g < HD / 16) {
                    t = (v8h*)dst + ((g >> 2) * 8 + (g & 3)) * 64 + (x & 63);
                    step = 4 * 64;
                } else {
                    t = (v8h*)(dst + VB) + (g - HD / 16) * 128 + (x & 63);
                    step = 64;
                }
                t[0] = u8x8(u[i].x, u[i].y);
                t[step] = u8x8(u[i].z, u[i].w);
            }
        }
    };
    if (it.seq < 0) return;  // (before the first copy to LDS)
    stage(0);
    W wa[NT];
    v8h* const qlo = (v8h*)(lds + 2 * BUF) + (QLO ? w * (NT * W::NDC * 64) + lane : 0);
    // the pages that every row of a tile sees whole, and the last that any row sees
    int hi[NT], lo[NT], last = 0;
#pragma unroll
    for (int x = 0; x < NT; ++x) {
        if (x >= nt) break;
        const int r = min(row_of(x), R - 1), t = r / a.gqa;
        wa[x].query(a.q + (int64_t)(sq.tok0 + t) * a.ldq + (int64_t)(kvh * a.gqa + r % a.gqa) * HD, kq, vecq);
        if constexpr (QLO)
#pragma unroll
            for (int dc = 0; dc < W::NDC; ++dc) qlo[(x * W::NDC + dc) * 64] = wa[x].ql[dc];
        const RowSight sight(a, sq, t);
        int h = sight.hi, l = sight.lo, e = sight.anc ? sq.npast + t : sight.hi;
#pragma unroll
        for (int y = 1; y < 16; y <<= 1) {
            h = min(h, __shfl_xor(h, y, 64));
            l = max(l, __shfl_xor(l, y, 64));
            e = max(e, __shfl_xor(e, y, 64));
        }
        hi[x] = __builtin_amdgcn_readfirstlane(h);
        lo[x] = __builtin_amdgcn_readfirstlane(l);
        last = max(last, __builtin_amdgcn_readfirstlane(e));
    }
    // page j for the wave's first N tiles; whether it takes a second visit
    auto work = [&](auto tiles, int j, bool second) -> bool {
        constexpr int N = decltype(tiles)::value;
        const int p0 = place(j) * FTX_PAGE;
        const uint8_t* buf = lds + (j & 1) * BUF;
        const float* scale = (const float*)(buf + 2 * VB);
        const bool ones = !Q8 && !__builtin_amdgcn_ballot_w64((scale[lane] != 1.f) | (scale[FTX_PAGE + lane] != 1.f));
        v4f s[N][4];
        staged_scores<W::NDC>(
            s, [&](int st, int dc) { return *(const v8h*)(buf + ((dc * 4 + st) * 64 + lane) * 16); },
            [&](int x, int dc) { return QLO ? qlo[(x * W::NDC + dc) * 64] : wa[x].ql[dc]; },
            [&](int x, int dc) { return wa[x].qh[dc]; });
        v8h ph[N][2], pl[N][2];
        typename W::Scales sc;
        int lev = 0;
        Kind kind = ALL;
        if (!ones) {
            W::load_four(sc.k, scale, kq);
            lev = __builtin_amdgcn_readfirstlane(*(const int*)(scale + 3 * FTX_PAGE));
            if (!Q8 && lev == W::NO_LEVEL) kind = second ? SMALL : LARGE;
#pragma unroll
            for (int x = 0; x < N; ++x) W::by_scale(s[x], sc);
        }
        auto vf = [&](int dt, int sp) { return *(const v8h*)(buf + VB + ((dt * 2 + sp) * 64 + lane) * 16); };
#pragma unroll
        for (int x = 0; x < N; ++x) {
            const bool whole = p0 + FTX_PAGE - 1 <= hi[x] && (p0 >= lo[x] || p0 + FTX_PAGE <= a.sinks);
            const bool leveled = whole && (Q8 || kind == ALL);
            if (!ones) W::load_four(sc.v, scale + (leveled ? 2 : 1) * FTX_PAGE, kq);
            const int pe = leveled ? lev : W::NO_LEVEL;
            uint64_t sight = 0;
            if (!whole) sight = RowSight(a, sq, min(row_of(x), R - 1) / a.gqa).page(p0);
            wa[x].soften(s[x], sc, ones, whole, pe, kind, sight, kq, ph[x], pl[x]);
        }
        staged_outputs<N>(wa, vf, ph, pl);
        return !Q8 && kind == LARGE;
    };
    commit(0);
    auto pages = [&](auto tiles) {
        for (int j = 0; j < n; ++j) {
            __builtin_amdgcn_s_waitcnt(0x0F70);  // this wave's direct copies of page j
            __syncthreads();                     // every wave's; the other buffer is free
            if (j + 1 < n) stage(j + 1);
            if (live && place(j) * FTX_PAGE <= last) {
#pragma clang loop unroll(disable)
                for (bool second = false; work(tiles, j, second);) second = true;
            }
            if (j + 1 < n) commit(j + 1);
        }
    };
    if constexpr (NT == 1)
        pages(std::integral_constant<int, 1>{});
    else if (nt == 2)  // (of every wave alike)
        pages(std::integral_constant<int, 2>{});
    else
        pages(std::integral_constant<int, 1>{});
    const bool part = it.part >= 0, vec = part || !(((uintptr_t)a.out | (uintptr_t)(a.ldo * 4)) & 15);
#pragma unroll
    for (int x = 0; x < NT; ++x) {
        if (x >= nt) return;
        wa[x].l += wa[x].lp;
        wa[x].l += __shfl_xor(wa[x].l, 16, 64);
        wa[x].l += __shfl_xor(wa[x].l, 32, 64);
        const int rr = row_of(x);
        if (rr >= R) return;
        const int64_t prow = ((int64_t)(it.part + tile_of(x)) * a.p.n_kv + kvh) * PAGED_TR + col;
        float* dst = part ? a.part + prow * HD
                          : a.out + (int64_t)(sq.tok0 + rr / a.gqa) * a.ldo + (int64_t)(kvh * a.gqa + rr % a.gqa) * HD;
        const float inv = part && wa[x].l == 0.f ? 0.f : 1.f / wa[x].l;  // (as in k_paged_attn)
#pragma unroll
        for (int dt = 0; dt < W::NDT; ++dt) {
            v4f y;
#pragma unroll
            for (int z = 0; z < 4; ++z) y[z] = ldexpf(wa[x].o[dt][z] * inv, wa[x].ev);
            st4(dst + 16 * dt + 4 * kq, y, vec);
        }
        if (part && kq == 0) {
            a.pml[2 * prow] = wa[x].off;
            a.pml[2 * prow + 1] = wa[x].l;
        }
    }
}

// out = sum_i 2^(m_i - M) l_i o_i / sum_i 2^(m_i - M) l_i of up to COMB_FEW
// partials: G rows a workgroup, HD / 4 threads each
constexpr int COMB_FEW = 8;
template <int HD>
__global__ void __launch_bounds__(256) k_paged_combine_few(PagedAttn a) {
    constexpr int D4 = HD / 4, G = 256 / D4;
    const int kvh = blockIdx.x % a.p.n_kv, d = threadIdx.x % D4;
    const int col = blockIdx.y * G + threadIdx.x / D4;
    const PagedComb c = a.combs[blockIdx.x / a.p.n_kv];
    const int rr = c.row0 + col;
    if (col >= PAGED_TR || rr >= c.M * a.gqa) return;
    const int64_t step = (int64_t)c.step * a.p.n_kv * PAGED_TR;
    const int64_t p0 = ((int64_t)c.part0 * a.p.n_kv + kvh) * PAGED_TR + col;
    const float2* ml = (const float2*)a.pml + p0;
    float2 t[COMB_FEW];
    v4f o[COMB_FEW];
#pragma unroll
    for (int i = 0; i < COMB_FEW; ++i) {
        const int64_t at = min(i, c.n - 1) * step;  // (past the last: its partial again, weight 0)
        t[i] = ml[at];
        o[i] = *(const v4f*)(a.part + (p0 + at) * HD + 4 * d);
    }
    float M = t[0].x, den = 0.f;
#pragma unroll
    for (int i = 1; i < COMB_FEW; ++i) M = fmaxf(M, t[i].x);
#pragma unroll
    for (int i = 0; i < COMB_FEW; ++i) {
        t[i].y *= i < c.n ? (t[i].x == M ? 1.f : __builtin_amdgcn_exp2f(t[i].x - M)) : 0.f;
        den += i < c.n ? t[i].y : 0.f;
    }
    v4f num = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < COMB_FEW; ++i)
        if (i < c.n) num += o[i] * (t[i].y / den);
    const int64_t tok = c.tok0 + rr / a.gqa;
    const bool vec = !(((uintptr_t)a.out | (uintptr_t)(a.ldo * 4)) & 15);
    st4(a.out + tok * a.ldo + (int64_t)(kvh * a.gqa + rr % a.gqa) * HD + 4 * d, num, vec);
}

// The same of any number: workgroup (row, kv head).  Every wave forms M and the
// sum itself; thread (g, d) adds the partials g, g + G, .. of dims
// 4 d .. 4 d + 3, the G sums meet in LDS.
template <int HD>
__global__ void __launch_bounds__(256) k_paged_combine(PagedAttn a) {
    constexpr int D4 = HD / 4, G = 256 / D4, PRE = 4;
    __shared__ v4f red[G][D4];
    const int kvh = blockIdx.x % a.p.n_kv, col = blockIdx.y;
    const PagedComb c = a.combs[blockIdx.x / a.p.n_kv];
    const int rr = c.row0 + col, lane = threadIdx.x & 63;
    if (rr >= c.M * a.gqa) return;
    const int64_t step = (int64_t)c.step * a.p.n_kv * PAGED_TR;
    const int64_t p0 = ((int64_t)c.part0 * a.p.n_kv + kvh) * PAGED_TR + col;
    const float2* ml = (const float2*)a.pml + p0;
    const int g = threadIdx.x / D4, d = threadIdx.x % D4;
    // the first partials of the thread, loaded beside the maxima and sums
    v4f first[PRE];
#pragma unroll
    for (int x = 0; x < PRE; ++x)
        first[x] = *(const v4f*)(a.part + (p0 + min(g + x * G, c.n - 1) * step) * HD + 4 * d);
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
    v4f num = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < PRE; ++x)
        if (g + x * G < c.n) num += first[x] * (weight(g + x * G) / den);
#pragma unroll 4
    for (int i = g + PRE * G; i < c.n; i += G) {
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
    const int64_t tok = c.tok0 + rr / a.gqa;
    const bool vec = !(((uintptr_t)a.out | (uintptr_t)(a.ldo * 4)) & 15);
    st4(a.out + tok * a.ldo + (int64_t)(kvh * a.gqa + rr % a.gqa) * HD + 4 * d, num, vec);
}

}  // namespace

// f<HD, KT> of the pool's head size and type
#define PAGED_TYPE(f, hd, kt) ((kt) == PT_Q4 ? f<hd, PT_Q4> : (kt) == PT_Q8 ? f<hd, PT_Q8> : f<hd, PT_F16>)
#define PAGED_CASE(f, hd, kt) \
    ((hd) == 64 ? PAGED_TYPE(f, 64, kt) : (hd) == 128 ? PAGED_TYPE(f, 128, kt) : PAGED_TYPE(f, 256, kt))

hipError_t launch_paged_write(hipStream_t st, const PagedView& p, int64_t max_new_pages, const float* k, int64_t ldk,
                              const float* v, int64_t ldv) {
    if (max_new_pages == 0) return hipSuccess;
    const dim3 grid((unsigned)((p.touch ? p.n_touch : max_new_pages) * 2 * p.n_kv), p.touch ? 1u : (unsigned)p.nseq);
    ktimed_launch(PAGED_CASE(k_paged_write, p.hd, p.kt), grid, dim3(256), 0, st, p, k, ldk, v, ldv);
    return hipGetLastError();
}

hipError_t launch_paged_read(hipStream_t st, const PagedView& p, int64_t max_pages, int context, float* k, int64_t ldk,
                             float* v, int64_t ldv) {
    if (max_pages == 0) return hipSuccess;
    const bool touch = p.touch && !context;
    const dim3 grid((unsigned)((touch ? p.n_touch : max_pages) * 2 * p.n_kv), touch ? 1u : (unsigned)p.nseq);
    ktimed_launch(PAGED_CASE(k_paged_read, p.hd, p.kt), grid, dim3(256), 0, st, p, context, k, ldk, v, ldv);
    return hipGetLastError();
}

template <int HD, int KT>
static hipError_t launch_many(hipStream_t st, const PagedAttn& a) {
    static std::atomic<uint64_t> lds_set{0};
    constexpr size_t bytes = 2 * (size_t)many_buf_bytes<HD>() + many_lo_bytes<HD>();
    const hipError_t e = lds_limit((const void*)k_paged_many<HD, KT>, bytes, lds_set);
    if (e != hipSuccess) return e;
    ktimed_launch(k_paged_many<HD, KT>, dim3((unsigned)a.n_many * (unsigned)a.p.n_kv), dim3(64 * NW_MANY),
                  (uint32_t)bytes, st, a);
    return hipGetLastError();
}

template <int HD, int KT>
static auto attn_four() {
    return k_paged_attn<HD, KT, 4>;
}
template <int HD, int KT>
static auto attn_wide() {
    return k_paged_attn<HD, KT, HD <= 128 ? 8 : 4>;
}

// of 4-bit rows and heads of 64 or 128 dims, by the most query rows of a sequence that
// has few (a chunk in the same step goes to the kernel of many)
typedef void (*paged_kernel)(PagedAttn);
template <int U, int NW>
static paged_kernel fold_hd(int hd) {
    return hd == 64 ? k_paged_fold<64, U, NW> : k_paged_fold<128, U, NW>;
}
static paged_kernel fold_of(int rows, int hd, bool wide) {
    if (rows <= 4) return wide ? fold_hd<4, 8>(hd) : fold_hd<4, 4>(hd);
    if (rows <= 8) return wide ? fold_hd<2, 8>(hd) : fold_hd<2, 4>(hd);
    return nullptr;
}

hipError_t launch_paged_attention(hipStream_t st, const PagedAttn& a) {
    hipError_t e = hipSuccess;
    if (a.n_many) e = PAGED_CASE(launch_many, a.p.hd, a.p.kt)(st, a);
    if (e != hipSuccess) return e;
    if (a.n_few) {
        const dim3 grid((unsigned)a.n_few * (unsigned)a.p.n_kv);
        auto* fold = a.p.kt != PT_Q4 || a.p.hd == 256 ? nullptr : fold_of(a.few_rows, a.p.hd, a.wide);
        if (fold)
            ktimed_launch(fold, grid, dim3(a.wide ? 512 : 256), 0, st, a);
        else if (a.wide)
            ktimed_launch(PAGED_CASE(attn_wide, a.p.hd, a.p.kt)(), grid, dim3(512), 0, st, a);
        else
            ktimed_launch(PAGED_CASE(attn_four, a.p.hd, a.p.kt)(), grid, dim3(256), 0, st, a);
    }
    e = hipGetLastError();
    if (e != hipSuccess || a.n_combs == 0) return e;
    const int rows = std::min(PAGED_TR, a.rows_max);
    const unsigned cx = (unsigned)a.n_combs * (unsigned)a.p.n_kv;
    if (a.comb_max <= COMB_FEW) {
        auto* f = a.p.hd == 64 ? k_paged_combine_few<64> : a.p.hd == 128 ? k_paged_combine_few<128> : k_paged_combine_few<256>;
        const int per = 256 / (a.p.hd / 4);
        hipLaunchKernelGGL(f, dim3(cx, (unsigned)((rows + per - 1) / per)), dim3(256), 0, st, a);
    } else {
        auto* f = a.p.hd == 64 ? k_paged_combine<64> : a.p.hd == 128 ? k_paged_combine<128> : k_paged_combine<256>;
        hipLaunchKernelGGL(f, dim3(cx, (unsigned)rows), dim3(256), 0, st, a);
    }
    return hipGetLastError();
}

hipError_t launch_paged_move(hipStream_t st, const PagedMove& m) {
    hipLaunchKernelGGL(k_paged_move, dim3((unsigned)m.n_kv, (unsigned)m.n_layer), dim3(256), 0, st, m);
    return hipGetLastError();
}
