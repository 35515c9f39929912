// paged_dev.h -- how a row of K or V is stored in its page (device code).
#pragma once

#include <type_traits>

#include "paged.h"

namespace {

constexpr float FLT_BIG = 3.402823466e38f;
// rows below this are stored as zeros
constexpr float ROW_TINY = 7.888609052210118e-31f;  // 2^-100

__device__ __forceinline__ uint8_t* page_block(const PagedView& p, int page, int kvh) {
    return p.data + ((int64_t)page * p.n_kv + kvh) * p.block;
}

// The largest of v over aligned groups of W lanes (8, 16, 32 or 64), in all of
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
    if constexpr (W > 8) step(std::integral_constant<int, 0x140>{});  // mirrored in 16
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

// |x| as an integer: ordered as the magnitudes are, infinity and NaN above all
__device__ __forceinline__ uint32_t mag(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu; }

// How a row of largest magnitude `amax` (mag) is stored (halves, 8 bits)
template <int KT>
struct RowForm {
    static constexpr bool Q8 = KT == PT_Q8;
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
        if (zero) return 0.f;  // (of no size: it must not set a level)
        if constexpr (Q8) return a / 127.f;
        return ldexpf(1.f, f16_exp(a));
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

// Rows of 4 bits: t(x) = max(x, 0) / 7 or max(-x, 0) / 8 (1/7: the float next to
// it) is the step that x needs, T the largest of a row.  A block of 32 dims takes
// steps of c s, s = T / 255 and c the integer that covers the block's largest t:
// within 1/255 of T of what it needs, so that a block of small values beside a
// large one keeps its precision, in one byte, and q c, at most 2040, is exact as
// a half.  Every operation is one IEEE rounding to fp32.
constexpr float Q4_TINY = 9.860761315262648e-32f;  // 2^-103: rows whose T is below are stored as zeros
__device__ __forceinline__ float q4_need(float x) { return x > 0.f ? x * (1.f / 7.f) : x * -0.125f; }
struct Q4Row {
    float s, up;
    bool ok, zero;
    // top: mag of the row's largest q4_need
    __device__ __forceinline__ explicit Q4Row(uint32_t top) {
        const float T = __builtin_bit_cast(float, top);
        ok = T <= FLT_BIG;
        zero = !ok || T < Q4_TINY;
        s = T / 255.f;
        up = 255.f / T;
    }
    __device__ __forceinline__ float scale() const { return !ok ? __builtin_nanf("") : zero ? 0.f : s; }
    // a block's multiplier from mag of its largest q4_need, and what its values are multiplied by
    __device__ __forceinline__ int mult(uint32_t t, float& r) const {
        const float c = zero ? 0.f : fminf(ceilf(__builtin_bit_cast(float, t) * up), 255.f);
        r = c > 0.f ? 1.f / (c * s) : 0.f;
        return (int)c;
    }
    // the nibble: q + 8
    __device__ __forceinline__ uint32_t bits(float x, float r) const {
        return (uint32_t)((int)rintf(ok ? x * r : 0.f) + 8);
    }
};

// A wave stores one row of HD values, at(d) the value of dim d, as slot `slot`'s
// K or V row of 4 bits in block blk
template <typename X>
__device__ __forceinline__ void q4_store_row(uint8_t* blk, int hd, int slot, bool isv, int lane, X at) {
    uint8_t* vals = blk + (isv ? paged_values_bytes(hd, PT_Q4) : 0);
    uint8_t* after = blk + 2 * paged_values_bytes(hd, PT_Q4);
    uint8_t* mult = after + 2 * FTX_PAGE * 4 + (isv ? paged_mult_bytes(hd, PT_Q4) : 0);
    const int n = hd / 2;  // bytes of the row: 32, 64 or 128, up to two a lane
    float x[2][2] = {};
    uint32_t t[2] = {};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int b = 64 * i + lane;
        if (b >= n) continue;
        const int d = isv ? paged_v_dim(b) : paged_k_dim(b);
        x[i][0] = at(d);
        x[i][1] = at(d + (isv ? 16 : 2));
        t[i] = max(mag(q4_need(x[i][0])), mag(q4_need(x[i][1])));
    }
    const Q4Row f(group_max<64>(max(t[0], t[1])));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int b = 64 * i + lane;
        const uint32_t bt = group_max<16>(t[i]);
        if (b >= n) continue;
        const int d = isv ? paged_v_dim(b) : paged_k_dim(b);
        float r;
        const int c = f.mult(bt, r);
        vals[isv ? paged_v_at(slot, d, PT_Q4) : paged_k_at(slot, d, PT_Q4)] =
            (uint8_t)(f.bits(x[i][0], r) | f.bits(x[i][1], r) << 4);
        if ((b & 15) == 0) mult[paged_c_at(slot, b >> 4)] = (uint8_t)c;
    }
    if (lane == 0) ((float*)after)[(isv ? FTX_PAGE : 0) + slot] = f.scale();
}

}  // namespace
