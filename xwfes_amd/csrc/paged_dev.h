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

}  // namespace
