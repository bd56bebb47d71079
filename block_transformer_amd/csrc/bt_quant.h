// The 8-bit quantiser that bt_quant_rows and the KV cache share (gfx950 only).
#pragma once

#include "bt_common.h"

namespace bt {

// Sum and maximum over the four lanes c, c + 16, c + 32, c + 48, in all of them: two lane swaps of gfx950, no LDS.
__device__ inline float max_over_groups(float x) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ inline float sum_over_groups(float x) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
// over all 64 lanes, the 16 of a row by DPP: ten instructions instead of six round trips through LDS
__device__ inline float sum64(float x) { return sum_over_groups(row16_sum_dpp(x)); }
__device__ inline float max64(float x) {
#define BT_MAX_DPP(ctrl) x = fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), ctrl, 0xf, 0xf, false)))
    BT_MAX_DPP(0x128);      // row_ror:8, row_ror:4, quad_perm [2,3,0,1], quad_perm [1,0,3,2]
    BT_MAX_DPP(0x124);
    BT_MAX_DPP(0x4e);
    BT_MAX_DPP(0xb1);
#undef BT_MAX_DPP
    return max_over_groups(x);
}

// s = fl32(amax / 127), code(x) = clamp(round_half_even(x / s), -127, 127) with the quotient taken exactly, without a division per
// value.
//   exact():  y = x * fl32(1 / s) is within 3 * 2^-24 |y| < 3e-5 of x / s, so with h = floor(y) + 1/2 the quotient lies in (h - 1, h + 1)
//             and the answer is one of h - 1/2, h + 1/2; which one is the sign of x / s - h, that is of e = x - h s, and a fused
//             multiply-add rounds that difference once: its sign, and whether it is zero (a tie: the even one), are exact.  1 / s would
//             leave the normal numbers for s < 2^-126 and e could be lost among subnormal ones: below 2^-60 both x and s are taken
//             times 2^64, which changes no quotient.
//   pack4():  four values at once.  x * fl32(1 / s) + 1.5 * 2^23, fused, leaves the code in the low byte of the sum's bits; only where the
//             product is within 1e-4 of the middle between two codes can that be the wrong one, and then exact() decides.  Four
//             instructions a value and one to pack.  Only for |x| <= amax and where `direct` says so.
struct Quantiser {
    float scale, s, inv, up;
    bool direct;
    __device__ inline explicit Quantiser(float amax) {
        scale = amax / 127.0f;
        direct = scale >= 0x1p-60f;
        up = direct ? 1.0f : 0x1p64f;
        s = scale * up;
        inv = s > 0.f ? 1.0f / s : 0.f;
    }
    // x finite or infinite (an infinity clamps); NaN gives 0
    __device__ inline int exact(float x) const {
        x *= up;
        const float y = fminf(fmaxf(x * inv, -127.0f), 127.0f);
        const float f = floorf(y);
        const float e = fmaf(-(f + 0.5f), s, x);
        float r = e > 0.f ? f + 1.0f : f;
        if (e == 0.f) r = rintf(f + 0.5f);
        r = fminf(fmaxf(r, -127.0f), 127.0f);
        return (x == x && inv != 0.f) ? (int)r : 0;
    }
    __device__ inline uint32_t pack4_exact(float a, float b, float c, float d) const {
        return (uint32_t)(exact(a) & 255) | (uint32_t)(exact(b) & 255) << 8 | (uint32_t)(exact(c) & 255) << 16 | (uint32_t)exact(d) << 24;
    }
    __device__ inline uint32_t pack4(float a, float b, float c, float d) const {
        constexpr float M = 12582912.f;
        const float x[4] = {a, b, c, d};
        uint32_t t[4];
        float off = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float v = fmaf(x[i], inv, M);
            t[i] = __float_as_uint(v);
            off = fmaxf(off, fabsf(fmaf(x[i], inv, M - v)));
        }
        if (off > 0.4999f) return pack4_exact(a, b, c, d);
        const uint32_t lo = __builtin_amdgcn_perm(t[1], t[0], 0x0c0c0400), hi = __builtin_amdgcn_perm(t[3], t[2], 0x04000c0c);
        return lo | hi;
    }
};

}  // namespace bt
