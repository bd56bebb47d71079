// The 8-bit quantiser that bt_quant_rows and the KV cache share (gfx950 only).
#pragma once

#include "bt_common.h"

namespace bt {

// s = fl32(amax / 127), code(x) = clamp(round_half_even(x / s), -127, 127) with the quotient taken exactly, without a division per
// value.  y = x * fl32(1 / s) is within 3 * 2^-24 |y| < 3e-5 of x / s, so with h = floor(y) + 1/2 the quotient lies in (h - 1, h + 1)
// and the answer is one of h - 1/2, h + 1/2; which one is the sign of x / s - h, that is of e = x - h s, and a fused multiply-add
// rounds that difference once: its sign, and whether it is zero (a tie: the even one), are exact.  1 / s would leave the normal numbers
// for s < 2^-126 and e could be lost among subnormal ones: below 2^-60 both x and s are taken times 2^64, which changes no quotient.
struct Quantiser {
    float scale, s, inv, up;
    __device__ inline explicit Quantiser(float amax) {
        scale = amax / 127.0f;
        up = scale < 0x1p-60f ? 0x1p64f : 1.0f;
        s = scale * up;
        inv = s > 0.f ? 1.0f / s : 0.f;
    }
    // x finite or infinite (an infinity clamps); NaN gives 0
    __device__ inline int code(float x) const {
        x *= up;
        const float y = fminf(fmaxf(x * inv, -127.0f), 127.0f);
        const float f = floorf(y);
        const float e = fmaf(-(f + 0.5f), s, x);
        float r = e > 0.f ? f + 1.0f : f;
        if (e == 0.f) r = rintf(f + 0.5f);
        r = fminf(fmaxf(r, -127.0f), 127.0f);
        return (x == x && inv != 0.f) ? (int)r : 0;
    }
};

}  // namespace bt
