// GELU of the bf16 epilogues (gfx950 only).
#pragma once

#include "bt_common.h"

namespace bt {

// GELU for the bf16 MFMA epilogues.  erff costs ~45 VALU instructions per value (measured: a K = 2048 GEMM with GELU ran
// 33 % slower than without), so the bf16 path evaluates  gelu(x) = x * Phi(x)  through the scaled normal tail
//     Phi(-a) = exp(-a^2 / 2) * R(a),   a = |x|,   R = degree-11 polynomial in u = a/3 - 1 (relative minimax fit on [0, 6])
//     gelu(x) = x * Phi(-a)          (x < 0)        = x * (1 - Phi(-a))   (x >= 0)
// which keeps RELATIVE accuracy in the negative tail (no 1 + erf cancellation).  In fp32 arithmetic the result is within
// 8.5e-6 relative of the exact erf GELU for x > -6 (|gelu| < 6e-9 beyond, absolute error < 8e-9): 1/230 of a bf16
// half-ulp (a degree-12 fit has a polynomial error of 2.2e-6 instead of 7.7e-6, both beside ~3e-6 of fp32 evaluation noise -- on every
// bf16 input in [-9, 9] both round to the correctly rounded bf16 value; a degree-10 fit, 2.7e-5, would flip 0.03 % of them, degree 9 0.5 %).
// The fp32 parity path (gemm_generic_kernel) keeps erff.  Two values per call: two independent chains of FMAs, so neither waits for
// its own last step.
typedef float v2f __attribute__((ext_vector_type(2)));

// min(|x|, 6) and max(x, 0) as single instructions: the builtins (fminf / fmaxf / fabsf) make hipcc quiet a possible signalling NaN
// first -- a v_max_f32 x, x in front of every min / max -- and materialise |x| with a v_and.  Plain asm (not volatile: the scheduler
// may move it); 6.0 is not an inline constant of the VOP3 encoding -> one SGPR for the whole kernel.
__device__ inline float min_abs_f32(float x, float hi) {
    float r;
    asm("v_min_f32_e64 %0, |%1|, %2" : "=v"(r) : "v"(x), "s"(hi));
    return r;
}
__device__ inline float relu_f32(float x) {
    float r;
    asm("v_max_f32_e32 %0, 0, %1" : "=v"(r) : "v"(x));
    return r;
}

__device__ inline v2f gelu_tail2(v2f x) {
    const v2f a = {min_abs_f32(x.x, 6.0f), min_abs_f32(x.y, 6.0f)};
    const v2f u = a * (1.0f / 3.0f) - 1.0f;
    v2f r = u * -3.976902133e-03f + 8.081740986e-03f;
    r = r * u + -2.753396143e-03f;
    r = r * u + 1.759199353e-03f;
    r = r * u + -1.408788524e-02f;
    r = r * u + 2.432763856e-02f;
    r = r * u + -3.125067898e-02f;
    r = r * u + 4.423156669e-02f;
    r = r * u + -6.233500973e-02f;
    r = r * u + 8.247426398e-02f;
    r = r * u + -1.032048037e-01f;
    r = r * u + 1.215130848e-01f;
    const v2f t = x * x * -0.72134752044448170368f;     // -x^2 / 2 * log2(e)  (unclamped: exp2 underflows to 0 beyond |x| ~ 14)
    const v2f e = {__builtin_amdgcn_exp2f(t.x), __builtin_amdgcn_exp2f(t.y)};
    const v2f q = e * r;                                 // Phi(-|x|)
    // x * Phi(x) = relu(x) - |x| * Phi(-|x|): the same value as selecting q or 1 - q by sign and multiplying (identical for x < 0,
    // x - x q for x >= 0), in one FMA instead of two compares, two selects, a subtraction and a multiply.  The clamped |x| is
    // used for the product: identical bits for |x| <= 6, and beyond that the term is < 1e-8 either way (q < 2e-9)
    const v2f relu = {relu_f32(x.x), relu_f32(x.y)};
    return relu - a * q;
}

__device__ inline void gelu4(float (&v)[4]) {
    const v2f lo = gelu_tail2(v2f{v[0], v[1]}), hi = gelu_tail2(v2f{v[2], v[3]});
    v[0] = lo.x; v[1] = lo.y; v[2] = hi.x; v[3] = hi.y;
}

}  // namespace bt
