// GELU of the 4-bit products, in fp32 with one special-function operation: x Phi(x) = max(x, 0) - z Phi(-z), z = |x|, and
// Phi(-z) = 2^P(z), P a polynomial fitted to log2 Phi(-z) (tests/gelu_fit.py: smallest largest error of z Phi(-z) on
// [0, 5.6], and from there to 14 a bound on both sides that has 2^P at 0 by the end, so that the tail vanishes).
// The few-row kernel and the tensor-core kernel use the same form for the same output.
//   fast, for fp16 and 4-bit output: degree 6, the fit off by at most 1.6e-7.
//   fine, for fp32 output: degree 10, 4.8e-9; with the roundings 1.9e-8 (root mean square over normal x; the erf form 2.5e-8),
//   and 2e-7 of the result for |x| <= 1. It costs 6 to 8% ([100000 x 512] x [512 x 2048] 157 -> 170 us).
// Of -Inf the result is 0, its limit. (x Phi(x) with erf gives NaN there; to have that takes one more operation per value,
// 6 to 9%: [100000 x 512] x [512 x 2048] fp16 122 -> 132 us.)
// (gemm_tc.cu's form takes two special-function operations: at 16 a clock and SM they alone make 345 us on [189809 x 1024] x
// [1024 x 4096]. Scalar instead of packed operations: 650 us there, against 587 then.)
#pragma once

#include <cuda_fp16.h>

#include "ptx.cuh"

namespace vb::mx4 {

template <class T> constexpr bool kFineGelu = sizeof(T) == 4;  // type of the output

template <bool FINE> __device__ __forceinline__ float2 gelu2(float2 x) {
    const float2 n = make_float2(fmaxf(-fabsf(x.x), -14.0f), fmaxf(-fabsf(x.y), -14.0f));
    // coefficients of n^i, i from 0
    constexpr float kFast[] = {-1.00000226f, 1.1511004f, -0.459087521f, 0.0529918112f, 0.00781395286f, 0.000689681154f, 2.41893795e-05f};
    constexpr float kFine[] = {-0.99999994f, 1.15110612f, -0.459203899f, 0.0524968468f, 0.00703849457f, 8.63318637e-05f,
                               -0.000230278238f, -5.91184435e-05f, -7.36460788e-06f, -4.60322411e-07f, -1.12841496e-08f};
    constexpr int kDegree = FINE ? 10 : 6;
    float2 p = make_float2(FINE ? kFine[10] : kFast[6], FINE ? kFine[10] : kFast[6]);
#pragma unroll
    for (int i = kDegree - 1; i >= 0; --i) {
        const float c = FINE ? kFine[i] : kFast[FINE ? 0 : i];
        p = __ffma2_rn(n, p, make_float2(c, c));
    }
    float2 r;
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r.x) : "f"(x.x));
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r.y) : "f"(x.y));
    return __ffma2_rn(n, make_float2(ptx::ex2f(p.x), ptx::ex2f(p.y)), r);
}

}  // namespace vb::mx4
