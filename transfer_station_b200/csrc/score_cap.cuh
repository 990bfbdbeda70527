// score_cap.cuh -- cap * tanh(s / cap) on the FMA pipe, shared by the attention kernels.
#pragma once
#include "sm100_ptx.cuh"

namespace ts {

// tanh(y) = y * q(y^2) on |y| <= 1: q of degree 5, fitted (numpy, iteratively reweighted least
// squares toward the minimax relative error), max relative error 6.9e-7 in fp32: a capped score of
// 50 is off by 3.5e-5, a hundredth of a bf16 rounding of its exponential.
constexpr float kTanhC[6] = {0.9999994039535522f, -0.3332904279232025f, 0.13281433284282684f,
                             -0.051605671644210815f, 0.016743112355470657f, -0.003067058976739645f};
constexpr float kTanhMaxSq = 1.0f;  // the fit's bound on y^2

// cap_out * q(w) for a pair, w = y^2; k = cap_out * kTanhC.
__device__ __forceinline__ float2 tanh_poly(float2 w, const float (&k)[6]) {
    float2 q = __ffma2_rn(make_float2(k[5], k[5]), w, make_float2(k[4], k[4]));
    q = __ffma2_rn(q, w, make_float2(k[3], k[3]));
    q = __ffma2_rn(q, w, make_float2(k[2], k[2]));
    q = __ffma2_rn(q, w, make_float2(k[1], k[1]));
    return __ffma2_rn(q, w, make_float2(k[0], k[0]));
}

// cap_out * tanh(y) for any y, given the polynomial's value: outside its interval 1 - 2 / (1 + e^2y),
// whose subtraction loses nothing once |tanh(y)| > 0.76.
__device__ __forceinline__ float cap_far(float y, float inside, float cap_out) {
    const float e = ex2(y * 2.8853900817779268f);
    const float outer = fmaf(-2.f * cap_out, __fdividef(1.f, 1.f + e), cap_out);
    return y * y > kTanhMaxSq ? outer : inside;
}

}  // namespace ts
