// score_cap.cuh -- cap * tanh(s / cap) on the FMA pipe, shared by the attention kernels.
#pragma once
#include "sm100_ptx.cuh"

namespace ts {

// tanh(y) = y * q(y^2) on |y| <= 1: q of degree 5, fitted (numpy, iteratively reweighted least
// squares toward the minimax relative error), max relative error 6.9e-7 in fp32: a capped score of
// 50 is off by 3.5e-5, a hundredth of a bf16 rounding of its exponential.
constexpr float kTanhC0 = 0.9999994039535522f, kTanhC1 = -0.3332904279232025f, kTanhC2 = 0.13281433284282684f,
                kTanhC3 = -0.051605671644210815f, kTanhC4 = 0.016743112355470657f, kTanhC5 = -0.003067058976739645f;
constexpr float kTanhMaxSq = 1.0f;  // the fit's bound on y^2

// cap_out * q(w), q the tanh polynomial (w = y^2), for a pair.
__device__ __forceinline__ float2 tanh_poly(float2 w, float cap_out) {
    const auto k = [cap_out](float c) { const float v = c * cap_out; return make_float2(v, v); };
    float2 q = __ffma2_rn(k(kTanhC5), w, k(kTanhC4));
    q = __ffma2_rn(q, w, k(kTanhC3));
    q = __ffma2_rn(q, w, k(kTanhC2));
    q = __ffma2_rn(q, w, k(kTanhC1));
    return __ffma2_rn(q, w, k(kTanhC0));
}

// cap_out * tanh(y) for any y: the polynomial where it holds, else 1 - 2 / (1 + e^2y), whose
// subtraction loses nothing once |tanh(y)| > 0.76.
__device__ __forceinline__ float cap_exact(float y, float cap_out) {
    const float w = y * y;
    const float e = ex2(y * 2.8853900817779268f);
    const float outer = fmaf(-2.f * cap_out, __fdividef(1.f, 1.f + e), cap_out);
    return w <= kTanhMaxSq ? y * tanh_poly(make_float2(w, w), cap_out).x : outer;
}

}  // namespace ts
