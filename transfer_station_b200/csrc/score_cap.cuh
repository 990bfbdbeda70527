// score_cap.cuh -- cap * tanh(s / cap) on the FMA pipe, shared by the attention kernels.
#pragma once
#include "sm100_ptx.cuh"

namespace ts {

// tanh(y) = y * q(y^2) on |y| <= 3/4: q of degree 4, fitted (numpy, iteratively reweighted least
// squares toward the minimax relative error), max relative error 6.9e-07 in fp32: a capped score of
// 50 is off by 3e-5, a hundredth of a bf16 rounding of its exponential. (Degree 5 reaches 1 as exactly;
// the FMA pipe is what bounds capped prompts, and scores past 3/4 of the cap are rare.)
constexpr float kTanhC[5] = {0.999999463558197f, -0.3332825005054474f, 0.13258983194828033f, -0.050056297332048416f,
                             0.012929629534482956f};
constexpr float kTanhMaxSq = 0.5625f;  // the fit's bound on y^2

// q(w) for a pair, with coefficients k: cap_out * kTanhC on w = y^2, or with the powers of cap_in folded
// in on the square of the raw score.
__device__ __forceinline__ float2 tanh_poly(float2 w, const float (&k)[5]) {
    float2 q = __ffma2_rn(make_float2(k[4], k[4]), w, make_float2(k[3], k[3]));
    q = __ffma2_rn(q, w, make_float2(k[2], k[2]));
    q = __ffma2_rn(q, w, make_float2(k[1], k[1]));
    return __ffma2_rn(q, w, make_float2(k[0], k[0]));
}

// cap_out * tanh(y) + add for any y, given the polynomial's value: outside its interval 1 - 2 / (1 + e^2y),
// whose subtraction loses nothing once |tanh(y)| > 0.63.
__device__ __forceinline__ float cap_far(float y, float inside, float cap_out, float add = 0.f) {
    const float e = ex2(y * 2.8853900817779268f);
    const float outer = fmaf(-2.f * cap_out, __fdividef(1.f, 1.f + e), cap_out) + add;
    return y * y > kTanhMaxSq ? outer : inside;
}

}  // namespace ts
