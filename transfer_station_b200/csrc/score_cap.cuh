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

// The scores of kernels with keys as the matrix rows, a lane's four at a time: keys g and g + 8 (elements 0, 1 and
// 2, 3), two query columns (elements 0, 2 and 1, 3), each column with its factor, reference, position.
__device__ __forceinline__ void cap_argument(float (&s)[4], const float (&fac)[2], float &far) {  // -> y, the largest y^2
#pragma unroll
    for (int h = 0; h < 4; h += 2) {
        const float2 y = __fmul2_rn(make_float2(s[h], s[h + 1]), make_float2(fac[0], fac[1]));
        s[h] = y.x, s[h + 1] = y.y;
        far = fmax3(far, y.x * y.x, y.y * y.y);
    }
}
__device__ __forceinline__ void cap_near(float (&s)[4], const float (&k)[5], const float (&ref)[2]) {
#pragma unroll
    for (int h = 0; h < 4; h += 2) {
        const float2 y = make_float2(s[h], s[h + 1]);
        const float2 z = __ffma2_rn(y, tanh_poly(__fmul2_rn(y, y), k), make_float2(-ref[0], -ref[1]));
        s[h] = z.x, s[h + 1] = z.y;
    }
}
// For a warp that holds a score past the polynomial's interval. The others' bits are cap_near's: whether a warp comes
// here may hang on a slot that no row sees, whose score is replaced later and whose content may be anything.
__device__ __forceinline__ void cap_any(float (&s)[4], const float (&k)[5], float cap_out, const float (&ref)[2]) {
    const float y[4] = {s[0], s[1], s[2], s[3]};
    cap_near(s, k, ref);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = cap_far(y[e], s[e], cap_out, -ref[e & 1]);
}
__device__ __forceinline__ void scale_less(float (&s)[4], const float (&fac)[2], const float (&ref)[2]) {
#pragma unroll
    for (int h = 0; h < 4; h += 2) {
        const float2 z = __ffma2_rn(make_float2(s[h], s[h + 1]), make_float2(fac[0], fac[1]), make_float2(-ref[0], -ref[1]));
        s[h] = z.x, s[h + 1] = z.y;
    }
}
// at: key g less the column's position; off: further keys on (exact sums: a context of 2^24 keys is past every use)
__device__ __forceinline__ void less_bias(float (&s)[4], float off, const float (&at)[2], const float (&near)[2],
                                          const float (&slope2)[2]) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
        s[e] = fmaf(-slope2[e & 1], fabsf(at[e & 1] + (off + 4.f * (e & 2))) - near[e & 1], s[e]);
}

}  // namespace ts
