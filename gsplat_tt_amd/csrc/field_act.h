// field_act.h - activations of the feature operators and their slopes, in fp32.
#pragma once

#include <hip/hip_runtime.h>

namespace gs {

enum { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3 };  // GS_ACT_*

// The normal distribution's Phi(z), and exp(-z^2 / 2) on the way: Phi(-|z|) =
// exp(-z^2 / 2) t P(t), t = 1 / (1 + 0.265 |z|). P is the polynomial of degree 8 with the
// least relative error over |z| <= 14, 1.2e-8, fitted to erfc (past 13.2 the exponential
// is 0 in fp32). What is left is rounding: the exponent's, z^2 2^-24, and a few units of
// the rest, so that the tail keeps its digits, as 1 + erf would not. The library's erff
// takes several times the instructions, which made the gelu passes bound by arithmetic.
__device__ __forceinline__ float normal_cdf(float z, float* pdf_exp) {
    const float e = __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);
    const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(z), 0.265f, 1.0f));
    float p = fmaf(t, 0.0308206789f, -0.144227788f);
    p = fmaf(t, p, 0.217813298f);
    p = fmaf(t, p, -0.116360791f);
    p = fmaf(t, p, 0.13795191f);
    p = fmaf(t, p, 0.0603135936f);
    p = fmaf(t, p, 0.102700867f);
    p = fmaf(t, p, 0.105246678f);
    p = fmaf(t, p, 0.10574156f);
    const float q = p * t * e;
    *pdf_exp = e;
    return z >= 0.0f ? 1.0f - q : q;
}
__device__ __forceinline__ float logistic(float z) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f));
}

template <int ACT>
__device__ __forceinline__ float act(float z) {
    if (ACT == kActRelu) return z > 0.0f ? z : (z != z ? z : 0.0f);
    if (ACT == kActSilu) return z * logistic(z);
    if (ACT == kActGelu) {
        float e;
        return z * normal_cdf(z, &e);
    }
    return z;
}
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
    if (ACT == kActRelu) return z > 0.0f ? 1.0f : 0.0f;
    if (ACT == kActSilu) {
        const float s = logistic(z);
        return s * fmaf(z, 1.0f - s, 1.0f);
    }
    if (ACT == kActGelu) {
        float e;
        const float c = normal_cdf(z, &e);
        return fmaf(z * 0.39894228040143268f, e, c);
    }
    return 1.0f;
}

}  // namespace gs
