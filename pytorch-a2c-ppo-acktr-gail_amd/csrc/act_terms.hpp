// Activations and their derivatives, shared by the epilogues of linear_act.hip.  All in fp32; exp and reciprocal are the
// hardware's base-2 exponential and reciprocal (1 ulp each), which leaves sigmoid, silu and tanh within ~4 ulp.
#pragma once
#include "common.hpp"
#include "../../include/acktr_hip.h"

namespace acktr {

constexpr float LOG2E = 1.44269504088896340736f;

__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }
__device__ __forceinline__ float fast_rcp(float x) { return __builtin_amdgcn_rcpf(x); }
// 1 / (1 + e^-x): e^-x overflows to infinity below x = -88, whose reciprocal is the right limit 0
__device__ __forceinline__ float sigmoid_f(float x) { return fast_rcp(1.f + fast_exp(-x)); }

// tanh: (1 - e^-2|x|) / (1 + e^-2|x|) with x's sign; near zero the difference cancels, there the series x - x^3/3 + 2x^5/15 - 17x^7/315
__device__ __forceinline__ float tanh_f(float x) {
    const float a = fabsf(x), e = fast_exp(-2.f * a);
    const float big = (1.f - e) * fast_rcp(1.f + e), q = x * x;
    const float small = a * (1.f + q * (-0.333333343f + q * (0.133333340f + q * -0.0539682545f)));
    return copysignf(a < 0.25f ? small : big, x);
}
// Complementary form of the normal distribution, 1 - Phi(|x|) = erfc(|x| / sqrt 2) / 2, by Abramowitz & Stegun 7.1.26: five terms in
// t = 1 / (1 + p |x| / sqrt 2), absolute error 7.5e-8 after the halving.  Forming the SMALL tail keeps gelu of large negative arguments
// relative to its own size.
__device__ __forceinline__ float normal_tail(float a, float e /* e^(-a*a/2) */) {
    const float t = fast_rcp(1.f + 0.23164189f * a);
    return 0.5f * e * t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
}

// y = act(z) and, with WANT, the slope act'(z); the two share their exponential
template <int ACT, bool WANT>
__device__ __forceinline__ float act_of(float z, float& slope) {
    if (ACT == ACKTR_ACT_RELU) {
        if (WANT) slope = z > 0.f ? 1.f : (z != z ? z : 0.f);
        return z > 0.f ? z : (z != z ? z : 0.f);
    }
    if (ACT == ACKTR_ACT_TANH) {
        if (WANT) {
            const float e = fast_exp(-2.f * fabsf(z)), r = fast_rcp(1.f + e);      // 1 / cosh^2, without 1 - tanh^2's cancellation
            slope = 4.f * e * r * r;
        }
        return tanh_f(z);
    }
    if (ACT == ACKTR_ACT_SILU) {
        const float s = sigmoid_f(z);
        if (WANT) slope = s * (1.f + z * (1.f - s));
        return z * s;
    }
    if (ACT == ACKTR_ACT_GELU) {
        const float a = fabsf(z), e = fast_exp(-0.5f * z * z), tail = normal_tail(a, e), cdf = z < 0.f ? tail : 1.f - tail;
        if (WANT) slope = cdf + z * e * 0.3989422804f;
        return z * cdf;
    }
    if (WANT) slope = 1.f;
    return z;
}

// What the backward pass keeps of an activation is its slope: fp32, or for 16-bit storage a fixed-point number with steps of 2^-14
// (slopes lie within (-0.13, 1.13)), which is off by 3e-5 at most.  The pre-activation itself, rounded to bf16, would put an error of
// up to 2^-9 |z act''(z)| into every gradient, and the exponential would have to be formed again.
constexpr short SLOPE_NAN = -32768;
template <class T> struct SlopeOf { typedef short type; };
template <> struct SlopeOf<float> { typedef float type; };
__device__ __forceinline__ void put_slope(short& c, float s) { c = s != s ? SLOPE_NAN : (short)__float2int_rn(s * 16384.f); }
__device__ __forceinline__ void put_slope(float& c, float s) { c = s; }
__device__ __forceinline__ float get_slope(short c) { return c == SLOPE_NAN ? __uint_as_float(0x7fc00000u) : (float)c * (1.f / 16384.f); }
__device__ __forceinline__ float get_slope(float c) { return c; }

}  // namespace acktr
