// Activations and their derivatives, shared by the epilogues of linear_act.hip, and the exponential they share with gated_scan.hip.  All
// in fp32; the hardware's base-2 exponential and reciprocal are off by an ulp each.
#pragma once
#include "common.hpp"
#include "../../include/acktr_hip.h"

namespace acktr {

constexpr float LOG2E = 1.44269504088896340736f;

__device__ __forceinline__ float fast_rcp(float x) { return __builtin_amdgcn_rcpf(x); }
// e^x.  The rounding of x log2(e) alone puts it off by |x| 6e-8, nothing beside the rounding of 16-bit storage.  ACC (fp32 storage, |x| at
// most 200): that rounding is carried along (`more`: what x itself lacks), which leaves 2 ulp.  e^x below 2^-126 is 0.
template <bool ACC>
__device__ __forceinline__ float exp_of(float x, float more = 0.f) {
    const float p = x * LOG2E;
    float e = __builtin_amdgcn_exp2f(p);
    if (ACC) {
        const float lo = fmaf(x, LOG2E, -p) + (x * 1.92596299e-8f + more * LOG2E);
        e = fmaf(e, lo * 0.693147182f, e);
    }
    return e;
}
// the magnitude that an exponent is formed of (minimum() keeps a NaN): beyond 100 sigmoid and tanh are at their limits
template <bool ACC>
__device__ __forceinline__ float magnitude(float x) { return ACC ? __builtin_elementwise_minimum(fabsf(x), 100.f) : fabsf(x); }

// s = 1 / (1 + e^-x) and ns = 1 - s, both within 5 ulp of their own size (down to 2^-126; 16-bit storage: 6e-8 |x| more)
template <bool ACC>
__device__ __forceinline__ void sigmoid_of(float x, float& s, float& ns) {
    const float e = exp_of<ACC>(-magnitude<ACC>(x)), big = fast_rcp(1.f + e), tail = e * big;
    s = x < 0.f ? tail : big;
    ns = x < 0.f ? big : tail;
}

// tanh: (1 - e^-2|x|) / (1 + e^-2|x|) with x's sign; near zero the difference cancels, there the series x - x^3/3 + 2x^5/15 - 17x^7/315.
// e: e^-2|x|, r: 1 / (1 + e).
__device__ __forceinline__ float tanh_f(float x, float e, float r) {
    const float a = fabsf(x), big = (1.f - e) * r, q = x * x;
    const float small = a * (1.f + q * (-0.333333343f + q * (0.133333340f + q * -0.0539682545f)));
    return copysignf(a < 0.25f ? small : big, x);
}
// Complementary form of the normal distribution, 1 - Phi(a) = e^(-a*a/2) t P(t) with t = 1 / (1 + 0.35 a), for 0 <= a: a polynomial of
// degree 8, fitted to the scaled complementary error function for the least relative error on [0, 13.5] (3e-8; beyond, the exponential
// is 0).  Formed of the SMALL tail, gelu of negative arguments is within 8 ulp of its own size wherever that is above 2^-118 (16-bit
// storage: 6e-8 z^2 more).
__device__ __forceinline__ float normal_tail(float a, float e /* e^(-a*a/2) */) {
    const float t = fast_rcp(fmaf(0.35f, a, 1.f));
    float q = -0.0291258693f;
    q = fmaf(q, t, 0.143872246f);
    q = fmaf(q, t, -0.255504608f);
    q = fmaf(q, t, 0.158929333f);
    q = fmaf(q, t, -0.0229371656f);
    q = fmaf(q, t, 0.10543295f);
    q = fmaf(q, t, 0.119852431f);
    q = fmaf(q, t, 0.13985908f);
    q = fmaf(q, t, 0.139621571f);
    return e * (t * q);
}

// y = act(z) and, with WANT, the slope act'(z); the two share their exponential
template <int ACT, bool WANT, bool ACC>
__device__ __forceinline__ float act_of(float z, float& slope) {
    if (ACT == ACKTR_ACT_RELU) {
        if (WANT) slope = z > 0.f ? 1.f : (z != z ? z : 0.f);
        return z > 0.f ? z : (z != z ? z : 0.f);
    }
    if (ACT == ACKTR_ACT_TANH) {
        const float e = exp_of<ACC>(-2.f * magnitude<ACC>(z)), r = fast_rcp(1.f + e);
        if (WANT) slope = 4.f * e * r * r;                                         // 1 / cosh^2, without 1 - tanh^2's cancellation
        return tanh_f(z, e, r);
    }
    if (ACT == ACKTR_ACT_SILU) {
        float s, ns;
        sigmoid_of<ACC>(z, s, ns);
        if (WANT) slope = s * (1.f + z * ns);
        return z * s;
    }
    if (ACT == ACKTR_ACT_GELU) {
        // held at 18, where the exponential is 0 already; ACC: z^2 / 2 with the rounding of z^2
        const float a = __builtin_elementwise_minimum(fabsf(z), 18.f), q = a * a;
        const float e = exp_of<ACC>(-0.5f * q, ACC ? -0.5f * fmaf(a, a, -q) : 0.f), tail = normal_tail(a, e), cdf = z < 0.f ? tail : 1.f - tail;
        if (WANT) slope = cdf + copysignf(a, z) * e * 0.3989422804f;
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
