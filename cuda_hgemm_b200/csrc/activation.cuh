// The activations of a feed-forward layer and their slopes, in FP32, for epilogues and the pass that
// multiplies an output's gradient by the slope.
//
//   relu       max(z, 0)                              slope  z > 0
//   gelu       z Phi(z), Phi(z) = (1 + erf(z/sqrt 2))/2   slope  Phi(z) + z exp(-z^2/2)/sqrt(2 pi)
//   gelu_tanh  z s, s = 1/(1 + exp(-w)), w = 2 sqrt(2/pi) (z + 0.044715 z^3)   slope  s + z s (1-s) w'
//   silu       z s, s = 1/(1 + exp(-z))               slope  s + z s (1-s)
//
// (0.5 (1 + tanh(w/2)) is that s: one exponential and one division instead of a tanh.) A NaN stays a NaN.
// Where s (1-s) has underflown, z is held at a bound before it multiplies it, so that a large z gives the
// slope 0 or 1 and not 0 * infinity. The value at +infinity is +infinity; at -infinity relu gives 0, the others z * 0 = NaN.
#pragma once

#include <stdint.h>

namespace b200 {

// The values of B200_ACT_* in the public header.
enum ActKind : uint32_t {
    kActNone = 0,
    kActRelu = 1,
    kActGelu = 2,
    kActGeluTanh = 3,
    kActSilu = 4,
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kGeluTanhScale = 1.5957691216057308f;  // 2 sqrt(2/pi)
constexpr float kGeluTanhCubic = 0.044715f;

// 2^x by the hardware's approximation (relative error about 2^-22, 0 and infinity at the ends).
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// z held within [-bound, bound]; a NaN stays
__device__ __forceinline__ float held(float z, float bound) {
    return z > bound ? bound : (z < -bound ? -bound : z);
}

// 1 - Phi(|z|) and exp(-z^2/2). The tail is exp(-z^2/2) times a function that falls off like 1/|z|, and that function
// is a polynomial in t = 1/(1 + 0.3 |z|): the form of Abramowitz and Stegun, Handbook of Mathematical Functions, 7.1.26, with
// eight terms instead of five, whose coefficients minimise the largest RELATIVE error for |z| <= 13.2 (1.2e-7, found by linear
// programming in 64 bits; the five-term form is good to 1.5e-7 absolute, which at z = -3 is 5e-5 of gelu's value).
// In FP32 the result is off by at most 1e-6 relative plus six roundings of z^2/2 (the exponential's argument).
// No branch, and fewer instructions than erff, which the epilogue warps would feel.
__device__ __forceinline__ float normal_tail(float z, float *gauss) {
    const float t = __fdividef(1.f, fmaf(0.3f, fabsf(z), 1.f));
    float poly = fmaf(0.0360886529f, t, -0.158932984f);
    poly = fmaf(poly, t, 0.209345162f);
    poly = fmaf(poly, t, -0.0564490594f);
    poly = fmaf(poly, t, 0.130032122f);
    poly = fmaf(poly, t, 0.0994652063f);
    poly = fmaf(poly, t, 0.120826296f);
    poly = fmaf(poly, t, 0.119624548f);
    *gauss = exp2_approx(-0.5f * kLog2e * (z * z));
    return poly * t * *gauss;
}

// 1 / (1 + exp(-w)): the gate of silu (w = z) and of gelu_tanh. Each has its own arithmetic: silu as the other with
// the cubic's constant 0 would multiply an infinite z by that 0.
template <uint32_t KIND>
__device__ __forceinline__ float logistic_gate(float z) {
    float w = z;
    if (KIND == kActGeluTanh) w *= fmaf(kGeluTanhScale * kGeluTanhCubic * z, z, kGeluTanhScale);
    return __fdividef(1.f, 1.f + exp2_approx(-kLog2e * w));
}

template <uint32_t KIND>
__device__ __forceinline__ float act_value(float z) {
    if (KIND == kActRelu) return z < 0.f ? 0.f : z;
    if (KIND == kActGelu) {
        float gauss;
        const float tail = normal_tail(z, &gauss);
        return z * (z < 0.f ? tail : 1.f - tail);
    }
    if (KIND == kActGeluTanh || KIND == kActSilu) return z * logistic_gate<KIND>(z);
    return z;
}

template <uint32_t KIND>
__device__ __forceinline__ float act_slope(float z) {
    if (KIND == kActRelu) return z <= 0.f ? 0.f : 1.f;
    if (KIND == kActGelu) {
        const float h = held(z, 16.f);  // exp(-128): gone
        float gauss;
        const float tail = normal_tail(h, &gauss);
        return (h < 0.f ? tail : 1.f - tail) + h * 0.3989422804014327f * gauss;
    }
    if (KIND == kActGeluTanh) {
        const float h = held(z, 16.f);
        const float s = logistic_gate<KIND>(h);
        return s + h * s * (1.f - s) * kGeluTanhScale * fmaf(3.f * kGeluTanhCubic * h, h, 1.f);
    }
    if (KIND == kActSilu) {
        const float h = held(z, 88.f);  // exp(88) is still finite, and its reciprocal already 0 (__fdividef, above 2^126)
        const float s = logistic_gate<KIND>(h);
        return s + h * s * (1.f - s);
    }
    return 1.f;
}

// COUNT values (FP32 bit patterns) through one activation; the choice is made once, outside the loop.
template <int COUNT, uint32_t KIND>
__device__ __forceinline__ void act_apply_kind(uint32_t *vals) {
#pragma unroll
    for (int j = 0; j < COUNT; ++j) vals[j] = __float_as_uint(act_value<KIND>(__uint_as_float(vals[j])));
}

template <int COUNT>
__device__ __forceinline__ void act_apply(uint32_t *vals, uint32_t kind) {
    if (kind == kActGeluTanh) {
        act_apply_kind<COUNT, kActGeluTanh>(vals);
    } else if (kind == kActSilu) {
        act_apply_kind<COUNT, kActSilu>(vals);
    } else if (kind == kActGelu) {
        act_apply_kind<COUNT, kActGelu>(vals);
    } else if (kind == kActRelu) {
        act_apply_kind<COUNT, kActRelu>(vals);
    }
}

}  // namespace b200
