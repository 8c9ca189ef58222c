// Activations of linear layers and their slopes, in fp32.
#pragma once
#include "common.cuh"

namespace ascb200 {
namespace act {

__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_fast(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLog2e = 1.4426950408889634f;

// 1 / (1 + e^-x): one ex2, one rcp; an overflowing exponential gives the limit 0.
__device__ __forceinline__ float sigmoid(float x) { return rcp_fast(1.0f + exp2_fast(-kLog2e * x)); }

// GELU's tanh form is z * sigmoid(2 u), u = sqrt(2 / pi) (z + 0.044715 z^3).  Beyond |z| = 32 the sigmoid is 0 or 1 to the last bit;
// the clamp keeps z^3 and z^2 finite.
constexpr float kTanh2u = 1.5957691216057308f;  // 2 sqrt(2 / pi)
__device__ __forceinline__ float clamp_nan(float z, float top)  // a NaN stays
{
    float r;
    asm("{\n\t.reg .f32 t;\n\tmax.NaN.f32 t, %1, %2;\n\tmin.NaN.f32 %0, t, %3;\n\t}" : "=f"(r) : "f"(z), "f"(-top), "f"(top));
    return r;
}
__device__ __forceinline__ float tanh_arg(float z)
{
    const float c = clamp_nan(z, 32.0f);
    return kTanh2u * c * fmaf(0.044715f * c, c, 1.0f);
}

// Upper tail of the normal distribution at |z|, and e = e^(-z^2 / 2).  The tail is e * R with a smooth R, which is t P(t) in t = 1 / (1 + 0.21 |z|): P of degree
// eight, fitted to R / t for |z| up to 14 with the smallest relative error (1.6e-8).  A tail that is right relative to itself keeps GELU so where z is
// negative: within 6e-7 of itself to |z| = 3, 2e-6 to 6, 8e-6 to 13 (z^2 times its rounding in the exponent); an approximation of
// erf with an absolute error of 1.5e-7 was off by 5e-4 at -4 and 1e-2 at -8 (its four steps less took 100.4 us instead of 102.1 in the layer of 4096 x
// 11008 x 1024 bf16 with z).  Beyond 13.2 e is below the normal numbers and taken as 0.
__device__ __forceinline__ float normal_tail(float z, float& e)
{
    const float t = rcp_fast(fmaf(0.21f, fabsf(z), 1.0f));
    float p = fmaf(-0.07165637f, t, 0.28358883f);
    p = fmaf(p, t, -0.33025384f);
    p = fmaf(p, t, 0.3494015f);
    p = fmaf(p, t, -0.09392552f);
    p = fmaf(p, t, 0.12487286f);
    p = fmaf(p, t, 0.069192134f);
    p = fmaf(p, t, 0.08506887f);
    p = fmaf(p, t, 0.08371157f);
    e = exp2_fast(-0.5f * kLog2e * (z * z));
    return p * t * e;
}

template <int ACT>
__device__ __forceinline__ float value(float z)
{
    if constexpr (ACT == ASCB200_ACT_FASTER_GELU) return z * sigmoid(1.702f * z);
    else if constexpr (ACT == ASCB200_ACT_RELU) {
        float r;
        asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(z));
        return r;
    } else if constexpr (ACT == ASCB200_ACT_GELU) {
        float e;
        const float tail = normal_tail(z, e);
        return z > 0.0f ? fmaf(-fminf(z, 64.0f), tail, z) : z * tail;  // (the tail is 0 long before 64: infinity stays)
    } else if constexpr (ACT == ASCB200_ACT_GELU_TANH) return z * sigmoid(tanh_arg(z));
    else if constexpr (ACT == ASCB200_ACT_SILU) return z * sigmoid(z);
    else return z;
}

template <int ACT>
__device__ __forceinline__ float slope(float z)
{
    if constexpr (ACT == ASCB200_ACT_FASTER_GELU) {
        const float a = 1.702f * z, g = sigmoid(a);
        return g * fmaf(fminf(fmaxf(a, -256.0f), 256.0f), 1.0f - g, 1.0f);  // (a may be infinite where z is not; g or 1 - g is 0 long before)
    } else if constexpr (ACT == ASCB200_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
    else if constexpr (ACT == ASCB200_ACT_GELU) {
        float e;
        const float tail = normal_tail(z, e);
        return fmaf(z * 0.3989422804014327f, e, z > 0.0f ? 1.0f - tail : tail);
    } else if constexpr (ACT == ASCB200_ACT_GELU_TANH) {
        const float c = clamp_nan(z, 32.0f);
        const float g = sigmoid(tanh_arg(c));
        return g * fmaf(kTanh2u * c * fmaf(0.134145f * c, c, 1.0f), 1.0f - g, 1.0f);
    } else if constexpr (ACT == ASCB200_ACT_SILU) {
        const float g = sigmoid(z);
        return g * fmaf(z, 1.0f - g, 1.0f);
    } else return 1.0f;
}

// Runs `body` with the activation as a compile-time constant `ACT`: the choice is made once per block of values.
#define ASCB200_ACT_SWITCH(act, body)                                                                   \
    switch (act) {                                                                                      \
        case ASCB200_ACT_FASTER_GELU: { constexpr int ACT = ASCB200_ACT_FASTER_GELU; body } break;      \
        case ASCB200_ACT_RELU: { constexpr int ACT = ASCB200_ACT_RELU; body } break;                    \
        case ASCB200_ACT_GELU: { constexpr int ACT = ASCB200_ACT_GELU; body } break;                    \
        case ASCB200_ACT_GELU_TANH: { constexpr int ACT = ASCB200_ACT_GELU_TANH; body } break;          \
        case ASCB200_ACT_SILU: { constexpr int ACT = ASCB200_ACT_SILU; body } break;                    \
        default: break;                                                                                 \
    }

}  // namespace act
}  // namespace ascb200
