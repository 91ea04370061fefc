// What the kernels of the gated feed-forward block share: the activation, conversions between fp32 and pairs of 16-bit
// elements, and the launcher of the few-row kernels.
#pragma once
#include "common.cuh"
#include "kernels.h"

namespace sbnet {

enum Act { kSilu = 0, kGelu = 1, kRelu = 2 };

template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi)
{
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi)
{
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t v);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t v)
{
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v)
{
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}

__device__ __forceinline__ float exp2_fast(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float recip_fast(float x)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// act of two values, and the derivatives where they are asked for.  The epilogues are bound by the special-function unit
// (16 operations a clock and SM) and by issue slots, hence:
//  silu: both sigmoids from one reciprocal, 1 / ((1 + e0)(1 + e1)); 2^60 bounds each factor (sigmoids below 2^-60 read
//        as 2^-60, an error of |g| 2^-60).
//  gelu: Phi(g) by the rational approximation of Abramowitz and Stegun 7.1.26 for erfc (|error| <= 1.5e-7), whose
//        exponential is the density that the derivative needs.
template <int ACT, bool SLOPE> __device__ __forceinline__ void activate2(float g0, float g1, float& a0, float& a1, float& s0, float& s1)
{
    if constexpr (ACT == kSilu) {
        const float f0 = 1.f + exp2_fast(fminf(g0 * -1.4426950408889634f, 60.f));
        const float f1 = 1.f + exp2_fast(fminf(g1 * -1.4426950408889634f, 60.f));
        const float r = recip_fast(f0 * f1), p0 = r * f1, p1 = r * f0;
        a0 = g0 * p0, a1 = g1 * p1;
        if (SLOPE)
            s0 = p0 + a0 * (1.f - p0), s1 = p1 + a1 * (1.f - p1);
    } else if constexpr (ACT == kGelu) {
        auto one = [](float g, float& a, float& s) {
            const float z = fabsf(g) * 0.70710678118654752f, t = recip_fast(1.f + 0.3275911f * z);
            const float e = exp2_fast(g * g * -0.72134752044448170f);        // exp(-g^2 / 2)
            const float q = 0.5f * e * t *
                            (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
            const float cdf = g < 0.f ? q : 1.f - q;
            a = g * cdf;
            if (SLOPE)
                s = cdf + g * 0.3989422804014327f * e;
        };
        one(g0, a0, s0), one(g1, a1, s1);
    } else {
        a0 = g0 != g0 ? g0 : fmaxf(g0, 0.f), a1 = g1 != g1 ? g1 : fmaxf(g1, 0.f);
        if (SLOPE)
            s0 = g0 > 0.f ? 1.f : 0.f, s1 = g1 > 0.f ? 1.f : 0.f;
    }
}
__device__ __forceinline__ float activate_any(int act, float g)
{
    float a, unused;
    if (act == kSilu)
        activate2<kSilu, false>(g, 0.f, a, unused, unused, unused);
    else if (act == kGelu)
        activate2<kGelu, false>(g, 0.f, a, unused, unused, unused);
    else
        activate2<kRelu, false>(g, 0.f, a, unused, unused, unused);
    return a;
}

// Rows to work on: all of them, or those of the live blocks of a stack whose count is on the device.
__device__ __forceinline__ long long live_rows(long long rows, const int32_t* blocks, int rowsPerBlock)
{
    return blocks == nullptr ? rows : min(rows, (long long)max(*blocks, 0) * rowsPerBlock);
}

// Up to 32 rows (gated_ffn_few.cu): h [rows, F] is scratch.  *taken tells whether the sizes suit the kernels.
template <typename T> cudaError_t launch_ffn_few(const FfnArgs& f, void* h, cudaStream_t stream, bool* taken);

} // namespace sbnet
