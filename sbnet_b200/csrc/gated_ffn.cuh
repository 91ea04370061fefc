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

// act(g), and its derivative where it is asked for.
template <int ACT, bool SLOPE> __device__ __forceinline__ float activate(float g, float& slope)
{
    if constexpr (ACT == kSilu) {
        const float s = __fdividef(1.f, 1.f + __expf(-g));
        if (SLOPE)
            slope = s * (1.f + g * (1.f - s));
        return g * s;
    } else if constexpr (ACT == kGelu) {
        const float cdf = 0.5f * (1.f + erff(g * 0.70710678118654752f));
        if (SLOPE)
            slope = cdf + g * 0.3989422804014327f * __expf(-0.5f * g * g);
        return g * cdf;
    } else {
        if (SLOPE)
            slope = g > 0.f ? 1.f : 0.f;
        return g != g ? g : fmaxf(g, 0.f);
    }
}
__device__ __forceinline__ float activate_any(int act, float g)
{
    float unused;
    return act == kSilu   ? activate<kSilu, false>(g, unused)
           : act == kGelu ? activate<kGelu, false>(g, unused)
                          : activate<kRelu, false>(g, unused);
}

// Rows to work on: all of them, or those of the live blocks of a stack whose count is on the device.
__device__ __forceinline__ long long live_rows(long long rows, const int32_t* blocks, int rowsPerBlock)
{
    return blocks == nullptr ? rows : min(rows, (long long)max(*blocks, 0) * rowsPerBlock);
}

// Up to 32 rows (gated_ffn_few.cu): h [rows, F] is scratch.  *taken tells whether the sizes suit the kernels.
template <typename T> cudaError_t launch_ffn_few(const FfnArgs& f, void* h, cudaStream_t stream, bool* taken);

} // namespace sbnet
