// What the kernels of the gated feed-forward block share: the activation, conversions between fp32 and pairs of 16-bit
// elements, tiles staged between registers and memory, tensor maps, and the launchers of the special cases.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>

#include "common.cuh"
#include "kernels.h"
#include "pairs.cuh"
#include "tensor_ptx.cuh"

namespace sbnet {

enum Act { kSilu = 0, kGelu = 1, kRelu = 2 };

constexpr int kStepK = 64;      // reduction steps of a shared-memory stage (128 bytes)

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
// The larger of two, or not a number where one is.
__device__ __forceinline__ float max_or_nan(float x, float y)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
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
//  silu: both sigmoids from one reciprocal, 1 / ((1 + e0)(1 + e1)); 2^60 bounds each factor.  Sigmoids below 2^-60, of g
//        below -60 ln 2, read as 2^-60, and g is bounded there too: silu is off by at most 42 * 2^-60 however far g is.
//  gelu: Phi(g) by the rational approximation of Abramowitz and Stegun 7.1.26 for erfc (|error| <= 1.5e-7), whose
//        exponential is the density that the derivative needs.
template <int ACT, bool SLOPE> __device__ __forceinline__ void activate2(F2 g, F2& a, F2& slope)
{
    const F2 one = f2(1.f, 1.f);
    if constexpr (ACT == kSilu) {
        const float2 x = unpair(mul2(g, f2(-1.4426950408889634f, -1.4426950408889634f)));
        const F2 e = f2(exp2_fast(fminf(x.x, 60.f)), exp2_fast(fminf(x.y, 60.f)));
        const float2 f = unpair(add2(e, one));
        const float r = recip_fast(f.x * f.y);
        const F2 sig = mul2(f2(r, r), f2(f.y, f.x));
        const float2 gs = unpair(g);
        a = mul2(f2(max_or_nan(gs.x, -41.588830833596717f), max_or_nan(gs.y, -41.588830833596717f)), sig);
        if (SLOPE)      // sig + a (1 - sig); 1 - sig as e sig, which vanishes with e: sig itself is off by its rounding, and a
                        // large g would carry that into the slope
            slope = fma2(a, mul2(e, sig), sig);
    } else if constexpr (ACT == kGelu) {
        const float2 gs = unpair(g);
        const float2 z = make_float2(fabsf(gs.x) * 0.70710678118654752f, fabsf(gs.y) * 0.70710678118654752f);
        const float2 den = unpair(fma2(f2(z.x, z.y), f2(0.3275911f, 0.3275911f), one));
        const F2 t = f2(recip_fast(den.x), recip_fast(den.y));
        const float2 x = unpair(mul2(mul2(g, g), f2(-0.72134752044448170f, -0.72134752044448170f)));
        const F2 e = f2(exp2_fast(x.x), exp2_fast(x.y));        // exp(-g^2 / 2)
        F2 q = f2(1.061405429f, 1.061405429f);
        q = fma2(q, t, f2(-1.453152027f, -1.453152027f));
        q = fma2(q, t, f2(1.421413741f, 1.421413741f));
        q = fma2(q, t, f2(-0.284496736f, -0.284496736f));
        q = fma2(q, t, f2(0.254829592f, 0.254829592f));
        const float2 tail = unpair(mul2(mul2(q, t), mul2(e, f2(0.5f, 0.5f))));
        const F2 cdf = f2(gs.x < 0.f ? tail.x : 1.f - tail.x, gs.y < 0.f ? tail.y : 1.f - tail.y);
        a = mul2(g, cdf);
        if (SLOPE)
            slope = fma2(mul2(g, f2(0.3989422804014327f, 0.3989422804014327f)), e, cdf);
    } else {
        const float2 gs = unpair(g);
        a = f2(gs.x != gs.x ? gs.x : fmaxf(gs.x, 0.f), gs.y != gs.y ? gs.y : fmaxf(gs.y, 0.f));
        if (SLOPE)
            slope = f2(gs.x > 0.f ? 1.f : 0.f, gs.y > 0.f ? 1.f : 0.f);
    }
}
__device__ __forceinline__ float activate_any(int act, float g)
{
    F2 a, unused;
    if (act == kSilu)
        activate2<kSilu, false>(f2(g, 0.f), a, unused);
    else if (act == kGelu)
        activate2<kGelu, false>(f2(g, 0.f), a, unused);
    else
        activate2<kRelu, false>(f2(g, 0.f), a, unused);
    return unpair(a).x;
}
// Two neighbouring accumulator words as a pair; a pair rounded to 16 bits.
__device__ __forceinline__ F2 words(uint32_t lo, uint32_t hi) { return f2(__uint_as_float(lo), __uint_as_float(hi)); }
template <typename T> __device__ __forceinline__ uint32_t pack2(F2 v)
{
    const float2 f = unpair(v);
    return pack2<T>(f.x, f.y);
}

// Rows to work on: all of them, or those of the live blocks of a stack whose count is on the device.
__device__ __forceinline__ long long live_rows(long long rows, const int32_t* blocks, int rowsPerBlock)
{
    return blocks == nullptr ? rows : min(rows, (long long)max(*blocks, 0) * rowsPerBlock);
}

// ---- 32 x 32 tiles of 16-bit elements between registers (one row per lane) and memory -----------------------
// Staged through 2 KB of shared memory so that global accesses are 64 contiguous bytes per row.  16-byte pieces
// are swizzled by row as TMA's 64-byte mode does it: eight lanes touch eight different pieces of 128 bytes whichever
// way the tile is walked, and one of the epilogues sends its tiles by TMA straight from here.
__device__ __forceinline__ uint32_t piece(uint32_t buf, int row, int c) { return buf + row * 64 + ((c ^ ((row >> 1) & 3)) << 4); }

__device__ __forceinline__ void stage_rows(uint32_t buf, int lane, const uint32_t (&w)[16])
{
#pragma unroll
    for (int c = 0; c < 4; ++c)
        sts128(piece(buf, lane, c), make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]));
}
// Where a lane's pieces of a tile lie in a matrix of pitch ld: rows r, r + 8, .. r + 24 (r = lane / 4) of row0.., of which
// the first `rows` pieces are below rowEnd, and columns col.., of which `cols` are below N.
struct Spot {
    long long at, step;
    int rows, cols;
};
__device__ __forceinline__ Spot spot(long long ld, long long row0, long long rowEnd, int col0, int N, int lane)
{
    const int r = lane >> 2, col = col0 + (lane & 3) * 8;
    const long long left = rowEnd - row0 - r;
    return {(row0 + r) * ld + col, 8 * ld, left <= 0 ? 0 : left >= 32 ? 4 : ((int)left + 7) >> 3, N - col};
}
// tile -> memory
template <typename T> __device__ __forceinline__ void store_tile(void* out, const Spot& s, bool wide, uint32_t buf, int lane)
{
    T* dst = static_cast<T*>(out) + s.at;
#pragma unroll
    for (int i = 0; i < 4; ++i, dst += s.step) {
        const uint4 v = lds128(piece(buf, i * 8 + (lane >> 2), lane & 3));
        if (i >= s.rows)
            continue;
        if (wide && s.cols >= 8) {
            *reinterpret_cast<uint4*>(dst) = v;
        } else {
            const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k < s.cols)
                    dst[k] = e[k];
        }
    }
}
// ---- host side ----
inline PFN_cuTensorMapEncodeTiled encoder()
{
    static const PFN_cuTensorMapEncodeTiled fn = [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            return reinterpret_cast<PFN_cuTensorMapEncodeTiled>(ptr);
        (void)cudaGetLastError();
        return static_cast<PFN_cuTensorMapEncodeTiled>(nullptr);
    }();
    return fn;
}

// A row-major matrix as TMA reads it (16-bit elements, boxes of 64 columns x boxRows rows) or writes it (boxes of 64
// bytes x 32 rows).
struct Matrix {
    const void* ptr;
    long long rows;
    int cols;
    long long ld;
};
inline cudaError_t encode(const Matrix& m, int boxRows, CUtensorMap* out, int boxCols = kStepK, int itemsize = 2)
{
    PFN_cuTensorMapEncodeTiled enc = encoder();
    if (enc == nullptr)
        return cudaErrorNotSupported;
    const cuuint64_t dims[2] = {(cuuint64_t)m.cols, (cuuint64_t)m.rows}, strides[1] = {(cuuint64_t)m.ld * itemsize};
    const cuuint32_t box[2] = {(cuuint32_t)boxCols, (cuuint32_t)boxRows}, estr[2] = {1, 1};
    return enc(out, itemsize == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(m.ptr), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, boxCols * itemsize == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? cudaSuccess
               : cudaErrorInvalidValue;
}

inline int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

// Up to 32 rows (gated_ffn_few.cu): h [rows, F] is scratch.  *taken tells whether the sizes suit the kernels.
template <typename T> cudaError_t launch_ffn_few(const FfnArgs& f, void* h, cudaStream_t stream, bool* taken);

// Where ffn_fused_suits(), both products in one kernel (gated_ffn_fused.cu).  The matrices are what TMA can read.
template <typename T>
cudaError_t launch_ffn_fused(const FfnArgs& f, const Matrix& x, const Matrix& wg, const Matrix& wu, const Matrix& wd,
                             cudaStream_t stream);
bool ffn_fused_suits(long long rows, int C);
cudaError_t read_ffn_fused_wait_timeouts(unsigned int* out);

} // namespace sbnet
