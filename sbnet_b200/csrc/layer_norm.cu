// Layer norm over the channels of a list of rows (a block stack [nB, bh, bw, C] is nB*bh*bw rows of C
// channels), forward and backward, for the per-position branches that run on a gathered stack.
//
//   mean = sum x / C    var = sum (x - mean)^2 / C    rstd = 1 / sqrt(var + eps)    xh = (x - mean) * rstd
//   y  = xh * w + b
//   dx = rstd * (gw - sum(gw) / C - xh * sum(gw * xh) / C)    with gw = g * w
//   dw = sum over rows of g * xh        db = sum over rows of g
//
// All three passes over the row (sum, squared distance from the mean, output) run on registers: a row is
// read once and written once, so the kernels are bound by HBM.  Statistics, products and sums are fp32
// whatever the element type; the only rounding to fewer bits is the one of each output element.
//
// Work split.  `threads per row` T is a power of two and every thread owns the same E = 8 or 16 channels of
// every row it meets, in vectors of VE elements spread T apart, so w, b and the gradient sums of those
// channels stay in registers for the whole kernel.  Up to 512 channels a row belongs to a part of a warp
// (T <= 32: reductions are shuffles, a warp works on 32/T rows at once); wider rows belong to a whole CTA
// (T = 64 .. 1024, one shared-memory exchange per reduction).  Rows of more than 16,384 channels re-read
// the row from L2 in a plain loop.  The vector width is the widest that the row pitch and the base
// addresses allow: 16 bytes, 4 bytes (two 16-bit elements) or one element.
//
// The column sums dw, db are not accumulated with atomics (their order would change the result): every CTA
// writes one fp32 partial row per gradient to the caller's workspace, and a second kernel adds the partial
// rows in a fixed order.
#include <algorithm>

#include "async_ptx.cuh"
#include "common.cuh"
#include "kernels.h"

namespace sbnet {
namespace {

constexpr int kWarpThreads = 256;   // CTA size where a row belongs to (part of) a warp

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// VE elements as raw words; kept packed until they are used.
template <typename T, int VE> struct Pack {
    static constexpr int kBytes = VE * (int)sizeof(T);
    typedef typename Vec<kBytes>::type Raw;
    Raw raw;
    __device__ __forceinline__ void load(const T* p) { raw = ld_stream(reinterpret_cast<const Raw*>(p)); }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Raw*>(p) = raw; }
    __device__ __forceinline__ void clear() { raw = vzero<kBytes>(); }
    __device__ __forceinline__ float get(int i) const { return to_f<T>(reinterpret_cast<const T*>(&raw)[i]); }
    __device__ __forceinline__ void set(int i, float v) { reinterpret_cast<T*>(&raw)[i] = from_f<T>(v); }
};

__device__ __forceinline__ float load_param(const void* p, int dtype, int i)
{
    if (dtype == 0)
        return static_cast<const float*>(p)[i];
    if (dtype == 1)
        return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_param(void* p, int dtype, int i, float v)
{
    if (dtype == 0)
        static_cast<float*>(p)[i] = v;
    else if (dtype == 1)
        static_cast<__half*>(p)[i] = __float2half_rn(v);
    else
        static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// Rows to work on: all of them, or the live blocks of a stack whose count is on the device.
__device__ __forceinline__ long long live_rows(const NormArgs& a)
{
    if (a.num_blocks_dev == nullptr)
        return a.rows;
    const long long n = max(*a.num_blocks_dev, 0);
    return min(n * a.rowsPerBlock, a.rows);
}

// Sum over the `width` lanes (a power of two) that share a row; every lane gets the same bits.
__device__ __forceinline__ float group_sum(float v, int width)
{
    for (int m = width >> 1; m > 0; m >>= 1)
        v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
}

// Sums over the whole CTA; two buffers used in turn let one barrier per reduction suffice.
template <int N> __device__ __forceinline__ void cta_sum(float (&v)[N], float* buf)
{
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < N; ++k)
        v[k] = group_sum(v[k], 32);
    if (lane == 0)
#pragma unroll
        for (int k = 0; k < N; ++k)
            buf[k * 32 + warp] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k)
        v[k] = group_sum(lane < warps ? buf[k * 32 + lane] : 0.f, 32);
}

// CTA == false: `tpr` threads (<= 32) share a row.  CTA == true: the whole CTA does (tpr == blockDim.x).
template <typename T, int VE, int NV, bool CTA> __global__ void __launch_bounds__(CTA ? 1024 : kWarpThreads)
layer_norm_kernel(NormArgs a, int tpr)
{
    __shared__ float red[4][32];
    pdl_wait();
    pdl_launch_dependents();
    const int t = CTA ? threadIdx.x : (threadIdx.x & (tpr - 1));
    const long long perPass = CTA ? gridDim.x : (long long)gridDim.x * (kWarpThreads / tpr);
    const long long first = CTA ? blockIdx.x : (long long)blockIdx.x * (kWarpThreads / tpr) + threadIdx.x / tpr;
    const long long rows = live_rows(a);
    const float inv = 1.f / (float)a.C;
    float w[NV * VE], b[NV * VE];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < VE; ++i) {
            const int c = (k * tpr + t) * VE + i;
            w[k * VE + i] = (a.weight != nullptr && c < a.C) ? load_param(a.weight, a.wdtype, c) : 1.f;
            b[k * VE + i] = (a.bias != nullptr && c < a.C) ? load_param(a.bias, a.wdtype, c) : 0.f;
        }
    // all lanes of a warp make the same number of turns (the shuffles need every lane); a lane without a
    // row of its own works on zeros and stores nothing
    const long long turns = (rows + perPass - 1) / perPass;
    int flip = 0;
    for (long long turn = 0; turn < turns; ++turn) {
        const long long row = first + turn * perPass;
        const bool live = row < rows;
        if (CTA && !live)
            break;      // the whole CTA leaves
        const T* x = static_cast<const T*>(a.x) + row * a.C;
        Pack<T, VE> v[NV];
        float s[1] = {0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * tpr + t) * VE;
            if (live && c < a.C)
                v[k].load(x + c);
            else
                v[k].clear();
        }
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < VE; ++i)
                s[0] += v[k].get(i);
        if (CTA)
            cta_sum(s, red[flip]);
        else
            s[0] = group_sum(s[0], tpr);
        const float mean = s[0] * inv;
        s[0] = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if ((k * tpr + t) * VE < a.C)
#pragma unroll
                for (int i = 0; i < VE; ++i) {
                    const float d = v[k].get(i) - mean;
                    s[0] += d * d;
                }
        if (CTA)
            cta_sum(s, red[flip + 1]);
        else
            s[0] = group_sum(s[0], tpr);
        flip ^= 2;
        const float rstd = rsqrtf(s[0] * inv + a.eps);
        if (live) {
            T* y = static_cast<T*>(a.y) + row * a.C;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int c = (k * tpr + t) * VE;
                Pack<T, VE> o;
#pragma unroll
                for (int i = 0; i < VE; ++i)
                    o.set(i, (v[k].get(i) - mean) * rstd * w[k * VE + i] + b[k * VE + i]);
                if (c < a.C)
                    o.store(y + c);
            }
            if (t == 0 && a.mean != nullptr)
                a.mean[row] = mean, a.rstd[row] = rstd;
        }
    }
}

// Any width: one CTA per row, the row read three times (the second and third time out of L2).
template <typename T> __global__ void __launch_bounds__(1024) layer_norm_loop_kernel(NormArgs a)
{
    __shared__ float red[4][32];
    pdl_wait();
    pdl_launch_dependents();
    const long long rows = live_rows(a);
    const float inv = 1.f / (float)a.C;
    int flip = 0;
    for (long long row = blockIdx.x; row < rows; row += gridDim.x, flip ^= 2) {
        const T* x = static_cast<const T*>(a.x) + row * a.C;
        T* y = static_cast<T*>(a.y) + row * a.C;
        float s[1] = {0.f};
        for (int c = threadIdx.x; c < a.C; c += blockDim.x)
            s[0] += to_f<T>(x[c]);
        cta_sum(s, red[flip]);
        const float mean = s[0] * inv;
        s[0] = 0.f;
        for (int c = threadIdx.x; c < a.C; c += blockDim.x) {
            const float d = to_f<T>(x[c]) - mean;
            s[0] += d * d;
        }
        cta_sum(s, red[flip + 1]);
        const float rstd = rsqrtf(s[0] * inv + a.eps);
        for (int c = threadIdx.x; c < a.C; c += blockDim.x) {
            const float w = a.weight != nullptr ? load_param(a.weight, a.wdtype, c) : 1.f;
            const float b = a.bias != nullptr ? load_param(a.bias, a.wdtype, c) : 0.f;
            y[c] = from_f<T>((to_f<T>(x[c]) - mean) * rstd * w + b);
        }
        if (threadIdx.x == 0 && a.mean != nullptr)
            a.mean[row] = mean, a.rstd[row] = rstd;
    }
}

// ---- backward --------------------------------------------------------------------------------------
template <typename T, int VE, int NV, bool CTA> __global__ void __launch_bounds__(CTA ? 1024 : kWarpThreads)
layer_norm_grad_kernel(NormArgs a, int tpr)
{
    constexpr int E = NV * VE;
    __shared__ float red[2][64];
    extern __shared__ float cols[];     // CTA == false: [rows at once][2][tpr * E] column sums
    pdl_wait();
    pdl_launch_dependents();
    const int t = CTA ? threadIdx.x : (threadIdx.x & (tpr - 1));
    const long long perPass = CTA ? gridDim.x : (long long)gridDim.x * (kWarpThreads / tpr);
    const long long first = CTA ? blockIdx.x : (long long)blockIdx.x * (kWarpThreads / tpr) + threadIdx.x / tpr;
    const float inv = 1.f / (float)a.C;
    float w[E], dw[E], db[E];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < VE; ++i) {
            const int c = (k * tpr + t) * VE + i;
            w[k * VE + i] = (a.weight != nullptr && c < a.C) ? load_param(a.weight, a.wdtype, c) : 1.f;
            dw[k * VE + i] = 0.f, db[k * VE + i] = 0.f;
        }
    const long long turns = (a.rows + perPass - 1) / perPass;
    int flip = 0;
    for (long long turn = 0; turn < turns; ++turn) {
        const long long row = first + turn * perPass;
        const bool live = row < a.rows;
        if (CTA && !live)
            break;
        const T* x = static_cast<const T*>(a.x) + row * a.C;
        const T* g = static_cast<const T*>(a.g) + row * a.C;
        Pack<T, VE> xv[NV], gv[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * tpr + t) * VE;
            if (live && c < a.C)
                xv[k].load(x + c), gv[k].load(g + c);
            else
                xv[k].clear(), gv[k].clear();
        }
        const float mean = live ? a.mean[row] : 0.f, rstd = live ? a.rstd[row] : 0.f;
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                const float xh = (xv[k].get(i) - mean) * rstd, gi = gv[k].get(i);    // gi == 0 past the row's end
                const float gw = gi * w[k * VE + i];
                dw[k * VE + i] += gi * xh, db[k * VE + i] += gi;
                s[0] += gw, s[1] += gw * xh;
            }
        if (CTA)
            cta_sum(s, red[flip]);
        else
            s[0] = group_sum(s[0], tpr), s[1] = group_sum(s[1], tpr);
        flip ^= 1;
        if (live) {
            T* dx = static_cast<T*>(a.y) + row * a.C;
            const float m0 = s[0] * inv, m1 = s[1] * inv;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int c = (k * tpr + t) * VE;
                Pack<T, VE> o;
#pragma unroll
                for (int i = 0; i < VE; ++i) {
                    const float xh = (xv[k].get(i) - mean) * rstd;
                    o.set(i, rstd * (gv[k].get(i) * w[k * VE + i] - m0 - xh * m1));
                }
                if (c < a.C)
                    o.store(dx + c);
            }
        }
    }
    if (a.partials == nullptr)
        return;
    float* pw = a.partials + (long long)blockIdx.x * 2 * a.C;
    if (CTA) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                const int c = (k * tpr + t) * VE + i;
                if (c < a.C)
                    pw[c] = dw[k * VE + i], pw[a.C + c] = db[k * VE + i];
            }
    } else {
        const int groups = kWarpThreads / tpr, grp = threadIdx.x / tpr, width = tpr * E;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                const int c = (k * tpr + t) * VE + i;
                cols[(grp * 2 + 0) * width + c] = dw[k * VE + i];
                cols[(grp * 2 + 1) * width + c] = db[k * VE + i];
            }
        __syncthreads();
        for (int c = threadIdx.x; c < 2 * a.C; c += kWarpThreads) {
            const int half = c >= a.C, cc = c - half * a.C;
            float s = 0.f;
            for (int q = 0; q < groups; ++q)
                s += cols[(q * 2 + half) * width + cc];
            pw[c] = s;
        }
    }
}

template <typename T> __global__ void __launch_bounds__(1024) layer_norm_grad_loop_kernel(NormArgs a)
{
    __shared__ float red[2][64];
    pdl_wait();
    pdl_launch_dependents();
    const float inv = 1.f / (float)a.C;
    float* pw = a.partials == nullptr ? nullptr : a.partials + (long long)blockIdx.x * 2 * a.C;
    if (pw != nullptr)
        for (int c = threadIdx.x; c < a.C; c += blockDim.x)
            pw[c] = 0.f, pw[a.C + c] = 0.f;      // each thread owns its columns throughout
    int flip = 0;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, flip ^= 1) {
        const T* x = static_cast<const T*>(a.x) + row * a.C;
        const T* g = static_cast<const T*>(a.g) + row * a.C;
        T* dx = static_cast<T*>(a.y) + row * a.C;
        const float mean = a.mean[row], rstd = a.rstd[row];
        float s[2] = {0.f, 0.f};
        for (int c = threadIdx.x; c < a.C; c += blockDim.x) {
            const float xh = (to_f<T>(x[c]) - mean) * rstd, gi = to_f<T>(g[c]);
            const float gw = gi * (a.weight != nullptr ? load_param(a.weight, a.wdtype, c) : 1.f);
            s[0] += gw, s[1] += gw * xh;
            if (pw != nullptr)
                pw[c] += gi * xh, pw[a.C + c] += gi;
        }
        cta_sum(s, red[flip]);
        const float m0 = s[0] * inv, m1 = s[1] * inv;
        for (int c = threadIdx.x; c < a.C; c += blockDim.x) {
            const float xh = (to_f<T>(x[c]) - mean) * rstd;
            const float gw = to_f<T>(g[c]) * (a.weight != nullptr ? load_param(a.weight, a.wdtype, c) : 1.f);
            dx[c] = from_f<T>(rstd * (gw - m0 - xh * m1));
        }
    }
}

// dw, db: the partial rows added in a fixed order, 32 columns a CTA, 32 rows of partials at a time.
__global__ void __launch_bounds__(1024) layer_norm_reduce_kernel(NormArgs a, int parts)
{
    __shared__ float tile[32][33];
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;
    float s = 0.f;
    if (c < 2 * a.C)
        for (int p = grp; p < parts; p += 32)
            s += a.partials[(long long)p * 2 * a.C + c];
    tile[grp][lane] = s;
    __syncthreads();
    const float v = group_sum(tile[lane][grp], 32);    // warp `grp` sums column `grp` of the tile
    const int col = blockIdx.x * 32 + grp;
    if (lane == 0 && col < 2 * a.C) {
        void* dst = col < a.C ? a.dweight : a.dbias;
        if (dst != nullptr)
            store_param(dst, a.wdtype, col < a.C ? col : col - a.C, v);
    }
}

// ---- launches ----------------------------------------------------------------------------------------
struct NormShape {
    int vecBytes;   // bytes of a vector
    int tpr;        // threads that share a row; 0: the loop kernels
    int elems;      // channels per thread (8 or 16)
    bool cta;
};

NormShape pick(int C, int itemsize, uintptr_t bits)
{
    NormShape s = {itemsize, 0, 0, false};
    const uintptr_t all = bits | (uintptr_t)((long long)C * itemsize);
    if ((all & 15) == 0)
        s.vecBytes = 16;
    else if (itemsize == 2 && (all & 3) == 0)
        s.vecBytes = 4;
    // up to 256 channels: 8 a thread; up to 512: 16 a thread, still inside a warp; then whole CTAs
    if (C <= 512) {
        s.elems = C <= 256 ? 8 : 16;
        s.tpr = 4;
        while (s.tpr * s.elems < C)
            s.tpr *= 2;
    } else if (C <= 16384) {
        s.cta = true;
        s.elems = C <= 8192 ? 8 : 16;
        s.tpr = 64;
        while (s.tpr * s.elems < C)
            s.tpr *= 2;
    }
    return s;
}

template <typename T, int VE, int NV> cudaError_t launch_fwd(const NormArgs& a, const NormShape& s, cudaStream_t stream)
{
    if (s.cta) {
        const long long grid = std::min<long long>(a.rows, (long long)sm_count() * (2048 / s.tpr) * 4);
        return launch_pdl(layer_norm_kernel<T, VE, NV, true>, dim3((unsigned)grid), dim3(s.tpr), 0, stream, a, s.tpr);
    }
    const long long ctas = (a.rows * s.tpr + kWarpThreads - 1) / kWarpThreads;
    const long long grid = std::min<long long>(ctas, (long long)sm_count() * 8);
    return launch_pdl(layer_norm_kernel<T, VE, NV, false>, dim3((unsigned)grid), dim3(kWarpThreads), 0, stream, a, s.tpr);
}

template <typename T, int VE, int NV> cudaError_t launch_bwd(const NormArgs& a, const NormShape& s, int grid, cudaStream_t stream)
{
    if (s.cta)
        return launch_pdl(layer_norm_grad_kernel<T, VE, NV, true>, dim3(grid), dim3(s.tpr), 0, stream, a, s.tpr);
    const size_t smem = a.partials == nullptr ? 0 : sizeof(float) * 2 * kWarpThreads * NV * VE;
    return launch_pdl(layer_norm_grad_kernel<T, VE, NV, false>, dim3(grid), dim3(kWarpThreads), smem, stream, a, s.tpr);
}

template <typename T> cudaError_t run_fwd(const NormArgs& a, cudaStream_t stream)
{
    const NormShape s = pick(a.C, sizeof(T), reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y));
    constexpr int V16 = 16 / (int)sizeof(T);
    if (s.tpr == 0)
        return launch_pdl(layer_norm_loop_kernel<T>, dim3((unsigned)std::min<long long>(a.rows, sm_count() * 2)), dim3(1024),
                          0, stream, a);
    if (s.vecBytes == 16)
        return s.elems == 8 ? launch_fwd<T, V16, 8 / V16>(a, s, stream) : launch_fwd<T, V16, 16 / V16>(a, s, stream);
    if constexpr (sizeof(T) == 2)
        if (s.vecBytes == 4)
            return s.elems == 8 ? launch_fwd<T, 2, 4>(a, s, stream) : launch_fwd<T, 2, 8>(a, s, stream);
    return s.elems == 8 ? launch_fwd<T, 1, 8>(a, s, stream) : launch_fwd<T, 1, 16>(a, s, stream);
}

template <typename T> cudaError_t run_bwd(const NormArgs& a, int grid, cudaStream_t stream)
{
    const NormShape s = pick(a.C, sizeof(T), reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y) |
                                                 reinterpret_cast<uintptr_t>(a.g));
    constexpr int V16 = 16 / (int)sizeof(T);
    if (s.tpr == 0)
        return launch_pdl(layer_norm_grad_loop_kernel<T>, dim3(grid), dim3(1024), 0, stream, a);
    if (s.vecBytes == 16)
        return s.elems == 8 ? launch_bwd<T, V16, 8 / V16>(a, s, grid, stream) : launch_bwd<T, V16, 16 / V16>(a, s, grid, stream);
    if constexpr (sizeof(T) == 2)
        if (s.vecBytes == 4)
            return s.elems == 8 ? launch_bwd<T, 2, 4>(a, s, grid, stream) : launch_bwd<T, 2, 8>(a, s, grid, stream);
    return s.elems == 8 ? launch_bwd<T, 1, 8>(a, s, grid, stream) : launch_bwd<T, 1, 16>(a, s, grid, stream);
}

} // namespace

// CTAs of the backward kernel = partial rows of the column sums.  Depends on the sizes only.
int layer_norm_grad_parts(long long rows, int C)
{
    const NormShape s = pick(C, 4, 0);
    if (s.tpr == 0)
        return (int)std::min<long long>(rows, sm_count());
    if (s.cta)
        return (int)std::min<long long>(rows, (long long)sm_count() * std::max(1, 1024 / s.tpr));
    return (int)std::min<long long>((rows * s.tpr + kWarpThreads - 1) / kWarpThreads, (long long)sm_count() * 4);
}

cudaError_t launch_layer_norm(const NormArgs& a, int dtype, cudaStream_t stream)
{
    note_site("layer_norm");
    if (dtype == 0)
        return run_fwd<float>(a, stream);
    return dtype == 1 ? run_fwd<__half>(a, stream) : run_fwd<__nv_bfloat16>(a, stream);
}

cudaError_t launch_layer_norm_grad(const NormArgs& a, int dtype, cudaStream_t stream)
{
    note_site("layer_norm_grad");
    const int parts = layer_norm_grad_parts(a.rows, a.C);
    cudaError_t e = a.rows == 0  ? cudaSuccess      // no rows: the weight gradients are sums of nothing
                    : dtype == 0   ? run_bwd<float>(a, parts, stream)
                    : dtype == 1 ? run_bwd<__half>(a, parts, stream)
                                 : run_bwd<__nv_bfloat16>(a, parts, stream);
    if (e != cudaSuccess || (a.dweight == nullptr && a.dbias == nullptr))
        return e;
    note_site("layer_norm_grad column sums");
    return launch_pdl(layer_norm_reduce_kernel, dim3((2u * a.C + 31) / 32), dim3(1024), 0, stream, a, parts);
}

} // namespace sbnet
