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
// (T <= 32: reductions are shuffles, a warp works on 32/T rows at once and has several such sets in flight);
// wider rows belong to a whole CTA (T = 64 .. 1024, one barrier a row, the next row loading behind it).  Rows of more than 16,384 channels re-read
// the row from L2 in a plain loop.  The vector width is the widest that the row pitch and the base
// addresses allow: 16 bytes, 4 bytes (two 16-bit elements) or one element.
//
// Measured: 419,328 x 128 fp16 45 us (4.8 TB/s); 419,328 x 256 bf16, forward and backward together, 202 us (5.3 TB/s),
// both at 0.7 of the issue slots; 40,000 x 1,024 fp32 (with a cold L2, launch included) 74 us (4.4 TB/s), backward 110.
// Those slots go to 20 instructions a channel forward and 27 backward, where the formula needs some five.  The launch
// bounds that keep three CTAs an SM leave 80 registers: two rows of 16 channels beside w and b spill 104 (fp16) and 80
// (bf16) bytes a thread, forms of narrow vectors up to 416.
//
// The column sums dw, db are not accumulated with atomics (their order would change the result): every CTA
// writes one fp32 partial row per gradient to the caller's workspace, and a second kernel adds the partial
// rows in a fixed order.
#include <algorithm>

#include "async_ptx.cuh"
#include "common.cuh"
#include "kernels.h"
#include "pairs.cuh"

namespace sbnet {
namespace {

constexpr int kWarpThreads = 256;   // CTA size where a row belongs to (part of) a warp
constexpr int kFwdCtas = 3;         // ... and such CTAs per SM, all resident: forward
constexpr int kGradCtas = 3;        // ... backward with 8 channels a thread
constexpr int kGradCtas16 = 2;      // ... with 16

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
    __device__ __forceinline__ void set2(int i, float2 v)    // elements i and i + 1, i even
    {
        if constexpr (std::is_same<T, __half>::value)
            reinterpret_cast<__half2*>(&raw)[i / 2] = __floats2half2_rn(v.x, v.y);
        else if constexpr (std::is_same<T, __nv_bfloat16>::value)
            reinterpret_cast<__nv_bfloat162*>(&raw)[i / 2] = __floats2bfloat162_rn(v.x, v.y);
        else
            reinterpret_cast<float2*>(&raw)[i / 2] = v;
    }
};

// A thread's E = NV * VE channels of a row as E / 2 pairs, and back.
template <typename T, int VE, int NV> __device__ __forceinline__ F2 pair_of(const Pack<T, VE> (&v)[NV], int j)
{
    return f2(v[2 * j / VE].get(2 * j % VE), v[(2 * j + 1) / VE].get((2 * j + 1) % VE));
}
template <typename T, int VE, int NV, bool FULL = false>
__device__ __forceinline__ void store_pairs(T* row, const F2 (&o)[NV * VE / 2], int t, int tpr, int C)
{
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (k * tpr + t) * VE;
        Pack<T, VE> p;
        if constexpr (VE == 1) {
            p.set(0, k % 2 ? unpair(o[k / 2]).y : unpair(o[k / 2]).x);
        } else {
#pragma unroll
            for (int i = 0; i < VE; i += 2)
                p.set2(i, unpair(o[(k * VE + i) / 2]));
        }
        if (FULL || c < C)
            p.store(row + c);
    }
}

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
    // CTAs have a power of two of warps: the lanes repeat the warps' sums, and a group of that width adds them up
#pragma unroll
    for (int k = 0; k < N; ++k)
        v[k] = group_sum(buf[k * 32 + (lane & (warps - 1))], warps);
}

// This thread's channels of a row; zeros past the end of the row and for rows that are not there.
template <typename T, int VE, int NV>
__device__ __forceinline__ void load_row(Pack<T, VE> (&v)[NV], const T* row, bool live, int t, int tpr, int C)
{
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (k * tpr + t) * VE;
        if (live && c < C)
            v[k].load(row + c);
        else
            v[k].clear();
    }
}

// Loads that run ahead of their use through shared memory: every thread copies its own vectors of the turns to come
// (cp.async) into slots of its own and reads them back itself, so nothing but the thread's own wait is needed and no
// registers are held meanwhile.  Vectors of one 16-bit element are too narrow for cp.async and are loaded when used.
constexpr int kAhead = 3;      // turns in shared memory: the current one and two in flight
constexpr int kAheadCta = 2;   // the same in the whole-CTA backward kernel, whose turns are two rows of two tensors
template <typename T, int VE> constexpr bool kCanRunAhead = VE * sizeof(T) >= 4;
template <typename T, int VE> constexpr int kSlotBytes = kCanRunAhead<T, VE> ? VE * (int)sizeof(T) : 0;

// FULL: the row is there and every thread's vectors lie inside it.
template <typename T, int VE, int NV, bool FULL = false>
__device__ __forceinline__ void copy_row(uint32_t slots, const T* row, bool live, int t, int tpr, int C)
{
    if constexpr (kCanRunAhead<T, VE>) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * tpr + t) * VE;
            const uint32_t dst = slots + k * blockDim.x * kSlotBytes<T, VE>;
            if (FULL || (live && c < C)) {
                if constexpr (VE * sizeof(T) == 16)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(row + c) : "memory");
                else
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(row + c) : "memory");
            }
        }
    }
}
template <typename T, int VE, int NV, bool FULL = false>
__device__ __forceinline__ void take_row(Pack<T, VE> (&v)[NV], uint32_t slots, const T* row, bool live, int t, int tpr, int C)
{
    if constexpr (kCanRunAhead<T, VE>) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const uint32_t src = slots + k * blockDim.x * kSlotBytes<T, VE>;
            if (!FULL)
                v[k].clear();
            if (FULL || (live && (k * tpr + t) * VE < C)) {
                if constexpr (VE * sizeof(T) == 16)
                    v[k].raw = lds128(src);
                else
                    v[k].raw = lds32(src);
            }
        }
    } else {
        load_row<T, VE, NV>(v, row, FULL || live, t, tpr, C);
    }
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory"); }
// Shared memory of `rows` rows (or pairs of rows) per turn and thread.
template <typename T, int VE, int NV> constexpr int slots_bytes(int threads, int rows) { return kAhead * rows * NV * threads * kSlotBytes<T, VE>; }

// The row as pairs; returns its sum.
template <typename T, int VE, int NV>
__device__ __forceinline__ float row_sum(const Pack<T, VE> (&v)[NV], F2 (&f)[NV * VE / 2])
{
    F2 s = f2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < NV * VE / 2; ++j) {
        f[j] = pair_of<T, VE, NV>(v, j);
        s = add2(s, f[j]);
    }
    return both(s);
}
// Replaces the row by its distances from `mean` (zero past the row's end); returns the sum of their squares.
template <int VE, int NV, bool FULL = false>
__device__ __forceinline__ float row_spread(F2 (&f)[NV * VE / 2], float mean, int t, int tpr, int C)
{
    const F2 m = f2(-mean, -mean);
#pragma unroll
    for (int j = 0; j < NV * VE / 2; ++j)
        f[j] = add2(f[j], m);
    if (!FULL && tpr * NV * VE != C) {    // some threads reach past the end
#pragma unroll
        for (int j = 0; j < NV * VE / 2; ++j) {
            float2 d = unpair(f[j]);
            if ((2 * j / VE * tpr + t) * VE >= C)
                d.x = 0.f;
            if (((2 * j + 1) / VE * tpr + t) * VE >= C)
                d.y = 0.f;
            f[j] = f2(d.x, d.y);
        }
    }
    F2 s = f2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < NV * VE / 2; ++j)
        s = fma2(f[j], f[j], s);
    return both(s);
}

template <int VE, int NV>
__device__ __forceinline__ void load_params(F2 (&w)[NV * VE / 2], const void* p, float dflt, int dtype, int t, int tpr, int C)
{
    auto at = [&](int e) {
        const int c = (e / VE * tpr + t) * VE + e % VE;
        return (p != nullptr && c < C) ? load_param(p, dtype, c) : dflt;
    };
#pragma unroll
    for (int j = 0; j < NV * VE / 2; ++j)
        w[j] = f2(at(2 * j), at(2 * j + 1));
}

// f: distances from the row's mean + `shift`
template <typename T, int VE, int NV, bool FULL = false>
__device__ __forceinline__ void store_normed(T* y, F2 (&f)[NV * VE / 2], float shift, float rstd, const F2 (&w)[NV * VE / 2],
                                             const F2 (&b)[NV * VE / 2], int t, int tpr, int C)
{
    const F2 m = f2(-shift, -shift), r = f2(rstd, rstd);
#pragma unroll
    for (int j = 0; j < NV * VE / 2; ++j)
        f[j] = fma2(mul2(shift == 0.f ? f[j] : add2(f[j], m), r), w[j], b[j]);
    store_pairs<T, VE, NV, FULL>(y, f, t, tpr, C);
}

// `tpr` threads (<= 32) share a row; every turn takes ROWS rows per group.
template <typename T, int VE, int NV, int ROWS>
__global__ void __launch_bounds__(kWarpThreads, kFwdCtas) layer_norm_warp_kernel(NormArgs a, int tpr)
{
    extern __shared__ __align__(16) uint8_t dyn[];
    pdl_wait();
    pdl_launch_dependents();
    const int t = threadIdx.x & (tpr - 1);
    const long long groups = (long long)gridDim.x * (kWarpThreads / tpr);
    const long long first = (long long)blockIdx.x * (kWarpThreads / tpr) + threadIdx.x / tpr;
    const long long rows = live_rows(a);
    const float inv = 1.f / (float)a.C;
    const T* x = static_cast<const T*>(a.x);
    constexpr int rowBytes = NV * kWarpThreads * kSlotBytes<T, VE>;
    const uint32_t slots = smem_u32(dyn) + threadIdx.x * kSlotBytes<T, VE>;
    // all lanes of a warp make the same number of turns (the shuffles need every lane); a lane without a
    // row of its own works on zeros and stores nothing
    const long long turns = (rows + groups * ROWS - 1) / (groups * ROWS);
    auto fetch = [&](auto full, long long turn, uint32_t stage) {
        const uint32_t at = slots + stage * ROWS * rowBytes;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const long long row = (turn * ROWS + r) * groups + first;
            copy_row<T, VE, NV, decltype(full)::value>(at + r * rowBytes, x + row * a.C, row < rows, t, tpr, a.C);
        }
        copies_commit();
    };
#pragma unroll
    for (int i = 0; i < kAhead - 1; ++i)
        fetch(std::false_type(), i, i);
    F2 w[NV * VE / 2], b[NV * VE / 2];
    load_params<VE, NV>(w, a.weight, 1.f, a.wdtype, t, tpr, a.C);
    load_params<VE, NV>(b, a.bias, 0.f, a.wdtype, t, tpr, a.C);
    // One turn; FULL: all of its rows are there, those it fetches too, and the threads cover the channels exactly, so that
    // nothing is checked (a fifth of the instructions of this kernel, which sits at the issue limit)
    uint32_t stage = 0;
    auto body = [&](auto full, long long turn) {
        constexpr bool FULL = decltype(full)::value;
        const long long row0 = turn * ROWS * groups + first;
        fetch(full, turn + kAhead - 1, stage == 0 ? kAhead - 1 : stage - 1);
        copies_wait();
        const uint32_t at = slots + stage * ROWS * rowBytes;
        F2 f[ROWS][NV * VE / 2];
        float mean[ROWS], rstd[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const long long row = row0 + r * groups;
            Pack<T, VE> v[NV];
            take_row<T, VE, NV, FULL>(v, at + r * rowBytes, x + row * a.C, row < rows, t, tpr, a.C);
            mean[r] = row_sum<T, VE, NV>(v, f[r]);
        }
        for (int m = tpr >> 1; m > 0; m >>= 1)
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
                mean[r] += __shfl_xor_sync(0xffffffffu, mean[r], m);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            mean[r] *= inv;
            rstd[r] = row_spread<VE, NV, FULL>(f[r], mean[r], t, tpr, a.C);
        }
        for (int m = tpr >> 1; m > 0; m >>= 1)
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
                rstd[r] += __shfl_xor_sync(0xffffffffu, rstd[r], m);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const long long row = row0 + r * groups;
            if (!FULL && row >= rows)
                continue;
            rstd[r] = rsqrtf(rstd[r] * inv + a.eps);
            store_normed<T, VE, NV, FULL>(static_cast<T*>(a.y) + row * a.C, f[r], 0.f, rstd[r], w, b, t, tpr, a.C);
            if (t == 0 && a.mean != nullptr)
                a.mean[row] = mean[r], a.rstd[row] = rstd[r];
        }
        stage = stage + 1 == kAhead ? 0 : stage + 1;
    };
    long long turn = 0;
    if (tpr * NV * VE == a.C)
        for (; turn + kAhead < turns; ++turn)       // the last turn may lack rows, and kAhead - 1 turns are fetched ahead
            body(std::true_type(), turn);
    for (; turn < turns; ++turn)
        body(std::false_type(), turn);
}

// The whole CTA shares a row.  Each warp takes mean and spread of its own channels, and the warps' results are joined
// (mean = sum n_w mean_w / C, spread = sum spread_w + n_w (mean_w - mean)^2), which needs one barrier a row.
template <typename T, int VE, int NV, int MAXT> __global__ void __launch_bounds__(MAXT, MAXT == 1024 ? 1 : 1024 / MAXT) layer_norm_cta_kernel(NormArgs a)
{
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ float red[2][64];
    pdl_wait();
    pdl_launch_dependents();
    const int t = threadIdx.x, tpr = blockDim.x, lane = t & 31, warp = t >> 5, warps = tpr >> 5;
    const long long rows = live_rows(a);
    const float inv = 1.f / (float)a.C;
    const T* x = static_cast<const T*>(a.x);
    const uint32_t rowBytes = NV * tpr * kSlotBytes<T, VE>, slots = smem_u32(dyn) + t * kSlotBytes<T, VE>;
    auto fetch = [&](long long row, uint32_t stage) {
        copy_row<T, VE, NV>(slots + stage * rowBytes, x + row * a.C, row < rows, t, tpr, a.C);
        copies_commit();
    };
#pragma unroll
    for (int i = 0; i < kAhead - 1; ++i)
        fetch(blockIdx.x + (long long)i * gridDim.x, i);
    F2 w[NV * VE / 2], b[NV * VE / 2];
    load_params<VE, NV>(w, a.weight, 1.f, a.wdtype, t, tpr, a.C);
    load_params<VE, NV>(b, a.bias, 0.f, a.wdtype, t, tpr, a.C);
    // channels of warp q: of each of the NV vectors, those of its 32 threads that the row reaches
    auto channels = [&](int q) {
        int n = 0;
#pragma unroll
        for (int k = 0; k < NV; ++k)
            n += min(max(a.C - (k * tpr + q * 32) * VE, 0), 32 * VE);
        return (float)n;
    };
    const float own = channels(warp), ownInv = own > 0.f ? 1.f / own : 0.f, laneCount = channels(lane & (warps - 1));
    uint32_t stage = 0;
    int flip = 0;
    for (long long row = blockIdx.x; row < rows; row += gridDim.x, flip ^= 1, stage = stage + 1 == kAhead ? 0 : stage + 1) {
        fetch(row + (kAhead - 1ll) * gridDim.x, stage == 0 ? kAhead - 1 : stage - 1);
        copies_wait();
        Pack<T, VE> v[NV];
        take_row<T, VE, NV>(v, slots + stage * rowBytes, x + row * a.C, true, t, tpr, a.C);
        F2 f[NV * VE / 2];
        const float m = group_sum(row_sum<T, VE, NV>(v, f), 32) * ownInv;
        const float q = group_sum(row_spread<VE, NV>(f, m, t, tpr, a.C), 32);
        if (lane == 0)
            red[flip][warp] = m, red[flip][32 + warp] = q;
        __syncthreads();
        const float mw = red[flip][lane & (warps - 1)], qw = red[flip][32 + (lane & (warps - 1))];
        const float mean = group_sum(mw * laneCount, warps) * inv;
        const float spread = group_sum(qw + laneCount * (mw - mean) * (mw - mean), warps);
        const float rstd = rsqrtf(spread * inv + a.eps);
        store_normed<T, VE, NV>(static_cast<T*>(a.y) + row * a.C, f, mean - m, rstd, w, b, t, tpr, a.C);
        if (t == 0 && a.mean != nullptr)
            a.mean[row] = mean, a.rstd[row] = rstd;
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
template <int E> __device__ __forceinline__ float element(const F2 (&v)[E / 2], int e)
{
    const float2 p = unpair(v[e / 2]);
    return e % 2 ? p.y : p.x;
}

// One row's products: adds to the column sums, keeps xh and gw, and returns sum(gw) and sum(gw * xh) of this thread's
// channels (g reads as zero past the row's end and for rows that are not there).
template <typename T, int VE, int NV>
__device__ __forceinline__ void grad_sums(const Pack<T, VE> (&xv)[NV], const Pack<T, VE> (&gv)[NV], float mean, float rstd,
                                          const F2 (&w)[NV * VE / 2], F2 (&dw)[NV * VE / 2], F2 (&db)[NV * VE / 2],
                                          F2 (&xh)[NV * VE / 2], F2 (&gw)[NV * VE / 2], float& s0, float& s1)
{
    const F2 m = f2(-mean, -mean), r = f2(rstd, rstd);
    F2 a0 = f2(0.f, 0.f), a1 = a0;
#pragma unroll
    for (int j = 0; j < NV * VE / 2; ++j) {
        const F2 gi = pair_of<T, VE, NV>(gv, j);
        xh[j] = mul2(add2(pair_of<T, VE, NV>(xv, j), m), r), gw[j] = mul2(gi, w[j]);
        dw[j] = fma2(gi, xh[j], dw[j]), db[j] = add2(db[j], gi);
        a0 = add2(a0, gw[j]), a1 = fma2(gw[j], xh[j], a1);
    }
    s0 = both(a0), s1 = both(a1);
}
template <typename T, int VE, int NV, bool FULL = false>
__device__ __forceinline__ void store_dx(T* dx, F2 (&xh)[NV * VE / 2], const F2 (&gw)[NV * VE / 2], float rstd, float m0, float m1,
                                         int t, int tpr, int C)
{
    const F2 r = f2(rstd, rstd), n0 = f2(-m0, -m0), n1 = f2(-m1, -m1);
#pragma unroll
    for (int j = 0; j < NV * VE / 2; ++j)
        xh[j] = mul2(r, fma2(xh[j], n1, add2(gw[j], n0)));
    store_pairs<T, VE, NV, FULL>(dx, xh, t, tpr, C);
}

template <typename T, int VE, int NV, int ROWS>
__global__ void __launch_bounds__(kWarpThreads, NV * VE == 8 ? kGradCtas : kGradCtas16) layer_norm_grad_warp_kernel(NormArgs a, int tpr)
{
    constexpr int E = NV * VE;
    extern __shared__ __align__(16) uint8_t dyn[];   // the slots, then [groups of the CTA][2][tpr * E] column sums
    float* cols = reinterpret_cast<float*>(dyn);
    pdl_wait();
    pdl_launch_dependents();
    const int t = threadIdx.x & (tpr - 1);
    const long long groups = (long long)gridDim.x * (kWarpThreads / tpr);
    const long long first = (long long)blockIdx.x * (kWarpThreads / tpr) + threadIdx.x / tpr;
    const float inv = 1.f / (float)a.C;
    const T *x = static_cast<const T*>(a.x), *g = static_cast<const T*>(a.g);
    constexpr int rowBytes = NV * kWarpThreads * kSlotBytes<T, VE>;
    const uint32_t slots = smem_u32(dyn) + threadIdx.x * kSlotBytes<T, VE>;
    const long long turns = (a.rows + groups * ROWS - 1) / (groups * ROWS);
    float meanNext[ROWS], rstdNext[ROWS];
    auto fetch = [&](auto full, long long turn, uint32_t stage) {
        constexpr bool FULL = decltype(full)::value;
        const uint32_t at = slots + stage * 2 * ROWS * rowBytes;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const long long row = (turn * ROWS + r) * groups + first;
            copy_row<T, VE, NV, FULL>(at + 2 * r * rowBytes, x + row * a.C, row < a.rows, t, tpr, a.C);
            copy_row<T, VE, NV, FULL>(at + (2 * r + 1) * rowBytes, g + row * a.C, row < a.rows, t, tpr, a.C);
        }
        copies_commit();
    };
    auto stats = [&](long long turn) {      // of the next turn: their latency passes behind this one's work
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const long long row = (turn * ROWS + r) * groups + first;
            meanNext[r] = row < a.rows ? a.mean[row] : 0.f, rstdNext[r] = row < a.rows ? a.rstd[row] : 0.f;
        }
    };
#pragma unroll
    for (int i = 0; i < kAhead - 1; ++i)
        fetch(std::false_type(), i, i);
    stats(0);
    F2 w[E / 2], dw[E / 2] = {}, db[E / 2] = {};
    load_params<VE, NV>(w, a.weight, 1.f, a.wdtype, t, tpr, a.C);
    uint32_t stage = 0;
    auto body = [&](auto full, long long turn) {
        constexpr bool FULL = decltype(full)::value;
        const long long row0 = turn * ROWS * groups + first;
        fetch(full, turn + kAhead - 1, stage == 0 ? kAhead - 1 : stage - 1);
        float mean[ROWS], rstd[ROWS], s0[ROWS], s1[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
            mean[r] = meanNext[r], rstd[r] = rstdNext[r];
        stats(turn + 1);
        copies_wait();
        const uint32_t at = slots + stage * 2 * ROWS * rowBytes;
        F2 xh[ROWS][E / 2], gw[ROWS][E / 2];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const long long row = row0 + r * groups;
            Pack<T, VE> xv[NV], gv[NV];
            take_row<T, VE, NV, FULL>(xv, at + 2 * r * rowBytes, x + row * a.C, row < a.rows, t, tpr, a.C);
            take_row<T, VE, NV, FULL>(gv, at + (2 * r + 1) * rowBytes, g + row * a.C, row < a.rows, t, tpr, a.C);
            grad_sums<T, VE, NV>(xv, gv, mean[r], rstd[r], w, dw, db, xh[r], gw[r], s0[r], s1[r]);
        }
        for (int m = tpr >> 1; m > 0; m >>= 1)
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                s0[r] += __shfl_xor_sync(0xffffffffu, s0[r], m);
                s1[r] += __shfl_xor_sync(0xffffffffu, s1[r], m);
            }
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const long long row = row0 + r * groups;
            if (FULL || row < a.rows)
                store_dx<T, VE, NV, FULL>(static_cast<T*>(a.y) + row * a.C, xh[r], gw[r], rstd[r], s0[r] * inv, s1[r] * inv, t, tpr, a.C);
        }
        stage = stage + 1 == kAhead ? 0 : stage + 1;
    };
    long long turn = 0;
    if (tpr * E == a.C)
        for (; turn + kAhead < turns; ++turn)
            body(std::true_type(), turn);
    for (; turn < turns; ++turn)
        body(std::false_type(), turn);
    // no copy is in flight into the slots that the sums go over: the last ones issued had no row
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    if (a.partials == nullptr)
        return;
    float* pw = a.partials + (long long)blockIdx.x * 2 * a.C;
    const int inCta = kWarpThreads / tpr, grp = threadIdx.x / tpr, width = tpr * E;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < VE; ++i) {
            const int c = (k * tpr + t) * VE + i;
            cols[(grp * 2 + 0) * width + c] = element<E>(dw, k * VE + i);
            cols[(grp * 2 + 1) * width + c] = element<E>(db, k * VE + i);
        }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * a.C; c += kWarpThreads) {
        const int half = c >= a.C, cc = c - half * a.C;
        float s = 0.f;
        for (int q = 0; q < inCta; ++q)
            s += cols[(q * 2 + half) * width + cc];
        pw[c] = s;
    }
}

// Rows that share a barrier: two, or what shared memory holds.
template <typename T, int MAXT> constexpr int kCtaRows = sizeof(T) == 4 && MAXT == 1024 ? 1 : 2;

// The whole CTA shares a row; two rows at a time share a barrier.  Their products are computed twice, before and after
// it, from the copies in shared memory: two rows of them would not fit the registers beside w, dw and db.
template <typename T, int VE, int NV, int MAXT> __global__ void __launch_bounds__(MAXT, MAXT == 256 ? 2 : 1) layer_norm_grad_cta_kernel(NormArgs a)
{
    constexpr int E = NV * VE, ROWS = kCtaRows<T, MAXT>;
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ float red[2][64 * ROWS];
    pdl_wait();
    pdl_launch_dependents();
    const int t = threadIdx.x, tpr = blockDim.x;
    const float inv = 1.f / (float)a.C;
    const T *x = static_cast<const T*>(a.x), *g = static_cast<const T*>(a.g);
    const uint32_t rowBytes = NV * tpr * kSlotBytes<T, VE>, slots = smem_u32(dyn) + t * kSlotBytes<T, VE>;
    float meanNext[ROWS], rstdNext[ROWS];
    auto fetch = [&](long long row0, uint32_t stage) {
        const uint32_t at = slots + stage * 2 * ROWS * rowBytes;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const long long row = row0 + (long long)r * gridDim.x;
            copy_row<T, VE, NV>(at + 2 * r * rowBytes, x + row * a.C, row < a.rows, t, tpr, a.C);
            copy_row<T, VE, NV>(at + (2 * r + 1) * rowBytes, g + row * a.C, row < a.rows, t, tpr, a.C);
        }
        copies_commit();
    };
    auto stats = [&](long long row0) {
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const long long row = row0 + (long long)r * gridDim.x;
            meanNext[r] = row < a.rows ? a.mean[row] : 0.f, rstdNext[r] = row < a.rows ? a.rstd[row] : 0.f;
        }
    };
    const long long step = (long long)ROWS * gridDim.x;
#pragma unroll
    for (int i = 0; i < kAheadCta - 1; ++i)
        fetch(blockIdx.x + i * step, i);
    stats(blockIdx.x);
    F2 w[E / 2], dw[E / 2] = {}, db[E / 2] = {};
    load_params<VE, NV>(w, a.weight, 1.f, a.wdtype, t, tpr, a.C);
    uint32_t stage = 0;
    int flip = 0;
    for (long long row0 = blockIdx.x; row0 < a.rows; row0 += step, flip ^= 1, stage = stage + 1 == kAheadCta ? 0 : stage + 1) {
        fetch(row0 + (kAheadCta - 1) * step, stage == 0 ? kAheadCta - 1 : stage - 1);
        float mean[ROWS], rstd[ROWS], s[2 * ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
            mean[r] = meanNext[r], rstd[r] = rstdNext[r];
        stats(row0 + step);
        asm volatile("cp.async.wait_group %0;" ::"n"(kAheadCta - 1) : "memory");
        const uint32_t at = slots + stage * 2 * ROWS * rowBytes;
        Pack<T, VE> xv[NV], gv[NV];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const long long row = row0 + (long long)r * gridDim.x;
            take_row<T, VE, NV>(xv, at + 2 * r * rowBytes, x + row * a.C, row < a.rows, t, tpr, a.C);
            take_row<T, VE, NV>(gv, at + (2 * r + 1) * rowBytes, g + row * a.C, row < a.rows, t, tpr, a.C);
            F2 xh[E / 2], gw[E / 2];
            grad_sums<T, VE, NV>(xv, gv, mean[r], rstd[r], w, dw, db, xh, gw, s[2 * r], s[2 * r + 1]);
        }
        cta_sum(s, red[flip]);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const long long row = row0 + (long long)r * gridDim.x;
            if (row >= a.rows)
                continue;
            take_row<T, VE, NV>(xv, at + 2 * r * rowBytes, x + row * a.C, true, t, tpr, a.C);
            take_row<T, VE, NV>(gv, at + (2 * r + 1) * rowBytes, g + row * a.C, true, t, tpr, a.C);
            F2 xh[E / 2], gw[E / 2];
            const F2 m = f2(-mean[r], -mean[r]), rs = f2(rstd[r], rstd[r]);
#pragma unroll
            for (int j = 0; j < E / 2; ++j)
                xh[j] = mul2(add2(pair_of<T, VE, NV>(xv, j), m), rs), gw[j] = mul2(pair_of<T, VE, NV>(gv, j), w[j]);
            store_dx<T, VE, NV>(static_cast<T*>(a.y) + row * a.C, xh, gw, rstd[r], s[2 * r] * inv, s[2 * r + 1] * inv, t, tpr, a.C);
        }
    }
    if (a.partials == nullptr)
        return;
    float* pw = a.partials + (long long)blockIdx.x * 2 * a.C;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < VE; ++i) {
            const int c = (k * tpr + t) * VE + i;
            if (c < a.C)
                pw[c] = element<E>(dw, k * VE + i), pw[a.C + c] = element<E>(db, k * VE + i);
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

// Up to 512 channels a row stays inside a warp, 16 channels a thread where that leaves at least 8 threads a row (fewer
// exchanges per channel); in the backward pass the column sums leave registers for 8 up to 256 channels.  Then whole
// CTAs: in 16-byte vectors 16 a thread (40 M elements of 1,024 channels in bf16, against 8 a thread: forward 43 -> 39 us,
// backward 57 -> 54), in narrower ones 8 up to 2,048 channels (20,011 x 1,001 fp32 forward: 46 us against 82 with 16).
// fp32 rows, whose copies take twice the shared memory, keep 8 in the backward pass.
NormShape pick(int C, int itemsize, uintptr_t bits, bool grad)
{
    NormShape s = {itemsize, 0, 0, false};
    const uintptr_t all = bits | (uintptr_t)((long long)C * itemsize);
    if ((all & 15) == 0)
        s.vecBytes = 16;
    else if (itemsize == 2 && (all & 3) == 0)
        s.vecBytes = 4;
    if (C <= 512) {
        s.elems = C <= (grad ? 256 : 64) ? 8 : 16;
        s.tpr = 4;
        while (s.tpr * s.elems < C)
            s.tpr *= 2;
    } else if (C <= (grad ? 8192 : 16384)) {   // backward: what shared memory holds
        s.cta = true;
        s.elems = (grad && itemsize == 4) || (s.vecBytes != 16 && C <= 2048) ? 8 : 16;
        s.tpr = 64;
        while (s.tpr * s.elems < C)
            s.tpr *= 2;
    }
    return s;
}

template <typename T, int VE, int NV, int MAXT> cudaError_t launch_fwd_cta(const NormArgs& a, const NormShape& s, cudaStream_t stream)
{
    auto kernel = layer_norm_cta_kernel<T, VE, NV, MAXT>;
    static std::atomic<bool> done[64] = {};
    if (cudaError_t e = allow_smem(kernel, slots_bytes<T, VE, NV>(MAXT, 1), done))
        return e;
    const int smem = slots_bytes<T, VE, NV>(s.tpr, 1);
    const long long grid = std::min<long long>(a.rows, (long long)sm_count() * (1024 / s.tpr));
    return launch_pdl(kernel, dim3((unsigned)grid), dim3(s.tpr), smem, stream, a);
}

template <typename T, int VE, int NV> cudaError_t launch_fwd(const NormArgs& a, const NormShape& s, cudaStream_t stream)
{
    constexpr int E = VE * NV;
    if (s.cta) {
        if constexpr (E == 16)
            return s.tpr <= 512 ? launch_fwd_cta<T, VE, NV, 512>(a, s, stream) : launch_fwd_cta<T, VE, NV, 1024>(a, s, stream);
        else if constexpr (VE * sizeof(T) != 16)
            return launch_fwd_cta<T, VE, NV, 256>(a, s, stream);
        return cudaErrorInvalidValue;    // no shape that pick() makes
    }
    // one row a group while that leaves SMs empty, two in flight per group and turn otherwise
    const long long ctas = (a.rows * s.tpr + kWarpThreads - 1) / kWarpThreads;
    const long long grid = std::min<long long>(ctas, (long long)sm_count() * kFwdCtas);
    if (ctas <= (long long)sm_count() * kFwdCtas) {
        auto kernel = layer_norm_warp_kernel<T, VE, NV, 1>;
        static std::atomic<bool> done[64] = {};
        constexpr int smem = slots_bytes<T, VE, NV>(kWarpThreads, 1);
        if (cudaError_t e = allow_smem(kernel, smem, done))
            return e;
        return launch_pdl(kernel, dim3((unsigned)grid), dim3(kWarpThreads), smem, stream, a, s.tpr);
    }
    constexpr int ROWS = sizeof(T) == 4 && E == 16 ? 1 : 2;     // 48 KB of slots a CTA
    auto kernel = layer_norm_warp_kernel<T, VE, NV, ROWS>;
    static std::atomic<bool> done[64] = {};
    constexpr int smem = slots_bytes<T, VE, NV>(kWarpThreads, ROWS);
    if (cudaError_t e = allow_smem(kernel, smem, done))
        return e;
    return launch_pdl(kernel, dim3((unsigned)grid), dim3(kWarpThreads), smem, stream, a, s.tpr);
}

template <typename T, int VE, int NV, int MAXT>
cudaError_t launch_bwd_cta(const NormArgs& a, const NormShape& s, int grid, cudaStream_t stream)
{
    auto kernel = layer_norm_grad_cta_kernel<T, VE, NV, MAXT>;
    static std::atomic<bool> done[64] = {};
    constexpr int perThread = kAheadCta * 2 * kCtaRows<T, MAXT> * NV * kSlotBytes<T, VE>;
    if (cudaError_t e = allow_smem(kernel, perThread * MAXT, done))
        return e;
    const int smem = perThread * s.tpr;
    return launch_pdl(kernel, dim3(grid), dim3(s.tpr), smem, stream, a);
}

template <typename T, int VE, int NV> cudaError_t launch_bwd(const NormArgs& a, const NormShape& s, int grid, cudaStream_t stream)
{
    constexpr int E = VE * NV;
    if (s.cta) {
        if constexpr (E == 8 && sizeof(T) == 4)
            return s.tpr <= 256   ? launch_bwd_cta<T, VE, NV, 256>(a, s, grid, stream)
                   : s.tpr <= 512 ? launch_bwd_cta<T, VE, NV, 512>(a, s, grid, stream)
                                  : launch_bwd_cta<T, VE, NV, 1024>(a, s, grid, stream);
        else if constexpr (E == 16 && sizeof(T) == 2)
            return launch_bwd_cta<T, VE, NV, 512>(a, s, grid, stream);
        else if constexpr (E == 8 && VE < 8)
            return launch_bwd_cta<T, VE, NV, 256>(a, s, grid, stream);
        return cudaErrorInvalidValue;    // no shape that pick() makes
    }
    constexpr int ROWS = E == 8 && sizeof(T) == 2 ? 2 : 1;
    auto kernel = layer_norm_grad_warp_kernel<T, VE, NV, ROWS>;
    static std::atomic<bool> done[64] = {};
    constexpr int smem = std::max(slots_bytes<T, VE, NV>(kWarpThreads, 2 * ROWS), (int)sizeof(float) * 2 * kWarpThreads * E);
    if (cudaError_t e = allow_smem(kernel, smem, done))
        return e;
    return launch_pdl(kernel, dim3(grid), dim3(kWarpThreads), smem, stream, a, s.tpr);
}

template <typename T> cudaError_t run_fwd(const NormArgs& a, cudaStream_t stream)
{
    const NormShape s = pick(a.C, sizeof(T), reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y), false);
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
                                                 reinterpret_cast<uintptr_t>(a.g), true);
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

// CTAs of the backward kernel (about 512 threads an SM, all resident) = partial rows of the column sums.  Depends on
// the sizes only.
static int grad_parts(long long rows, int C, int itemsize, uintptr_t bits)
{
    const NormShape s = pick(C, itemsize, bits, true);
    if (s.tpr == 0)
        return (int)std::min<long long>(rows, sm_count());
    if (s.cta)
        return (int)std::min<long long>(rows, (long long)sm_count() * std::max(1, 512 / s.tpr));
    return (int)std::min<long long>((rows * s.tpr + kWarpThreads - 1) / kWarpThreads, (long long)sm_count() * (s.elems == 8 ? kGradCtas : kGradCtas16));
}

// The most that any element type and alignment asks for.
int layer_norm_grad_parts(long long rows, int C)
{
    return std::max(std::max(grad_parts(rows, C, 2, 0), grad_parts(rows, C, 4, 0)), std::max(grad_parts(rows, C, 2, 1), grad_parts(rows, C, 4, 1)));
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
    const int parts = grad_parts(a.rows, a.C, dtype == 0 ? 4 : 2, reinterpret_cast<uintptr_t>(a.x) |
                                 reinterpret_cast<uintptr_t>(a.y) | reinterpret_cast<uintptr_t>(a.g));
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
