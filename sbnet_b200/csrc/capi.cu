// The C ABI (include/sbnet_b200.h): argument checks the reference performs in its OpKernels
// (sbnet_ops/reduce_mask.cc:132-138, sbnet_ops/sparse_gather.cc:164,173,322-327), then the launch.
#include <limits.h>
#include <stdarg.h>
#include <stdio.h>
#include <sched.h>
#include <time.h>

#include "../../include/sbnet_b200.h"
#include <stdlib.h>
#include <string.h>

#include <mutex>

#include "common.cuh"
#include "kernels.h"
#include "options.h"

#define SBNET_EXPORT extern "C" __attribute__((visibility("default")))

namespace {

thread_local char g_err[320] = "";
thread_local const char* g_site = "";
constexpr int32_t kCountSentinel = SBNET_COUNT_PENDING;

int reject(int code, const char* fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
    return code;
}

inline int cuda_status(cudaError_t e)
{
    if (e != cudaSuccess)
        snprintf(g_err, sizeof(g_err), "CUDA error %d: %s%s%s", (int)e, cudaGetErrorString(e), g_site[0] ? " at " : "",
                 g_site);
    return (int)e;
}

// Geometry limits shared by all ops: positive sizes/strides and every pixel coordinate inside 31 bits.
int check_geometry(const char* op, int bOffsH, int bOffsW, int bSzH, int bSzW, int bStrH, int bStrW,
                   long long maxBlockH, long long maxBlockW)
{
    if (bSzH < 1 || bSzW < 1)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: block size must be positive, got [%d, %d]", op,
                      bSzH, bSzW);
    if (bStrH < 1 || bStrW < 1)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: block stride must be positive, got [%d, %d]",
                      op, bStrH, bStrW);
    const long long lim = 1ll << 30;
    const long long absH = bOffsH < 0 ? -(long long)bOffsH : bOffsH;
    const long long absW = bOffsW < 0 ? -(long long)bOffsW : bOffsW;
    if (absH + maxBlockH * bStrH + bSzH >= lim || absW + maxBlockW * bStrW + bSzW >= lim ||
        (long long)bSzH * bSzW >= lim)
        return reject(SBNET_ERR_UNSUPPORTED, "%s: block geometry exceeds 2^30 pixels", op);
    return SBNET_OK;
}

int blocks_call(const char* op, int mode, int dtype, int N, int H, int W, int C,
                void* image, void* stack, int bOffsH, int bOffsW, int bSzH, int bSzW, int bStrH,
                int bStrW, int numActive, const int32_t* numActiveDev, const int16_t* idx,
                int transpose, void* stream)
{
    g_site = "";
    if (dtype != SBNET_F32 && dtype != SBNET_F16 && dtype != SBNET_BF16)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d", op, dtype);
    if (N < 1 || H < 1 || W < 1 || C < 1)
        return reject(SBNET_ERR_INVALID_ARGUMENT,
                      "%s: tensor must be rank 4 with positive dimensions, got [%d, %d, %d, %d]", op,
                      N, H, W, C);
    if (numActive < 0)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: negative block count %d", op, numActive);
    if (int rc = check_geometry(op, bOffsH, bOffsW, bSzH, bSzW, bStrH, bStrW, 32767, 32767))
        return rc;
    if (numActive == 0)
        return SBNET_OK;
    if (image == nullptr || stack == nullptr || idx == nullptr)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: null tensor pointer", op);
    // a pointer off its element's boundary would be a misaligned access on the device, not an error code
    const uintptr_t elem = dtype == SBNET_F32 ? 4 : 2;
    if (((reinterpret_cast<uintptr_t>(image) | reinterpret_cast<uintptr_t>(stack)) & (elem - 1)) != 0 ||
        (reinterpret_cast<uintptr_t>(idx) & 1) != 0 || (reinterpret_cast<uintptr_t>(numActiveDev) & 3) != 0)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: tensor pointer not aligned to its element size", op);
    const long long lim = 1ll << 31;
    const long long blockElems = (long long)bSzH * bSzW * C;
    const long long chunks = ((long long)C * 4 + 127) / 128;
    if (blockElems >= lim || (long long)numActive * bSzH >= lim ||
        (long long)numActive * chunks * ((long long)bSzH * bSzW / 128 + 1) >= lim)
        return reject(SBNET_ERR_UNSUPPORTED, "%s: more than 2^31 work items", op);

    sbnet::BlockArgs a;
    a.image = image, a.stack = stack, a.idx = idx, a.num_active_dev = numActiveDev;
    a.numActive = numActive, a.N = N, a.H = H, a.W = W, a.C = C;
    a.bOffsH = bOffsH, a.bOffsW = bOffsW, a.bSzH = bSzH, a.bSzW = bSzW, a.bStrH = bStrH,
    a.bStrW = bStrW;
    return cuda_status(sbnet::launch_blocks(a, dtype, mode, transpose != 0, (cudaStream_t)stream));
}

int scatter_mode(const char* op, int add, int atomic, int bSzH, int bSzW, int bStrH, int bStrW,
                 int* mode)
{
    if (add && !atomic && !(bStrH >= bSzH && bStrW >= bSzW))
        return reject(SBNET_ERR_INVALID_ARGUMENT,
                      "%s: Only non-overlapping blocks are supported with add=True, atomic=False", op);
    *mode = !add ? sbnet::kScatterSet : (atomic ? sbnet::kScatterAtomic : sbnet::kScatterAdd);
    return SBNET_OK;
}

} // namespace

namespace sbnet {
// Lets other translation units of the library report through sbnet_last_error().
void set_last_error(const char* text) { snprintf(g_err, sizeof(g_err), "%s", text); }
void note_site(const char* site) { g_site = site; }

static int env_number(const char* name, int dflt)
{
    const char* v = getenv(name);
    return (v && *v) ? atoi(v) : dflt;
}

Options& options()
{
    static Options opt;
    static std::once_flag once;
    std::call_once(once, [] {
        const char* planes = getenv("SBNET_PLANES");
        opt.planes = (planes && planes[0] == 't') ? (planes[1] == 'i' ? 2 : 1) : env_number("SBNET_PLANES", 0);   // tma | tile | 0..5
        opt.disableTma = env_number("SBNET_DISABLE_TMA", 0) == 1;
        opt.tileBlocks = env_number("SBNET_TILE_BLOCKS", 0);
        opt.rmKernel = env_number("SBNET_RM_KERNEL", 0);
        opt.rmCtasPerSm = env_number("SBNET_RM_CTAS_PER_SM", 8);
        opt.rmResident = env_number("SBNET_RM_RESIDENT", 0);
        opt.pdl = env_number("SBNET_PDL", 1);
        opt.tmaL2 = env_number("SBNET_TMA_L2", 3);
    });
    return opt;
}
} // namespace sbnet

namespace {
struct OptionName {
    const char* name;
    int sbnet::Options::*field;
};
const OptionName kOptionNames[] = {
    {"planes", &sbnet::Options::planes},          {"disable_tma", &sbnet::Options::disableTma},
    {"tile_blocks", &sbnet::Options::tileBlocks}, {"rm_kernel", &sbnet::Options::rmKernel},
    {"rm_ctas_per_sm", &sbnet::Options::rmCtasPerSm}, {"pdl", &sbnet::Options::pdl},
    {"rm_resident", &sbnet::Options::rmResident},
    {"tma_l2", &sbnet::Options::tmaL2},
};
} // namespace

SBNET_EXPORT int sbnet_set_option(const char* name, int value)
{
    for (const OptionName& o : kOptionNames)
        if (name != nullptr && strcmp(name, o.name) == 0) {
            sbnet::options().*(o.field) = value;
            return SBNET_OK;
        }
    return reject(SBNET_ERR_INVALID_ARGUMENT, "sbnet_set_option: unknown option '%s'", name ? name : "(null)");
}

SBNET_EXPORT int sbnet_get_option(const char* name, int* value)
{
    for (const OptionName& o : kOptionNames)
        if (name != nullptr && value != nullptr && strcmp(name, o.name) == 0) {
            *value = sbnet::options().*(o.field);
            return SBNET_OK;
        }
    return reject(SBNET_ERR_INVALID_ARGUMENT, "sbnet_get_option: unknown option '%s'", name ? name : "(null)");
}

SBNET_EXPORT int sbnet_version(void) { return 100; }

SBNET_EXPORT const char* sbnet_last_error(void) { return g_err; }

SBNET_EXPORT int sbnet_reduce_mask(const float* mask, int N, int H, int W, float tol, int avgpool,
                                   int bOffsH, int bOffsW, int bSzH, int bSzW, int bStrH, int bStrW,
                                   int bCntH, int bCntW, int16_t* active_block_indices,
                                   int32_t* scratch_dev, int32_t* count_host, int flags,
                                   void* stream)
{
    const char* op = "ReduceMask";
    if (N < 1 || H < 1 || W < 1)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: mask must be [N,H,W,1] with positive dimensions, "
                      "got [%d, %d, %d]", op, N, H, W);
    if (bCntH < 1 || bCntW < 1)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: block counts must be positive, got [%d, %d]", op,
                      bCntH, bCntW);
    if (N > 32767 || bCntH > 32767 || bCntW > 32767)
        return reject(SBNET_ERR_INVALID_ARGUMENT,
                      "%s: N, bCntH and bCntW must fit the int16 index triples (<= 32767), got %d, %d, %d",
                      op, N, bCntH, bCntW);
    if ((long long)N * bCntH * bCntW >= (1ll << 31))
        return reject(SBNET_ERR_UNSUPPORTED, "%s: N*bCntH*bCntW = %lld candidate blocks do not fit the int32 count",
                      op, (long long)N * bCntH * bCntW);
    if (int rc = check_geometry(op, bOffsH, bOffsW, bSzH, bSzW, bStrH, bStrW, bCntH, bCntW))
        return rc;
    if (mask == nullptr || active_block_indices == nullptr || scratch_dev == nullptr)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: null tensor pointer", op);
    if (reinterpret_cast<uintptr_t>(scratch_dev) & 15)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: scratch_dev must be 16-byte aligned", op);
    if ((reinterpret_cast<uintptr_t>(mask) & 3) != 0 || (reinterpret_cast<uintptr_t>(active_block_indices) & 1) != 0)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: tensor pointer not aligned to its element size", op);

    cudaStream_t s = (cudaStream_t)stream;
    int32_t* hostDev = nullptr;   // device-visible alias of count_host when it is pinned
    if (count_host != nullptr) {
        cudaPointerAttributes attr;
        if (cudaPointerGetAttributes(&attr, count_host) == cudaSuccess &&
            attr.type == cudaMemoryTypeHost && attr.devicePointer != nullptr)
            hostDev = static_cast<int32_t*>(attr.devicePointer);
        else
            (void)cudaGetLastError();
    }
    if ((flags & SBNET_COUNT_NOWAIT) && hostDev == nullptr)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: SBNET_COUNT_NOWAIT needs count_host in pinned host memory", op);
    if (hostDev != nullptr && (flags & (SBNET_COUNT_POLL | SBNET_COUNT_NOWAIT)))
        *count_host = kCountSentinel;
    if (!(flags & SBNET_SCRATCH_CLEAN))
        if (cudaError_t e = cudaMemsetAsync(scratch_dev, 0, sizeof(int32_t) * SBNET_REDUCE_MASK_SCRATCH_INTS, s))
            return cuda_status(e);
    if (cudaError_t e = sbnet::launch_reduce_mask(mask, N, H, W, tol, avgpool != 0, bOffsH, bOffsW, bSzH,
                                                  bSzW, bStrH, bStrW, bCntH, bCntW,
                                                  active_block_indices, scratch_dev, hostDev,
                                                  (flags & SBNET_MASK_STABLE) != 0, s))
        return cuda_status(e);
    if (count_host != nullptr && !(flags & SBNET_COUNT_NOWAIT)) {
        if (hostDev != nullptr && (flags & SBNET_COUNT_POLL)) {
            // The kernel stores the count straight into pinned memory: watching that word is several
            // times quicker than putting the thread to sleep in a stream synchronisation.  A count is
            // never negative, so the sentinel written before the launch cannot be mistaken for one.
            volatile int32_t* word = count_host;
            timespec t0;
            clock_gettime(CLOCK_MONOTONIC, &t0);
            const bool yield = (flags & SBNET_COUNT_YIELD) != 0;
            for (unsigned spins = 0; *word == kCountSentinel; ++spins) {
                if (yield)
                    sched_yield();   // several such threads (one per GPU) may share this core
                if (yield || (spins & 1023u) == 1023u) {
                    timespec t1;
                    clock_gettime(CLOCK_MONOTONIC, &t1);
                    if ((t1.tv_sec - t0.tv_sec) * 1000000000ll + (t1.tv_nsec - t0.tv_nsec) > 200000000ll)
                        break;   // 0.2 s: let the runtime wait (and report a failed launch, if any)
                }
            }
            if (*word != kCountSentinel)
                return SBNET_OK;
        }
        if (hostDev == nullptr)
            if (cudaError_t e = cudaMemcpyAsync(count_host, scratch_dev, sizeof(int32_t),
                                                cudaMemcpyDeviceToHost, s))
                return cuda_status(e);
        if (cudaError_t e = cudaStreamSynchronize(s))
            return cuda_status(e);
    }
    return SBNET_OK;
}

SBNET_EXPORT int sbnet_sparse_gather(const void* x, int dtype, int N, int H, int W, int C, void* y,
                                     int bOffsH, int bOffsW, int bSzH, int bSzW, int bStrH,
                                     int bStrW, int numActive, const int16_t* active_block_indices,
                                     int transpose, void* stream)
{
    return blocks_call("SparseGather", sbnet::kGather, dtype, N, H, W, C, const_cast<void*>(x), y,
                       bOffsH, bOffsW, bSzH, bSzW, bStrH, bStrW, numActive, nullptr,
                       active_block_indices, transpose, stream);
}

SBNET_EXPORT int sbnet_sparse_gather_dyn(const void* x, int dtype, int N, int H, int W, int C,
                                         void* y, int bOffsH, int bOffsW, int bSzH, int bSzW,
                                         int bStrH, int bStrW, int maxActive,
                                         const int32_t* num_active_dev,
                                         const int16_t* active_block_indices, int transpose,
                                         void* stream)
{
    if (num_active_dev == nullptr)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "SparseGather: num_active_dev is null");
    return blocks_call("SparseGather", sbnet::kGather, dtype, N, H, W, C, const_cast<void*>(x), y,
                       bOffsH, bOffsW, bSzH, bSzW, bStrH, bStrW, maxActive, num_active_dev,
                       active_block_indices, transpose, stream);
}

SBNET_EXPORT int sbnet_sparse_scatter(const void* x, int dtype, int N, int H, int W, int C, void* y,
                                      int bOffsH, int bOffsW, int bSzH, int bSzW, int bStrH,
                                      int bStrW, int numActive, const int16_t* active_block_indices,
                                      int add, int transpose, int atomic, void* stream)
{
    int mode = 0;
    if (int rc = scatter_mode("SparseScatter", add, atomic, bSzH, bSzW, bStrH, bStrW, &mode))
        return rc;
    return blocks_call("SparseScatter", mode, dtype, N, H, W, C, y, const_cast<void*>(x), bOffsH,
                       bOffsW, bSzH, bSzW, bStrH, bStrW, numActive, nullptr, active_block_indices,
                       transpose, stream);
}

SBNET_EXPORT int sbnet_sparse_scatter_dyn(const void* x, int dtype, int N, int H, int W, int C,
                                          void* y, int bOffsH, int bOffsW, int bSzH, int bSzW,
                                          int bStrH, int bStrW, int maxActive,
                                          const int32_t* num_active_dev,
                                          const int16_t* active_block_indices, int add,
                                          int transpose, int atomic, void* stream)
{
    int mode = 0;
    if (num_active_dev == nullptr)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "SparseScatter: num_active_dev is null");
    if (int rc = scatter_mode("SparseScatter", add, atomic, bSzH, bSzW, bStrH, bStrW, &mode))
        return rc;
    return blocks_call("SparseScatter", mode, dtype, N, H, W, C, y, const_cast<void*>(x), bOffsH,
                       bOffsW, bSzH, bSzW, bStrH, bStrW, maxActive, num_active_dev,
                       active_block_indices, transpose, stream);
}

SBNET_EXPORT int sbnet_copy_tensor(void* dst, const void* src, size_t bytes, void* stream)
{
    if (bytes != 0 && (dst == nullptr || src == nullptr))
        return reject(SBNET_ERR_INVALID_ARGUMENT, "CopyTensor: null pointer");
    return cuda_status(sbnet::launch_copy(dst, src, bytes, (cudaStream_t)stream));
}

SBNET_EXPORT int sbnet_cuda_timer_start(int64_t* handle)
{
    if (handle == nullptr)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "CudaTimerStart: null handle");
    cudaEvent_t ev;
    if (cudaError_t e = cudaEventCreate(&ev))
        return cuda_status(e);
    if (cudaError_t e = cudaEventRecord(ev, 0)) {
        cudaEventDestroy(ev);
        return cuda_status(e);
    }
    *handle = (int64_t)reinterpret_cast<intptr_t>(ev);
    return SBNET_OK;
}

SBNET_EXPORT int sbnet_cuda_timer_end(int64_t handle, float* elapsed_ms)
{
    if (handle == 0 || elapsed_ms == nullptr)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "CudaTimerEnd: null handle or output");
    cudaEvent_t start = reinterpret_cast<cudaEvent_t>((intptr_t)handle), stop;
    if (cudaError_t e = cudaEventCreate(&stop))
        return cuda_status(e);
    cudaError_t e = cudaEventRecord(stop, 0);
    if (e == cudaSuccess)
        e = cudaEventSynchronize(stop);
    if (e == cudaSuccess)
        e = cudaEventElapsedTime(elapsed_ms, start, stop);
    cudaEventDestroy(stop);
    cudaEventDestroy(start);
    return cuda_status(e);
}

SBNET_EXPORT int sbnet_wait_timeouts(unsigned int* count)
{
    if (count == nullptr)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "sbnet_wait_timeouts: null output");
    unsigned int planes = 0, mask = 0, rows = 0, ffn = 0;
    if (cudaError_t e = sbnet::read_wait_timeouts(&planes))
        return cuda_status(e);
    if (cudaError_t e = sbnet::read_rm_wait_timeouts(&mask))
        return cuda_status(e);
    if (cudaError_t e = sbnet::read_rows_wait_timeouts(&rows))
        return cuda_status(e);
    if (cudaError_t e = sbnet::read_ffn_wait_timeouts(&ffn))
        return cuda_status(e);
    *count = planes + mask + rows + ffn;
    return SBNET_OK;
}

namespace {
bool known_dtype(int dtype) { return dtype == SBNET_F32 || dtype == SBNET_F16 || dtype == SBNET_BF16; }
uintptr_t address(const void* p) { return reinterpret_cast<uintptr_t>(p); }
uintptr_t elem_mask(int dtype) { return dtype == SBNET_F32 ? 3 : 1; }

// Memory of a call: nothing where p is null.
struct Span {
    const void* p;
    size_t n;
    bool meets(const Span& o) const
    {
        return p != nullptr && o.p != nullptr && address(p) < address(o.p) + o.n && address(o.p) < address(p) + n;
    }
};
// Whether one of `out` overlaps one of `in` or another of `out`: what one block writes another reads or writes too.
template <size_t O, size_t I> bool overlap(const Span (&out)[O], const Span (&in)[I])
{
    for (size_t o = 0; o < O; ++o) {
        for (const Span& i : in)
            if (out[o].meets(i))
                return true;
        for (size_t q = 0; q < o; ++q)
            if (out[o].meets(out[q]))
                return true;
    }
    return false;
}

// Rules shared by the row operators: types, sizes (row counts and element counts are 64-bit).
int check_rows(const char* op, int dtype, int64_t rows, int C)
{
    if (!known_dtype(dtype))
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d", op, dtype);
    if (rows < 0 || C < 1)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: needs rows >= 0 and at least one channel, got [%lld, %d]", op,
                      (long long)rows, C);
    if (C > (1 << 24) || rows > (1ll << 40) / C)
        return reject(SBNET_ERR_UNSUPPORTED, "%s: more than 2^24 channels or 2^40 elements", op);
    return SBNET_OK;
}

int norm_call(const void* x, int dtype, int64_t rows, int rowsPerBlock, const int32_t* num_blocks_dev, int C,
              const void* weight, const void* bias, int wdtype, float eps, void* y, float* mean, float* rstd, void* stream)
{
    const char* op = "LayerNorm";
    g_site = "";
    if (int rc = check_rows(op, dtype, rows, C))
        return rc;
    if ((weight != nullptr || bias != nullptr) && wdtype != dtype && wdtype != SBNET_F32)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: weight and bias must share the tensor's dtype or be fp32", op);
    if (!(eps >= 0.f))
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: eps must not be negative", op);
    if ((mean == nullptr) != (rstd == nullptr))
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: mean and rstd go together", op);
    if (rows == 0)
        return SBNET_OK;
    if (x == nullptr || y == nullptr)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: null tensor pointer", op);
    if (((address(x) | address(y)) & elem_mask(dtype)) || ((address(weight) | address(bias)) & elem_mask(wdtype)) ||
        ((address(mean) | address(rstd) | address(num_blocks_dev)) & 3))
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: tensor pointer not aligned to its element size", op);
    const size_t bytes = (size_t)rows * C * (elem_mask(dtype) + 1), pbytes = (size_t)C * (elem_mask(wdtype) + 1), sbytes = (size_t)rows * 4;
    const Span in[] = {{x, bytes}, {weight, pbytes}, {bias, pbytes}, {num_blocks_dev, 4}},
               out[] = {{y, bytes}, {mean, sbytes}, {rstd, sbytes}};
    if (overlap(out, in))
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: an output must not overlap another tensor", op);
    sbnet::NormArgs a = {};
    a.x = x, a.y = y, a.weight = weight, a.bias = bias, a.mean = mean, a.rstd = rstd;
    a.num_blocks_dev = num_blocks_dev, a.rows = rows, a.rowsPerBlock = rowsPerBlock, a.C = C, a.wdtype = wdtype, a.eps = eps;
    return cuda_status(sbnet::launch_layer_norm(a, dtype, (cudaStream_t)stream));
}
} // namespace

SBNET_EXPORT int sbnet_layer_norm(const void* x, int dtype, int64_t rows, int C, const void* weight, const void* bias,
                                  int wdtype, float eps, void* y, float* mean, float* rstd, void* stream)
{
    return norm_call(x, dtype, rows, 1, nullptr, C, weight, bias, wdtype, eps, y, mean, rstd, stream);
}

SBNET_EXPORT int sbnet_layer_norm_dyn(const void* x, int dtype, int64_t maxBlocks, int rowsPerBlock,
                                      const int32_t* num_blocks_dev, int C, const void* weight, const void* bias,
                                      int wdtype, float eps, void* y, float* mean, float* rstd, void* stream)
{
    if (num_blocks_dev == nullptr)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "LayerNorm: num_blocks_dev is null");
    if (maxBlocks < 0 || rowsPerBlock < 1 || maxBlocks > (1ll << 40) / rowsPerBlock)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "LayerNorm: bad stack of %lld blocks of %d rows", (long long)maxBlocks,
                      rowsPerBlock);
    return norm_call(x, dtype, maxBlocks * rowsPerBlock, rowsPerBlock, num_blocks_dev, C, weight, bias, wdtype, eps, y,
                     mean, rstd, stream);
}

SBNET_EXPORT size_t sbnet_layer_norm_grad_workspace(int64_t rows, int C)
{
    if (rows < 1 || C < 1)
        return 0;
    return sizeof(float) * 2 * (size_t)C * sbnet::layer_norm_grad_parts(rows, C);
}

SBNET_EXPORT int sbnet_layer_norm_grad(const void* dy, const void* x, int dtype, int64_t rows, int C, const void* weight,
                                       int wdtype, const float* mean, const float* rstd, void* dx, void* dweight,
                                       void* dbias, void* workspace, size_t workspace_bytes, void* stream)
{
    const char* op = "LayerNormGrad";
    g_site = "";
    if (int rc = check_rows(op, dtype, rows, C))
        return rc;
    const bool sums = dweight != nullptr || dbias != nullptr;
    if ((weight != nullptr || sums) && wdtype != dtype && wdtype != SBNET_F32)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: weight and bias must share the tensor's dtype or be fp32", op);
    if (rows == 0 && !sums)
        return SBNET_OK;
    if (rows > 0 && (dy == nullptr || x == nullptr || dx == nullptr || mean == nullptr || rstd == nullptr))
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: null tensor pointer", op);
    if (((address(x) | address(dy) | address(dx)) & elem_mask(dtype)) ||
        ((address(weight) | address(dweight) | address(dbias)) & elem_mask(wdtype)) || ((address(mean) | address(rstd)) & 3))
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: tensor pointer not aligned to its element size", op);
    // dweight and dbias are written when all of the inputs have been read
    const size_t bytes = (size_t)rows * C * (elem_mask(dtype) + 1), pbytes = (size_t)C * (elem_mask(wdtype) + 1), sbytes = (size_t)rows * 4;
    const Span in[] = {{x, bytes}, {dy, bytes}, {weight, pbytes}, {mean, sbytes}, {rstd, sbytes}}, dxs[] = {{dx, bytes}};
    const Span none[] = {{nullptr, 0}}, out[] = {{dx, bytes}, {dweight, pbytes}, {dbias, pbytes}};
    if (rows > 0 && (overlap(dxs, in) || overlap(out, none)))
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: dx must not overlap an input, nor an output another", op);
    if (sums && rows > 0 && (workspace == nullptr || (address(workspace) & 15) ||
                 workspace_bytes < sbnet_layer_norm_grad_workspace(rows, C)))
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: needs %zu bytes of 16-byte aligned workspace", op,
                      sbnet_layer_norm_grad_workspace(rows, C));
    sbnet::NormArgs a = {};
    a.x = x, a.g = dy, a.y = dx, a.weight = weight, a.mean = const_cast<float*>(mean), a.rstd = const_cast<float*>(rstd);
    a.partials = sums ? static_cast<float*>(workspace) : nullptr, a.dweight = dweight, a.dbias = dbias;
    a.rows = rows, a.rowsPerBlock = 1, a.C = C, a.wdtype = wdtype;
    return cuda_status(sbnet::launch_layer_norm_grad(a, dtype, (cudaStream_t)stream));
}

namespace {
int check_ffn(const char* op, int dtype, int64_t rows, int C, int F, int act)
{
    if (int rc = check_rows(op, dtype, rows, C))
        return rc;
    if (dtype == SBNET_F32)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: fp16 and bf16 only (the tensor cores' operand types)", op);
    if (F < 1)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: needs at least one hidden channel, got %d", op, F);
    if (act != SBNET_ACT_SILU && act != SBNET_ACT_GELU && act != SBNET_ACT_RELU)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: unknown activation %d", op, act);
    if (F > (1 << 24) || rows >= (1ll << 31) - 256 || (rows / 128 + 1) * ((C > F ? C : F) / 128 + 1) >= (1ll << 31) / 256)
        return reject(SBNET_ERR_UNSUPPORTED, "%s: more than 2^31 work items", op);
    return SBNET_OK;
}

int check_workspace(const char* op, const void* workspace, size_t bytes, size_t need)
{
    if (need != 0 && (workspace == nullptr || (address(workspace) & 255) || bytes < need))
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: needs %zu bytes of 256-byte aligned workspace, got %zu", op, need, bytes);
    return SBNET_OK;
}

int ffn_call(const void* x, int dtype, int64_t rows, int rowsPerBlock, const int32_t* num_blocks_dev, int C, int F,
             const void* w_gate, const void* w_up, const void* w_down, int act, void* y, float* kept, void* workspace, size_t workspace_bytes, void* stream)
{
    const char* op = "GatedFfn";
    g_site = "";
    if (int rc = check_ffn(op, dtype, rows, C, F, act))
        return rc;
    if (rows == 0)
        return SBNET_OK;
    if (x == nullptr || y == nullptr || w_gate == nullptr || w_up == nullptr || w_down == nullptr)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: null tensor pointer", op);
    const uintptr_t inputs = address(x) | address(w_gate) | address(w_up) | address(w_down);
    if (((inputs | address(y)) & 1) || (address(num_blocks_dev) & 3) || (address(kept) & 15))
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: tensor pointer not aligned to its element size (kept: 16 bytes)", op);
    const size_t bytes = (size_t)rows * C * 2, wbytes = (size_t)F * C * 2, kbytes = (size_t)rows * ((F + 7) / 8 * 8) * 8;
    const Span in[] = {{x, bytes}, {w_gate, wbytes}, {w_up, wbytes}, {w_down, wbytes}, {num_blocks_dev, 4}}, out[] = {{y, bytes}, {kept, kbytes}};
    if (overlap(out, in))
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: an output must not overlap another tensor", op);
    if (int rc = check_workspace(op, workspace, workspace_bytes,
                                 sbnet::gated_ffn_workspace(rows, C, F, false, kept != nullptr, (inputs & 15) == 0)))
        return rc;
    sbnet::FfnArgs f = {};
    f.x = x, f.w_gate = w_gate, f.w_up = w_up, f.w_down = w_down, f.y = y, f.kept = kept;
    f.num_blocks_dev = num_blocks_dev, f.workspace = workspace, f.rows = rows, f.rowsPerBlock = rowsPerBlock;
    f.C = C, f.F = F, f.act = act;
    return cuda_status(sbnet::launch_gated_ffn(f, dtype, (cudaStream_t)stream));
}
} // namespace

SBNET_EXPORT size_t sbnet_gated_ffn_workspace(int64_t rows, int C, int F, int mode, int aligned)
{
    if (rows < 1 || C < 1 || F < 1)
        return 0;
    return sbnet::gated_ffn_workspace(rows, C, F, mode == SBNET_FFN_BACKWARD, mode == SBNET_FFN_FORWARD_KEEP, aligned != 0);
}

SBNET_EXPORT int sbnet_gated_ffn(const void* x, int dtype, int64_t rows, int C, int F, const void* w_gate,
                                 const void* w_up, const void* w_down, int act, void* y, float* kept, void* workspace,
                                 size_t workspace_bytes, void* stream)
{
    return ffn_call(x, dtype, rows, 1, nullptr, C, F, w_gate, w_up, w_down, act, y, kept, workspace, workspace_bytes, stream);
}

SBNET_EXPORT int sbnet_gated_ffn_dyn(const void* x, int dtype, int64_t maxBlocks, int rowsPerBlock,
                                     const int32_t* num_blocks_dev, int C, int F, const void* w_gate, const void* w_up,
                                     const void* w_down, int act, void* y, void* workspace, size_t workspace_bytes,
                                     void* stream)
{
    if (num_blocks_dev == nullptr)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "GatedFfn: num_blocks_dev is null");
    if (maxBlocks < 0 || rowsPerBlock < 1 || maxBlocks > (1ll << 40) / rowsPerBlock)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "GatedFfn: bad stack of %lld blocks of %d rows", (long long)maxBlocks,
                      rowsPerBlock);
    return ffn_call(x, dtype, maxBlocks * rowsPerBlock, rowsPerBlock, num_blocks_dev, C, F, w_gate, w_up, w_down, act, y,
                    nullptr, workspace, workspace_bytes, stream);
}

SBNET_EXPORT int sbnet_gated_ffn_grad(const void* dy, const void* x, const float* kept, int dtype, int64_t rows, int C, int F, const void* w_gate, const void* w_up,
                                      const void* w_down, int act, void* dx, void* dw_gate, void* dw_up, void* dw_down,
                                      void* workspace, size_t workspace_bytes, void* stream)
{
    const char* op = "GatedFfnGrad";
    g_site = "";
    if (int rc = check_ffn(op, dtype, rows, C, F, act))
        return rc;
    if ((dw_gate == nullptr) != (dw_up == nullptr))
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: dw_gate and dw_up go together", op);
    if ((address(dx) | address(dw_gate) | address(dw_up) | address(dw_down)) & 1)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: tensor pointer not aligned to its element size", op);
    cudaStream_t s = (cudaStream_t)stream;
    if (rows == 0) {     // sums over no rows
        for (void* w : {dw_gate, dw_up, dw_down})
            if (w != nullptr)
                if (cudaError_t e = cudaMemsetAsync(w, 0, (size_t)F * C * 2, s))
                    return cuda_status(e);
        return SBNET_OK;
    }
    if (dy == nullptr || x == nullptr || w_gate == nullptr || w_up == nullptr || w_down == nullptr)
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: null tensor pointer", op);
    const uintptr_t inputs = address(dy) | address(x) | address(w_gate) | address(w_up) | address(w_down);
    if ((inputs & 1) || (address(kept) & 15))
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: tensor pointer not aligned to its element size (kept: 16 bytes)", op);
    const size_t bytes = (size_t)rows * C * 2, wbytes = (size_t)F * C * 2, kbytes = (size_t)rows * ((F + 7) / 8 * 8) * 8;
    const Span in[] = {{dy, bytes}, {x, bytes}, {kept, kbytes}, {w_gate, wbytes}, {w_up, wbytes}, {w_down, wbytes}},
               out[] = {{dx, bytes}, {dw_gate, wbytes}, {dw_up, wbytes}, {dw_down, wbytes}};
    if (overlap(out, in))
        return reject(SBNET_ERR_INVALID_ARGUMENT, "%s: an output must not overlap another tensor", op);
    if (int rc = check_workspace(op, workspace, workspace_bytes,
                                 sbnet::gated_ffn_workspace(rows, C, F, true, false, (inputs & 15) == 0)))
        return rc;
    sbnet::FfnArgs f = {};
    f.dy = dy, f.x = x, f.kept = const_cast<float*>(kept);
    f.w_gate = w_gate, f.w_up = w_up, f.w_down = w_down;
    f.dx = dx, f.dw_gate = dw_gate, f.dw_up = dw_up, f.dw_down = dw_down;
    f.workspace = workspace, f.rows = rows, f.rowsPerBlock = 1, f.C = C, f.F = F, f.act = act;
    return cuda_status(sbnet::launch_gated_ffn_grad(f, dtype, s));
}
