#include "fake_runtime.h"

#include "options.h"

namespace fake {
State& state()
{
    static State s;
    return s;
}
} // namespace fake

namespace sbnet {
Options& options()
{
    static Options o;
    return o;
}
int sm_count() { return 148; }
void note_site(const char*) {}
} // namespace sbnet

using fake::state;

static unsigned cluster_of(const cudaLaunchConfig_t* cfg)
{
    for (unsigned i = 0; i < cfg->numAttrs; ++i)
        if (cfg->attrs[i].id == cudaLaunchAttributeClusterDimension)
            return cfg->attrs[i].val.clusterDim.x;
    return 1;
}

extern "C" {
cudaError_t cudaGetDevice(int* device)
{
    *device = 0;
    return cudaSuccess;
}
cudaError_t cudaGetLastError(void) { return cudaSuccess; }
cudaError_t cudaFuncSetAttribute(const void* kernel, cudaFuncAttribute attr, int value)
{
    if (attr != cudaFuncAttributeMaxDynamicSharedMemorySize || value > 227 * 1024)
        return cudaErrorInvalidValue;
    {
        std::lock_guard<std::mutex> guard(state().lock);
        state().limit[kernel] = value;
    }
    if (state().afterSet)
        state().afterSet(value);
    return cudaSuccess;
}
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* cfg, const void* kernel, void**)
{
    std::lock_guard<std::mutex> guard(state().lock);
    const auto limit = state().limit.find(kernel);
    if (cfg->dynamicSmemBytes > (limit == state().limit.end() ? 48u * 1024u : (size_t)limit->second))
        return cudaErrorInvalidValue;
    state().launches.push_back({kernel, cfg->gridDim.x, cluster_of(cfg), cfg->dynamicSmemBytes});
    return cudaSuccess;
}
cudaError_t cudaLaunchKernel(const void*, dim3, dim3, void**, size_t, cudaStream_t) { return cudaErrorNotSupported; }
cudaError_t cudaOccupancyMaxActiveClusters(int* n, const void* kernel, const cudaLaunchConfig_t* cfg)
{
    return state().occupancy(n, kernel, (int)cluster_of(cfg));
}
// registration of the device code, which is never run
void** __cudaRegisterFatBinary(void*)
{
    static void* handle = nullptr;
    return &handle;
}
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char*, char*, const char*, int, uint3*, uint3*, dim3*, dim3*, int*) {}
void __cudaRegisterVar(void**, char*, char*, const char*, int, size_t, int, int) {}
char __cudaInitModule(void**) { return 1; }
unsigned __cudaPushCallConfiguration(dim3, dim3, size_t, struct CUstream_st*) { return 1; }
cudaError_t __cudaPopCallConfiguration(dim3*, dim3*, size_t*, void*) { return cudaErrorNotSupported; }
}
