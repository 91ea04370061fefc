// A CUDA runtime for programs that link the library's launch code without a device: nothing runs, and what the code
// asks for -- limits, occupancy, launches -- goes to hooks that a test sets.
#pragma once
#include <cuda_runtime.h>

#include <functional>
#include <map>
#include <mutex>
#include <vector>

namespace fake {

struct Launch {
    const void* kernel;
    unsigned grid, cluster;
    size_t smem;
};
struct State {
    std::mutex lock;
    std::map<const void*, int> limit;       // dynamic shared memory that a kernel may ask for
    std::vector<Launch> launches;           // those that were accepted
    std::function<void(int bytes)> afterSet;                                         // in cudaFuncSetAttribute, the limit is set
    std::function<cudaError_t(int* n, const void* kernel, int cluster)> occupancy;   // cudaOccupancyMaxActiveClusters
};
State& state();

} // namespace fake
