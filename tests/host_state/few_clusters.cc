// The few-row feed-forward kernels' question of how many clusters a device holds: every kernel gets its own answer, a
// question that failed is asked again, and threads may ask at once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <cstdio>
#include <set>
#include <thread>

#include "fake_runtime.h"
#include "kernels.h"

namespace sbnet {
template <typename T> cudaError_t launch_ffn_few(const FfnArgs& f, void* h, cudaStream_t stream, bool* taken);
}

namespace {

int bad = 0;
void expect(bool ok, const char* what)
{
    if (!ok)
        printf("not so: %s\n", what), bad = 1;
}

template <typename T> bool call(int rows, int C, int F)
{
    sbnet::FfnArgs f = {};
    f.x = reinterpret_cast<void*>(1 << 20), f.w_gate = reinterpret_cast<void*>(1 << 24), f.w_up = reinterpret_cast<void*>(1 << 25);
    f.w_down = reinterpret_cast<void*>(1 << 26), f.y = reinterpret_cast<void*>(1 << 28);
    f.rows = rows, f.C = C, f.F = F, f.rowsPerBlock = 1;
    bool taken = false;
    const size_t before = fake::state().launches.size();
    expect(sbnet::launch_ffn_few<T>(f, reinterpret_cast<void*>(1 << 27), nullptr, &taken) == cudaSuccess, "the call succeeds");
    expect(fake::state().launches.size() - before == (taken ? 2u : 0u), "both kernels are launched, or none");
    return taken;
}

} // namespace

int main()
{
    auto& s = fake::state();
    // 24 rows of 4,096 hidden channels: the output kernel's X fits shared memory only where a cluster splits it
    int asked = 0;
    s.occupancy = [&](int*, const void*, int) { return ++asked, cudaErrorUnknown; };
    expect(!call<__half>(24, 512, 4096), "not taken while nobody knows how many clusters fit");
    expect(asked > 0, "the device was asked");
    const int before = asked;
    s.occupancy = [&](int* n, const void*, int cluster) { return *n = 132 / cluster, ++asked, cudaSuccess; };
    expect(call<__half>(24, 512, 4096), "taken once the device answers");
    expect(asked > before, "the device was asked again");
    const int answered = asked;
    expect(call<__half>(24, 512, 4096) && asked == answered, "an answer is kept");

    // few groups: splits are chosen for want of groups; kernels that differ in what the device holds of them
    std::map<const void*, int> most;
    s.occupancy = [&](int* n, const void* kernel, int cluster) {
        if (!most.count(kernel))
            most[kernel] = most.size() % 2 ? 3 : 140;
        return *n = most[kernel], (void)cluster, cudaSuccess;
    };
    s.launches.clear();
    for (int i = 0; i < 2; ++i) {
        call<__nv_bfloat16>(1, 4096, 1024), call<__half>(1, 4096, 1024);
        call<__nv_bfloat16>(1, 1024, 4096), call<__half>(1, 1024, 4096);
        call<__nv_bfloat16>(20, 1024, 4096);        // (the half kernels of that many rows have their answers from above)
    }
    std::set<const void*> kernels;
    for (const auto& l : s.launches)
        if (l.cluster > 1) {
            kernels.insert(l.kernel);
            expect(most.count(l.kernel) != 0, "the device was asked about this kernel");
            expect((int)(l.grid / l.cluster) <= most[l.kernel], "a grid of no more clusters than that kernel's answer");
        }
    expect(kernels.size() >= 2, "several kernels ran in clusters");

    // many threads at once, every answer the same
    s.occupancy = [&](int* n, const void*, int cluster) { return *n = 140 / cluster, cudaSuccess; };
    std::thread threads[8];
    for (int t = 0; t < 8; ++t)
        threads[t] = std::thread([] {
            for (int i = 0; i < 50; ++i) {
                sbnet::FfnArgs f = {};
                f.x = f.w_gate = f.w_up = f.w_down = reinterpret_cast<void*>(1 << 20), f.y = reinterpret_cast<void*>(1 << 28);
                f.rows = 1 + i % 16, f.C = 256, f.F = 2048, f.rowsPerBlock = 1;
                bool taken = false;
                sbnet::launch_ffn_few<__half>(f, reinterpret_cast<void*>(1 << 27), nullptr, &taken);
            }
        });
    for (auto& t : threads)
        t.join();
    puts(bad ? "FAIL" : "PASS");
    return bad;
}
