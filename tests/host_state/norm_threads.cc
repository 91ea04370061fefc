// Layer norm's launch code from two host threads at once, a wide call and a narrower one of the same kernel: whichever
// thread raises the kernel's shared-memory limit last, both calls and every later one are launched.
#include <chrono>
#include <condition_variable>
#include <cstdio>
#include <thread>

#include "fake_runtime.h"
#include "kernels.h"

namespace {

struct Race {
    std::mutex m;
    std::condition_variable cv;
    bool wideHasSet = false, narrowIsDone = false;
    template <typename P> bool wait(P p)
    {
        std::unique_lock<std::mutex> l(m);
        return cv.wait_for(l, std::chrono::milliseconds(500), p);
    }
    void set(bool& what)
    {
        std::lock_guard<std::mutex> l(m);
        what = true;
        cv.notify_all();
    }
};
thread_local bool t_wide = false;

cudaError_t call(bool grad, int dtype, int C)
{
    sbnet::NormArgs a = {};
    a.x = reinterpret_cast<void*>(1 << 20), a.g = reinterpret_cast<void*>(1 << 24), a.y = reinterpret_cast<void*>(1 << 28);
    a.mean = reinterpret_cast<float*>(1 << 16), a.rstd = reinterpret_cast<float*>(1 << 17);
    a.rows = 10, a.rowsPerBlock = 1, a.C = C, a.wdtype = dtype, a.eps = 1e-5f;
    return grad ? sbnet::launch_layer_norm_grad(a, dtype, nullptr) : sbnet::launch_layer_norm(a, dtype, nullptr);
}

int race(bool grad, int dtype, int narrow, int wide)
{
    Race r;
    // the wide call has set its limit and not yet gone on when the narrow one comes
    fake::state().afterSet = [&](int) {
        if (t_wide) {
            r.set(r.wideHasSet);
            r.wait([&] { return r.narrowIsDone; });
        }
    };
    cudaError_t wideResult = cudaErrorUnknown, narrowResult = cudaErrorUnknown;
    std::thread b([&] {
        t_wide = true;
        wideResult = call(grad, dtype, wide);
        r.set(r.wideHasSet);
    });
    r.wait([&] { return r.wideHasSet; });
    std::thread a([&] {
        narrowResult = call(grad, dtype, narrow);
        r.set(r.narrowIsDone);
    });
    a.join(), b.join();
    fake::state().afterSet = nullptr;
    const cudaError_t later = call(grad, dtype, wide);
    printf("%s dtype %d, %d beside %d channels: narrow %d, wide %d, wide again %d\n", grad ? "backward" : "forward", dtype, narrow,
           wide, (int)narrowResult, (int)wideResult, (int)later);
    return narrowResult || wideResult || later;
}

} // namespace

int main()
{
    int bad = 0;
    // forward: 2,049 to 8,192 fp32 channels are one kernel, 48 and 96 KB; 8,193 to 16,384 another
    bad |= race(false, 0, 4096, 8192);
    for (int dtype = 1; dtype <= 2; ++dtype)
        bad |= race(true, dtype, 4096, 8192);       // 64 and 128 KB
    // every width once more, one after the other, both directions and types
    for (int dtype = 0; dtype <= 2; ++dtype)
        for (int C = 1; C <= 20000; C += C < 700 ? 37 : 613)
            for (int grad = 0; grad < 2; ++grad)
                if (cudaError_t e = call(grad != 0, dtype, C / 8 * 8 + (C & 1 ? 0 : 8))) {
                    printf("width %d dtype %d grad %d: error %d\n", C, dtype, grad, (int)e);
                    bad = 1;
                }
    puts(bad ? "FAIL" : "PASS");
    return bad;
}
