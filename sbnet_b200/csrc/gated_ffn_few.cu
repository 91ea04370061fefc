// The gated feed-forward block for up to 32 rows (single positions of a batch): every weight is read once for a handful
// of rows, so the two kernels are weight streams and bound by HBM.
//
//   gate kernel: H = act(X Wg^T) * (X Wu^T)        output kernel: Y = H Wd^T
//
// Both are the same code: a group is 16 weight rows (8 of Wg and the same 8 of Wu, or 16 of Wd), and a warp multiplies
// pieces of a group with all rows of X by mma.sync m16n8k16 (rows of X are the 16-high operand, weight rows the 8-wide
// one).  The tcgen05 path would have to bring the weights through shared memory for a 128-row operand that is mostly
// padding; here they go from global memory straight into the registers that the instruction reads.  That works with
// 16-byte loads because the order of the reduction is free: lane (g, t) loads 8 consecutive elements of weight row g
// and of rows g and g + 8 of X, at the same 8 positions, and hands them out as the fragments of two instructions.
//
// The eight warps of a CTA split the reduction in pieces of 64, so that together they read 1 KB runs of every weight
// row; 16 16-byte loads per lane are in flight, each reissued as soon as its registers have been multiplied (64 KB per
// CTA, and up to 16 rows two CTAs share an SM).  A CTA sums its
// warps' results in shared memory in a fixed order.  Where the groups do not fill the SMs evenly, or X does not fit
// shared memory, a cluster of 2, 4 or 8 CTAs splits the reduction further and sums over distributed shared memory,
// again in a fixed order.
#include <algorithm>

#include "gated_ffn.cuh"
#include "tensor_ptx.cuh"

namespace sbnet {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kBatch = 4;            // pieces of 64 that a warp loads ahead
constexpr int kMaxRows = 32;
constexpr int kSmemLimit = 224 * 1024, kSmemHalf = 110 * 1024;     // of a CTA that has an SM alone, or shares it

struct FewArgs {
    const void *x, *w0, *w1;         // X [M, K]; the group's first and second 8 weight rows
    void* out;                       // [M, N]
    float *gate, *up;                // gate kernel: G and U [M, N], or nullptr
    const int32_t* num_blocks_dev;
    long long M;
    int rowsPerBlock, K, N, act;
    int groups, perCluster;          // groups of the whole product and, at most, of one cluster
    int pieces, perCta;              // 64-long pieces of the reduction, and at most of one CTA
};

template <typename T> __device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ld_cluster(uint32_t addr)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, int rank)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}

template <int MT> constexpr int kPartFloats = kWarps * MT * 16 * 16;     // [warp][row of X][weight row of the group]

// MT: 16-high tiles of X.  GATE: which of the two kernels.
template <typename T, int MT, bool GATE> __global__ void __launch_bounds__(kThreads, MT == 1 ? 2 : 1) few_kernel(FewArgs p, int splits)
{
    extern __shared__ __align__(16) uint8_t dyn[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rank = splits > 1 ? (int)cluster_rank() : 0, cluster = blockIdx.x / splits, clusters = gridDim.x / splits;
    const int c0 = (int)((long long)p.pieces * rank / splits), nPieces = (int)((long long)p.pieces * (rank + 1) / splits) - c0;
    const int pitch = p.perCta * 128 + 64;                   // of X here: 8 lanes' 16-byte reads hit 8 different pieces of 128 bytes
    const int M = (int)p.M;
    const uint32_t xs = smem_u32(dyn);
    float* part = reinterpret_cast<float*>(dyn + (size_t)M * pitch);        // [2][kPartFloats]
    float* sums = part + 2 * kPartFloats<MT>;                               // splits > 1: [perCluster][16 MT][16]
    const T *w0 = static_cast<const T*>(p.w0), *w1 = static_cast<const T*>(p.w1);
    const int batches = (nPieces + kWarps * kBatch - 1) / (kWarps * kBatch);
    const int myGroups = cluster < p.groups ? (p.groups - cluster + clusters - 1) / clusters : 0;

    uint4 next[kBatch][2][2];
    // this warp's piece of slot c in batch b of group number gi
    auto load = [&](int gi, int b, int c) {
        const int group = cluster + gi * clusters;
        const int r0 = GATE ? group * 8 + g : group * 16 + g, r1 = GATE ? r0 : r0 + 8;
        const int piece = warp + kWarps * (b * kBatch + c);
        const bool in = gi < myGroups && piece < nPieces;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = (c0 + piece) * 64 + h * 32 + t * 8;
            next[c][h][0] = next[c][h][1] = make_uint4(0, 0, 0, 0);
            if (in && k < p.K && r0 < p.N)
                next[c][h][0] = ld_stream(reinterpret_cast<const uint4*>(w0 + (long long)r0 * p.K + k));
            if (in && k < p.K && r1 < p.N)
                next[c][h][1] = ld_stream(reinterpret_cast<const uint4*>(w1 + (long long)r1 * p.K + k));
        }
    };
    if (GATE)
        pdl_wait();
    // the output kernel's weights are not what the gate kernel before it writes, and that kernel let this one start only
    // after everything before it was done
#pragma unroll
    for (int c = 0; c < kBatch; ++c)
        load(0, 0, c);
    if (!GATE)
        pdl_wait();
    pdl_launch_dependents();

    // X of this CTA's pieces; zeros past the end of the reduction.  Every warp copies what it will read itself, its first
    // batch as a group of its own, so that nobody waits for all of X.
    auto stage_x = [&](int from, int to) {
        for (int j = from; j < to; ++j) {
            const int piece = warp + kWarps * j;
            if (piece >= nPieces)
                break;
            const int k = (c0 + piece) * 64 + (lane & 7) * 8;
            const T* src = static_cast<const T*>(p.x) + k;
            const uint32_t dst = xs + piece * 128 + (lane & 7) * 16;
#pragma unroll 4
            for (int row = lane >> 3; row < M; row += 4) {
                if (k < p.K)
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(dst + row * pitch), "l"(src + (long long)row * p.K) : "memory");
                else
                    sts128(dst + row * pitch, make_uint4(0, 0, 0, 0));
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    stage_x(0, kBatch);
    stage_x(kBatch, batches * kBatch);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();

    const int rowEnd = (int)live_rows(p.M, p.num_blocks_dev, p.rowsPerBlock);
    auto finish = [&](int group, int tok, int r, float s0, float s1) {      // r < 8: weight rows r and r + 8 of the group
        if (tok >= rowEnd)
            return;
        if (GATE) {
            const long long at = (long long)tok * p.N + group * 8 + r;
            static_cast<T*>(p.out)[at] = T(activate_any(p.act, s0) * s1);
            if (p.gate != nullptr)
                p.gate[at] = s0, p.up[at] = s1;
        } else {
            const int col = group * 16 + r;
            T* y = static_cast<T*>(p.out) + (long long)tok * p.N + col;
            if (col < p.N)
                y[0] = T(s0);
            if (col + 8 < p.N)
                y[8] = T(s1);
        }
    };

    for (int gi = 0; gi < myGroups; ++gi) {
        float acc[MT][2][4] = {};
        for (int b = 0; b < batches; ++b) {
            const bool last = b + 1 == batches;
            if (gi == 0 && b == 1) {
                asm volatile("cp.async.wait_all;" ::: "memory");
                __syncwarp();
            }
#pragma unroll
            for (int c = 0; c < kBatch; ++c) {
                const int piece = warp + kWarps * (b * kBatch + c);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (piece >= nPieces)
                        break;
                    const uint32_t at = xs + piece * 128 + h * 64 + t * 16;
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        // rows past M repeat the last one; their results are not stored
                        const uint4 lo = lds128(at + min(m * 16 + g, M - 1) * pitch), hi = lds128(at + min(m * 16 + 8 + g, M - 1) * pitch);
                        const uint32_t a0[4] = {lo.x, hi.x, lo.y, hi.y}, a1[4] = {lo.z, hi.z, lo.w, hi.w};
#pragma unroll
                        for (int s = 0; s < 2; ++s) {
                            mma16816<T>(acc[m][s], a0, next[c][h][s].x, next[c][h][s].y);
                            mma16816<T>(acc[m][s], a1, next[c][h][s].z, next[c][h][s].w);
                        }
                    }
                }
                load(last ? gi + 1 : gi, last ? 0 : b + 1, c);     // the slot's next use
            }
        }
        float* mine = part + (gi & 1) * kPartFloats<MT>;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                float* q = mine + ((warp * MT + m) * 16 + g) * 16 + s * 8 + 2 * t;
                *reinterpret_cast<float2*>(q) = make_float2(acc[m][s][0], acc[m][s][1]);
                *reinterpret_cast<float2*>(q + 8 * 16) = make_float2(acc[m][s][2], acc[m][s][3]);
            }
        __syncthreads();    // one a group: the other buffer is free again once every warp has passed here
        for (int i = threadIdx.x; i < M * 8; i += kThreads) {
            const int tok = i >> 3, r = i & 7;
            float s0 = 0.f, s1 = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float* q = mine + (w * MT * 16 + tok) * 16 + r;
                s0 += q[0], s1 += q[8];
            }
            if (splits == 1)
                finish(cluster + gi * clusters, tok, r, s0, s1);
            else
                sums[(gi * MT * 16 + tok) * 16 + r] = s0, sums[(gi * MT * 16 + tok) * 16 + 8 + r] = s1;
        }
    }
    if (splits > 1) {
        cluster_sync();
        for (int gi = rank; gi < myGroups; gi += splits)
            for (int i = threadIdx.x; i < M * 8; i += kThreads) {
                const int tok = i >> 3, r = i & 7;
                const uint32_t at = smem_u32(sums + (gi * MT * 16 + tok) * 16 + r);
                float s0 = 0.f, s1 = 0.f;
                for (int q = 0; q < splits; ++q) {
                    const uint32_t there = in_cta(at, q);
                    s0 += ld_cluster(there), s1 += ld_cluster(there + 32);
                }
                finish(cluster + gi * clusters, tok, r, s0, s1);
            }
        cluster_sync();     // nobody leaves while its sums are being read
    }
}

int few_smem(int M, int mt, int perCta, int splits, int perCluster)
{
    return M * (perCta * 128 + 64) + 4 * (2 * kWarps * mt * 256 + (splits > 1 ? perCluster * mt * 256 : 0));
}

cudaLaunchConfig_t config(int grid, int smem, int splits, cudaStream_t stream, cudaLaunchAttribute (&attr)[2])
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = smem, cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = splits, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = options().pdl ? 2 : 1;
    return cfg;
}

struct FewPlan {
    int splits, clusters, smem;
};

// Clusters of `splits` CTAs that the device holds at once, with `smem` bytes of shared memory each or, for `perSm` == 2,
// half of an SM's.  Asked once per kernel, device and size: it depends on how the SMs are grouped, not on the call.  A
// question that fails is asked again by the next call.
struct Residency {      // one kernel's answers, 0 where there is none yet; shared by the host threads
    std::atomic<int> known[64][2][4];
};
template <typename K> int resident_clusters(K kernel, Residency& residency, int splits, int perSm)
{
    if (splits == 1)
        return sm_count() * perSm;
    int device = 0, slot = splits == 2 ? 1 : splits == 4 ? 2 : 3;
    if (cudaGetDevice(&device) != cudaSuccess || device >= 64)
        return 0;
    std::atomic<int>& known = residency.known[device][perSm - 1][slot];
    int n = known.load(std::memory_order_relaxed);
    if (n == 0) {
        cudaLaunchAttribute attr[2];
        cudaLaunchConfig_t cfg = config(sm_count() * perSm / splits * splits, perSm == 2 ? kSmemHalf : kSmemLimit, splits, nullptr, attr);
        cfg.numAttrs = 1;
        if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
            (void)cudaGetLastError();
            return 0;
        }
        n = n > 0 ? n : -1;
        known.store(n, std::memory_order_relaxed);
    }
    return std::max(n, 0);
}

// The split of the reduction under which the SMs stay busiest (the share of the last round of groups that is in use),
// more CTAs to a cluster only where that gains 4 % a step; none where X and the sums do not fit shared memory.
template <typename K> FewPlan plan_few(K kernel, Residency& residency, int M, int mt, int K_, int groups)
{
    FewPlan best = {0, 0, 0};
    double score = 0;
    const int pieces = (K_ + 63) / 64;
    for (int perSm = mt == 1 ? 2 : 1; perSm >= 1; --perSm)
        for (int s = 1, step = 0; s <= 8; s *= 2, ++step) {
            if (s > pieces)
                break;
            const int clusters = std::min(groups, resident_clusters(kernel, residency, s, perSm));
            if (clusters < 1)
                continue;
            const int per = (groups + clusters - 1) / clusters, smem = few_smem(M, mt, (pieces + s - 1) / s, s, per);
            if (smem > (perSm == 2 ? kSmemHalf : kSmemLimit))
                continue;
            const double busy = (double)groups / per * s / (sm_count() * perSm) - 0.04 * step - (perSm == 1 && mt == 1 ? 0.3 : 0.);
            if (busy > score)
                score = busy, best = {s, clusters, smem};
        }
    return best;
}

template <typename T, int MT, bool GATE> cudaError_t run(FewArgs& a, cudaStream_t stream, bool dry, bool* fits)
{
    auto kernel = few_kernel<T, MT, GATE>;
    static std::atomic<bool> done[64] = {};
    static Residency residency = {};
    if (cudaError_t e = allow_smem(kernel, kSmemLimit, done))
        return e;
    a.groups = GATE ? a.N / 8 : (a.N + 15) / 16;
    a.pieces = (a.K + 63) / 64;
    const FewPlan plan = plan_few(kernel, residency, (int)a.M, MT, a.K, a.groups);
    *fits = plan.splits > 0;
    if (!*fits || dry)
        return cudaSuccess;
    a.perCta = (a.pieces + plan.splits - 1) / plan.splits;
    a.perCluster = (a.groups + plan.clusters - 1) / plan.clusters;
    cudaLaunchAttribute attr[2];
    const cudaLaunchConfig_t cfg = config(plan.clusters * plan.splits, plan.smem, plan.splits, stream, attr);
    return cudaLaunchKernelEx(&cfg, kernel, a, plan.splits);
}

template <typename T, int MT> cudaError_t both(const FfnArgs& f, void* h, cudaStream_t stream, bool* taken)
{
    FewArgs gate = {}, out = {};
    gate.x = f.x, gate.w0 = f.w_gate, gate.w1 = f.w_up, gate.out = h;
    if (f.kept != nullptr)
        gate.gate = f.kept, gate.up = f.kept + (size_t)f.rows * f.F;
    gate.K = f.C, gate.N = f.F, gate.act = f.act;
    out.x = h, out.w0 = out.w1 = f.w_down, out.out = f.y, out.K = f.F, out.N = f.C;
    gate.M = out.M = f.rows;
    gate.num_blocks_dev = out.num_blocks_dev = f.num_blocks_dev, gate.rowsPerBlock = out.rowsPerBlock = f.rowsPerBlock;
    bool fits = false;
    if (cudaError_t e = run<T, MT, false>(out, stream, true, &fits))
        return e;
    if (!fits)
        return cudaSuccess;
    note_site("gated_ffn projections (few rows)");
    if (cudaError_t e = run<T, MT, true>(gate, stream, false, taken))
        return e;
    if (!*taken)
        return cudaSuccess;
    note_site("gated_ffn output (few rows)");
    return run<T, MT, false>(out, stream, false, &fits);
}

} // namespace

// Taken for up to 32 rows of at most 2^17 elements of X or H together; 16-byte loads need rows of a multiple of 8 elements
// on 16-byte boundaries.  With more of X to keep in shared memory the clusters' pieces become so short that the sums per
// group cost more than the tensor cores' padding (4096 x 12288 fp16: 1 row 56 against 94 us, 8 rows 67 against 75, 16 rows
// 83 against 75; 2048 x 8192: 16 rows 32 against 36, 32 rows 36 either way; 1024 x 4096: 32 rows 20 against 23).
template <typename T> cudaError_t launch_ffn_few(const FfnArgs& f, void* h, cudaStream_t stream, bool* taken)
{
    *taken = false;
    const uintptr_t bits = reinterpret_cast<uintptr_t>(f.x) | reinterpret_cast<uintptr_t>(f.w_gate) |
                           reinterpret_cast<uintptr_t>(f.w_up) | reinterpret_cast<uintptr_t>(f.w_down);
    if (f.rows > kMaxRows || f.rows * std::max(f.C, f.F) > (1 << 17) || f.C % 8 != 0 || f.F % 8 != 0 || (bits & 15) != 0)
        return cudaSuccess;
    return f.rows <= 16 ? both<T, 1>(f, h, stream, taken) : both<T, 2>(f, h, stream, taken);
}
template cudaError_t launch_ffn_few<__half>(const FfnArgs&, void*, cudaStream_t, bool*);
template cudaError_t launch_ffn_few<__nv_bfloat16>(const FfnArgs&, void*, cudaStream_t, bool*);

} // namespace sbnet
