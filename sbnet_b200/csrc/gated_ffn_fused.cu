// The gated feed-forward block in one kernel, for the channel counts of a convolutional network's stacks (up to 256) and
// many rows:  Y = (act(X Wg^T) * (X Wu^T)) Wd^T  with neither G, U nor H in memory.
//
// With few channels the two-kernel form is bound by H on its way to memory and back (8 F bytes a row against 4 C for X
// and Y).  Here a pair of CTAs keeps its 256 rows of X in shared memory and walks the hidden channels in chunks of 64:
//
//   GU(j) = X [Wg_j ; Wu_j]^T      256 x 128 accumulator in TMEM, two of them in turn
//   H(j)  = act(G) * U             registers -> shared memory, laid out as the next product's operand
//   Y    += H(j) Wd_j^T            256 x C accumulator in TMEM
//
// so that X and Y move once and the weights stream out of L2 (each CTA of the pair loads half of every weight tile:
// rows of Wg or of Wu, half the rows of Wd).  GU and Y are issued by a
// warp each, GU up to two chunks ahead, and two groups of eight epilogue warps take the chunks in turn, so the tensor
// cores, the special-function units (two exponentials and a reciprocal for two values of H) and the loads overlap.
// Waits are bounded as in the other matrix kernels.
//
// Measured (one call with a cold L2, launch included): 419,328 rows x 128 channels x 512 hidden, fp16, silu 179 us, the
// tensor pipe 0.50 and the issue slots 0.63 busy; 102,400 x 256 x 1,024 bf16 136 us.  Beyond 64 channels
// a thread reloads 36 bytes from spills.
#include <algorithm>

#include "gated_ffn.cuh"

namespace sbnet {
namespace {

__device__ unsigned int g_fused_timeouts = 0;

constexpr int kRows = 256, kCtaRows = 128;      // of a tile, and of each CTA of the pair
constexpr int kChunk = 64;                      // hidden channels of a step
constexpr int kGroupWarps = 8;                  // epilogue warps of each of the two groups
// Warps: 0 loads X and the weights of GU, 1 issues GU, then the epilogue's, then one that loads Wd and one that issues Y.
constexpr int kWdWarp = 2 + 2 * kGroupWarps, kYWarp = kWdWarp + 1, kThreads = (kYWarp + 1) * 32;

// KC: 64-channel pieces of C.  Stage counts and buffers by what shared memory holds.
template <int KC> struct Fused {
    static constexpr int kXBytes = KC * kCtaRows * 128;            // X of a tile, per CTA
    static constexpr int kXBufs = KC <= 2 ? 2 : 1;
    static constexpr int kW1Bytes = KC * kChunk * 128;             // this CTA's half of a GU chunk's weights
    static constexpr int kWdBytes = KC * 32 * 128;                 // ... of a Y chunk's
    static constexpr int kStages = KC <= 2 ? 3 : 2;
    static constexpr int kHBytes = kCtaRows * 128;
    static constexpr int kYCols = KC * 64;                         // columns of Y's accumulator
    static constexpr int kYBufs = KC <= 2 ? 2 : 1;
    static constexpr int kStaging = 2 * kGroupWarps * 2048;
    static constexpr int kX = 0, kW1 = kX + kXBufs * kXBytes, kWd = kW1 + kStages * kW1Bytes, kH = kWd + kStages * kWdBytes,
                         kStage = kH + 2 * kHBytes, kBars = kStage + kStaging, kSmem = 1024 + kBars + 256;
};

struct FusedMaps {
    CUtensorMap x, wg, wu, wd;
};
struct FusedArgs {
    void* y;
    const int32_t* num_blocks_dev;
    long long rows;
    int rowsPerBlock, C, chunks, act;
};

template <typename T, int ACT>
__device__ __forceinline__ void gate_words(const uint32_t (&g)[32], const uint32_t (&u)[32], uint32_t (&h)[16])
{
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        F2 a, unused;
        activate2<ACT, false>(words(g[2 * i], g[2 * i + 1]), a, unused);
        h[i] = pack2<T>(mul2(a, words(u[2 * i], u[2 * i + 1])));
    }
}

// Barriers (8 bytes each).  Those the tensor cores wait for are the first CTA's, and both CTAs' loads and epilogue
// warps arrive there; those that free a buffer are signalled in both CTAs.
template <int S> struct Bars {
    static constexpr int w1Full = 0, w1Empty = w1Full + S, wdFull = w1Empty + S, wdEmpty = wdFull + S, xFull = wdEmpty + S,
                         xEmpty = xFull + 2, guFull = xEmpty + 2, guEmpty = guFull + 2, hFull = guEmpty + 2, hEmpty = hFull + 2,
                         yFull = hEmpty + 2, yEmpty = yFull + 2, drain = yEmpty + 2, drainY = drain + 1, count = drainY + 1;
};

template <typename T, int KC>
__global__ void __launch_bounds__(kThreads, 1) fused_kernel(const __grid_constant__ FusedMaps maps, const __grid_constant__ FusedArgs p)
{
    typedef Fused<KC> L;
    constexpr int S = L::kStages;
    typedef Bars<S> B;
    extern __shared__ uint8_t raw[];
    const uint32_t smem = (smem_u32(raw) + 1023) & ~1023u, bars = smem + L::kBars;
    __shared__ uint32_t tmemSlot;
    __shared__ int abortFlag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = (int)cluster_rank();
    auto bar = [&](int i) { return bars + 8 * i; };

    if (threadIdx.x == 0) {
        for (int i = 0; i < B::count; ++i) {
            int arrivals = 1;
            if (i >= B::guEmpty && i < B::hEmpty)
                arrivals = 2 * kGroupWarps;             // guEmpty, hFull: one group of each CTA
            else if (i >= B::yEmpty && i < B::drain)
                arrivals = 4 * kGroupWarps;             // both groups of each CTA
            mbar_init(bar(i), arrivals);
        }
        mbar_init_fence();
        abortFlag = 0;
        prefetch_map(&maps.x), prefetch_map(&maps.wg), prefetch_map(&maps.wu), prefetch_map(&maps.wd);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(&tmemSlot), 512);
        tmem_relinquish();
        tc_fence_before();
    }
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = *const_cast<volatile uint32_t*>(&tmemSlot);
    volatile int* abort = &abortFlag;
    pdl_wait();
    pdl_launch_dependents();

    const long long rowEnd = live_rows(p.rows, p.num_blocks_dev, p.rowsPerBlock);
    const int tiles = (int)((rowEnd + kRows - 1) / kRows), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1, n = p.chunks;
    auto wait = [&](int i, uint32_t parity) { return mbar_wait_warp(bar(i), parity & 1, abort, &g_fused_timeouts); };

    if (warp == 0) {
        // ---- loads: X of a tile, then per chunk the weights of GU ----
        const bool lead = elect_one();
        const uint32_t first = in_first_cta(bars);
        uint32_t turn = 0, q = 0;
        bool ok = true;
        for (int t = pair; ok && t < tiles; t += pairs, ++turn) {
            const uint32_t xb = turn % L::kXBufs, use = turn / L::kXBufs;
            if (use > 0 && !(ok = wait(B::xEmpty + xb, use - 1)))
                break;
            if (lead) {
                if (rank == 0)
                    mbar_expect_tx(bar(B::xFull + xb), 2 * L::kXBytes);
                for (int k = 0; k < KC; ++k)
                    tma_load_2d(smem + L::kX + xb * L::kXBytes + k * kCtaRows * 128, &maps.x, k * 64, t * kRows + rank * kCtaRows,
                                first + 8 * (B::xFull + xb));
            }
            __syncwarp();
            for (int j = 0; j < n; ++j, ++q) {
                const uint32_t st = q % S, again = q / S;
                if (again > 0 && !(ok = wait(B::w1Empty + st, again - 1)))
                    break;
                if (lead) {
                    if (rank == 0)
                        mbar_expect_tx(bar(B::w1Full + st), 2 * L::kW1Bytes);
                    for (int k = 0; k < KC; ++k)
                        tma_load_2d(smem + L::kW1 + st * L::kW1Bytes + k * kChunk * 128, rank == 0 ? &maps.wg : &maps.wu, k * 64, j * kChunk,
                                    first + 8 * (B::w1Full + st));
                }
                __syncwarp();
            }
        }
        if (*abort && rank == 0) {      // shared memory is not given back with copies (of either CTA) in flight
            int own = 0;
            for (int i = 0; i < S; ++i) {
                if (q > (uint32_t)i)
                    mbar_wait_bounded(bar(B::w1Full + i), ((q - 1 - i) / S) & 1, &own, &g_fused_timeouts);
            }
            for (int i = 0; i < L::kXBufs; ++i)
                if (turn > (uint32_t)i)
                    mbar_wait_bounded(bar(B::xFull + i), ((turn - 1 - i) / L::kXBufs) & 1, &own, &g_fused_timeouts);
        }
    } else if (warp == kWdWarp) {
        // ---- loads of Wd, which is used later than GU's weights: a warp of their own keeps them from holding those up ----
        const bool lead = elect_one();
        const uint32_t first = in_first_cta(bars);
        uint32_t q = 0;
        bool ok = true;
        for (int t = pair; ok && t < tiles; t += pairs)
            for (int j = 0; j < n; ++j, ++q) {
                const uint32_t st = q % S, again = q / S;
                if (again > 0 && !(ok = wait(B::wdEmpty + st, again - 1)))
                    break;
                if (lead) {
                    if (rank == 0)
                        mbar_expect_tx(bar(B::wdFull + st), 2 * L::kWdBytes);
                    tma_load_2d(smem + L::kWd + st * L::kWdBytes, &maps.wd, j * kChunk, rank * (KC * 32), first + 8 * (B::wdFull + st));
                }
                __syncwarp();
            }
        if (*abort && rank == 0) {
            int own = 0;
            for (int i = 0; i < S; ++i)
                if (q > (uint32_t)i)
                    mbar_wait_bounded(bar(B::wdFull + i), ((q - 1 - i) / S) & 1, &own, &g_fused_timeouts);
        }
    } else if (warp == 1 && rank == 0) {
        // ---- GU's matrix instructions: the first CTA's, for both ----
        const bool lead = elect_one();
        constexpr int format = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
        constexpr uint32_t idesc = instr_desc<false, false>(format, 2 * kChunk);
        uint32_t turn = 0, q = 0, st = 0, phase = 0;
        bool ok = true;
        for (int t = pair; ok && t < tiles; t += pairs, ++turn) {
            const uint32_t xb = turn % L::kXBufs;
            if (!(ok = wait(B::xFull + xb, turn / L::kXBufs)))
                break;
            for (int j = 0; j < n; ++j, ++q) {
                const uint32_t gb = q & 1;
                if ((q >= 2 && !wait(B::guEmpty + gb, (q >> 1) - 1)) || !wait(B::w1Full + st, phase)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                if (lead) {
#pragma unroll
                    for (int k = 0; k < KC; ++k) {
                        const uint64_t da = operand_desc<false>(smem + L::kX + xb * L::kXBytes + k * kCtaRows * 128),
                                       db = operand_desc<false>(smem + L::kW1 + st * L::kW1Bytes + k * kChunk * 128);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            mma_f16(tmem + gb * 128, da + i * kDescStep<false>, db + i * kDescStep<false>, idesc, k > 0 || i > 0);
                    }
                    mma_commit_pair(bar(B::guFull + gb));
                    mma_commit_pair(bar(B::w1Empty + st));
                    if (j == n - 1)
                        mma_commit_pair(bar(B::xEmpty + xb));
                }
                __syncwarp();
                if (++st == S)
                    st = 0, phase ^= 1;
            }
        }
        if (*abort) {
            int own = 0;
            if (lead)
                mma_commit_pair(bar(B::drain));
            mbar_wait_bounded(bar(B::drain), 0, &own, &g_fused_timeouts);
        }
    } else if (warp == kYWarp && rank == 0) {
        // ---- Y's: from a warp of their own, so that neither product's waits hold up the other's instructions ----
        const bool lead = elect_one();
        constexpr int format = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
        constexpr uint32_t idesc = instr_desc<false, false>(format, L::kYCols);
        uint32_t turn = 0, q = 0, st = 0, phase = 0;
        bool ok = true;
        for (int t = pair; ok && t < tiles; t += pairs, ++turn) {
            const uint32_t yb = turn % L::kYBufs, d = tmem + 256 + yb * L::kYCols;
            if (turn >= L::kYBufs && !(ok = wait(B::yEmpty + yb, turn / L::kYBufs - 1)))
                break;
            for (int j = 0; j < n; ++j, ++q) {
                const uint32_t hb = q & 1;
                if (!wait(B::wdFull + st, phase) || !wait(B::hFull + hb, q >> 1)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                if (lead) {
                    const uint64_t da = operand_desc<false>(smem + L::kH + hb * L::kHBytes), db = operand_desc<false>(smem + L::kWd + st * L::kWdBytes);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma_f16(d, da + k * kDescStep<false>, db + k * kDescStep<false>, idesc, j > 0 || k > 0);
                    mma_commit_pair(bar(B::hEmpty + hb));
                    mma_commit_pair(bar(B::wdEmpty + st));
                    if (j == n - 1)
                        mma_commit_pair(bar(B::yFull + yb));
                }
                __syncwarp();
                if (++st == S)
                    st = 0, phase ^= 1;
            }
        }
        if (*abort) {
            int own = 0;
            if (lead)
                mma_commit_pair(bar(B::drainY));
            mbar_wait_bounded(bar(B::drainY), 0, &own, &g_fused_timeouts);
        }
    } else if (warp >= 2 && warp < kWdWarp) {
        // ---- epilogue: group 0 takes the even chunks (over all tiles), group 1 the odd ones; of a chunk's 64 columns a warp
        // has 32, of Y's columns every fourth 32 ----
        const int e = warp - 2, quarter = warp & 3, group = e >> 3, share = (e >> 2) & 1, all = group * 2 + share;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16, first = in_first_cta(bars);
        const uint32_t staging = smem + L::kStage + e * 2048;
        const int row = quarter * 32 + lane;
        const bool wide = (p.C & 7) == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0;
        uint32_t turn = 0, q = 0, stored = 0;
        bool ok = true;
        // Y of the oldest tile that is not stored yet
        auto finish = [&]() -> bool {
            if (stored == turn)
                return true;
            const uint32_t yb = stored % L::kYBufs;
            if (!wait(B::yFull + yb, stored / L::kYBufs))
                return false;
            tc_fence_after();
            const long long row0 = (long long)(pair + (int)stored * pairs) * kRows + rank * kCtaRows + quarter * 32;
#pragma unroll 1
            for (int c = all * 32; c < L::kYCols; c += 128) {
                uint32_t v[32], h[16];
                tmem_load32(tmem + lanes + 256 + yb * L::kYCols + c, v);
                tmem_wait_load();
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    h[i] = pack2<T>(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
                stage_rows(staging, lane, h);
                __syncwarp();
                store_tile<T>(p.y, spot(p.C, row0, rowEnd, c, p.C, lane), wide, staging, lane);
                __syncwarp();
            }
            tc_fence_before();
            if (lane == 0)
                mbar_arrive_cluster(first + 8 * (B::yEmpty + yb));
            __syncwarp();
            ++stored;
            return true;
        };
        for (int t = pair; ok && t < tiles; t += pairs, ++turn) {
            bool taken = false;     // a chunk of this tile: Y of the tile before is stored behind it, when it has long been done
            for (int j = 0; j < n; ++j, ++q) {
                if ((int)(q & 1) != group)
                    continue;
                if (!(ok = wait(B::guFull + group, q >> 1)))
                    break;
                tc_fence_after();
                uint32_t g[32], u[32], h[16];
                tmem_load32(tmem + lanes + group * 128 + share * 32, g);
                tmem_load32(tmem + lanes + group * 128 + 64 + share * 32, u);
                tmem_wait_load();
                tc_fence_before();
                if (lane == 0)
                    mbar_arrive_cluster(first + 8 * (B::guEmpty + group));
                __syncwarp();
                if (p.act == kSilu)
                    gate_words<T, kSilu>(g, u, h);
                else if (p.act == kGelu)
                    gate_words<T, kGelu>(g, u, h);
                else
                    gate_words<T, kRelu>(g, u, h);
                if (q >= 2 && !(ok = wait(B::hEmpty + group, (q >> 1) - 1)))
                    break;
                // K-major operand, 128-byte swizzle: 64 hidden channels of a row are 128 bytes
                const uint32_t at = smem + L::kH + group * L::kHBytes + row * 128;
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    sts128(at + (((share * 4 + c) ^ (row & 7)) << 4), make_uint4(h[4 * c], h[4 * c + 1], h[4 * c + 2], h[4 * c + 3]));
                fence_async_smem();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive_cluster_release(first + 8 * (B::hFull + group));
                __syncwarp();
                if (!taken && !(ok = finish()))
                    break;
                taken = true;
            }
            if (!ok || (!taken && !(ok = finish())))
                break;
        }
        if (ok && turn > 0)
            finish();
    }
    // every wait is bounded, so both CTAs get here; neither leaves while the other may still signal its barriers or multiply
    // out of its shared memory
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_free(tmem, 512);
    }
}

template <typename T, int KC>
cudaError_t launch(const FusedMaps& maps, const FusedArgs& p, int tiles, cudaStream_t stream)
{
    auto kernel = fused_kernel<T, KC>;
    constexpr int smem = Fused<KC>::kSmem;
    static_assert(smem <= 227 * 1024, "shared memory of one SM");
    static std::atomic<bool> done[64] = {};
    if (cudaError_t e = allow_smem(kernel, smem, done))
        return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * (unsigned)std::min(tiles, sm_count() / 2)), cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem, cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = options().pdl ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, maps, p);
}

} // namespace

// A pair takes whole row tiles, so it pays once half of the pairs have one.
bool ffn_fused_suits(long long rows, int C) { return C <= 256 && 2 * ((rows + kRows - 1) / kRows) >= sm_count() / 2; }

template <typename T>
cudaError_t launch_ffn_fused(const FfnArgs& f, const Matrix& x, const Matrix& wg, const Matrix& wu, const Matrix& wd,
                             cudaStream_t stream)
{
    const int kc = ceil_div(f.C, 64);
    FusedMaps maps;
    if (cudaError_t e = encode(x, kCtaRows, &maps.x))
        return e;
    if (cudaError_t e = encode(wg, kChunk, &maps.wg))
        return e;
    if (cudaError_t e = encode(wu, kChunk, &maps.wu))
        return e;
    if (cudaError_t e = encode(wd, kc * 32, &maps.wd))
        return e;
    FusedArgs p = {};
    p.y = f.y, p.num_blocks_dev = f.num_blocks_dev, p.rows = f.rows, p.rowsPerBlock = f.rowsPerBlock, p.C = f.C;
    p.chunks = ceil_div(f.F, kChunk), p.act = f.act;
    const int tiles = ceil_div(f.rows, kRows);
    note_site("gated_ffn (one kernel)");
    switch (kc) {
    case 1: return launch<T, 1>(maps, p, tiles, stream);
    case 2: return launch<T, 2>(maps, p, tiles, stream);
    case 3: return launch<T, 3>(maps, p, tiles, stream);
    default: return launch<T, 4>(maps, p, tiles, stream);
    }
}
template cudaError_t launch_ffn_fused<__half>(const FfnArgs&, const Matrix&, const Matrix&, const Matrix&, const Matrix&, cudaStream_t);
template cudaError_t launch_ffn_fused<__nv_bfloat16>(const FfnArgs&, const Matrix&, const Matrix&, const Matrix&, const Matrix&, cudaStream_t);

cudaError_t read_ffn_fused_wait_timeouts(unsigned int* out) { return cudaMemcpyFromSymbol(out, g_fused_timeouts, sizeof(*out)); }

} // namespace sbnet
