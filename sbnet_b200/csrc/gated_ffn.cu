// The gated feed-forward block over a list of rows, forward and backward, on the fifth-generation tensor cores:
//
//   G = X Wg^T   U = X Wu^T   H = act(G) * U   Y = H Wd^T               X [R,C], Wg and Wu [F,C], Wd [C,F]
//   dH = dY Wd   dU = dH * act(G)   dG = dH * U * act'(G)
//   dX = dG Wg + dU Wu    dWg = dG^T X    dWu = dU^T X    dWd = dY^T H
//
// One kernel, gemm_kernel, computes all of them as D[m,n] = sum_k A[m,k] B[n,k]; what differs is which
// operand's memory order has the reduction contiguous ("K-major") or not ("MN-major") and what the epilogue
// does with an accumulator tile:
//
//   kGate   both projections at once: a tile's B operand is 128 rows of Wg followed by 128 rows of Wu, so G and
//           U of the same positions come out of one instruction stream side by side in TMEM and the epilogue
//           writes H without either having been to memory (in training of many channels it also keeps G and U, in
//           fp32: rounded to 16 bits they would show in every gradient)
//   kGrad   the hidden gradients with nothing but the forward pass' inputs: a tile multiplies dH (128 columns) and
//           then G and U again (256 columns), and the epilogue takes all three from TMEM and writes H, dG and dU.
//           Costs 4 R F C of 16 R F C operations
//   kKept   the same from the kept G and U, which the epilogue reads: 16 bytes of HBM traffic per hidden element
//           instead, so it wins with many channels (8192 x 2048 x 8192 bf16: 352 us against 729)
//   kStore  a plain product, rounded once
//
// H, dG and dU are held between kernels in the type of X (they are operands of the next product, and the tensor
// cores multiply 16-bit types); accumulators and every element-wise step are fp32.
//
// Structure: persistent pairs of CTAs (one CTA per SM) over 256 x 256 (or 256 x 128) output tiles.  A pair
// multiplies as one (cta_group::2): each CTA holds its own 128 rows of A and half of B, so a stage of 64
// reduction steps costs 32 KB of L2 reads per SM where single CTAs with 128 x 256 tiles need 48 KB.  In each
// CTA one thread feeds a ring of shared-memory stages by TMA (128-byte swizzle; rows and columns past the
// matrix read as zero); one thread of the first CTA issues tcgen05.mma; eight or sixteen warps run the epilogue
// on one TMEM accumulator while the other is being filled.  Tiles are walked in groups of 8 row tiles so that the
// operands of neighbouring pairs meet in L2.  Where a product has few tiles, its reduction is split (split_count):
// every piece writes fp32 partial sums to the workspace and a second kernel adds them in a fixed order (no
// atomics: the same call gives the same bits).
//
// Measured (bf16): 4,096 rows through 4,096 x 12,288 weights 920 us, 1.34 PFLOP/s, which is 0.95 of what a long run of
// dense products sustains under the power cap; a training step of 8,192 x 2,048 x 8,192 2,151 us, 1.15 PFLOP/s; of
// 102,400 x 256 x 1,024 658 us, 190 of them for the hidden gradients (tensor pipe 0.42 busy, 574 MB written).
//
// A matrix whose rows do not start on 16-byte boundaries cannot be read by TMA; it is first copied to the
// workspace at the next pitch that can.
//
// Waits are bounded; a wait that gives up raises a CTA-wide flag, counts itself, and the CTA lets its copies and
// matrix instructions land, frees its TMEM and returns.
#include <algorithm>

#include "gated_ffn.cuh"

namespace sbnet {
namespace {

constexpr int kTileM = 256;                      // rows of a tile
constexpr int kCtaM = 128;                       // ... in each CTA of the pair
enum Epilogue { kStore, kGate, kGrad, kKept };
// Epilogue warps: the element-wise epilogues are chains of special functions, shared and global accesses, which four
// warps per scheduler hide better than two; kKept is bound by the loads of G and U, which 8 warps keep in flight in shared
// memory (8 KB each) while they work on the 8 KB before.
template <int EPI> constexpr int kEpiWarps = EPI == kStore || EPI == kKept ? 8 : 16;
template <int EPI> constexpr int kGemmThreads = (2 + kEpiWarps<EPI>) * 32;
// 32 x 32 tiles of 16-bit elements (2 KB) that a warp stages between registers and memory
template <int EPI> constexpr int kStaged = EPI == kStore ? 1 : EPI == kKept ? 8 : EPI == kGrad ? 3 : 2;
template <int EPI> constexpr int kStagingBytes = kEpiWarps<EPI> * kStaged<EPI> * 2048;
constexpr int kGroupM = 8;

__device__ unsigned int g_ffn_timeouts = 0;

struct Maps {
    CUtensorMap a[2], b[2], c;     // c: kGrad's Wd
    CUtensorMap out, g, u;         // H and the kept G and U, which kGate writes by TMA
};

struct Plan {
    int mTiles, nTiles;            // tiles of D
    FastDiv perGroup;              // kGroupM * nTiles
    int batch;                     // products of one shape in this launch: product z reads a[z], b[z], writes out[z]
    int segs;                      // reduction segments: segment s reads a[s], b[s]  (batch == 1)
    int kIters;                    // stages of one segment
    int splits;                    // pieces of the reduction (> 1: fp32 partials)
    int N;                         // columns of the output
    long long M;                   // rows of the output
    const int32_t* num_blocks_dev; // live rows = min(count * rowsPerBlock, M), or nullptr
    int rowsPerBlock;
    int act;
    void* out[2];                  // kStore: D of product z.  kGate: H
    long long ldo;
    float *gate, *up;              // kGate: written unless null, kKept: read; pitch ldo
    void *hid, *dgate, *dup;       // kGrad, kKept: written, pitch ldo
    float* partials;               // splits > 1: [splits][batch][mTiles * 256][nTiles * BN]
};

template <int EPI, int BN> constexpr int kStages = EPI == kGate ? 5 : EPI == kGrad ? 4 : EPI == kKept ? 3 : BN == 256 ? 6 : 8;
template <int BN> constexpr int kStageBytes = (kCtaM + BN / 2) * kStepK * 2;    // of one CTA
template <int EPI, int BN> constexpr int kGemmSmem = 1024 + kStages<EPI, BN> * kStageBytes<BN> + kStagingBytes<EPI> + 256;

template <typename T, int ACT>
__device__ __forceinline__ void gate_chunk(const uint32_t (&g)[32], const uint32_t (&u)[32], uint32_t (&h)[16])
{
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        F2 a, unused;
        activate2<ACT, false>(words(g[2 * i], g[2 * i + 1]), a, unused);
        h[i] = pack2<T>(mul2(a, words(u[2 * i], u[2 * i + 1])));
    }
}
// H, dG and dU of 16 columns
template <typename T, int ACT>
__device__ __forceinline__ void grad_chunk(const uint32_t (&dh)[16], const uint32_t (&g)[16], const uint32_t (&u)[16], uint32_t (&h)[8],
                                             uint32_t (&dg)[8], uint32_t (&du)[8])
{
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const F2 d = words(dh[2 * i], dh[2 * i + 1]), up = words(u[2 * i], u[2 * i + 1]);
        F2 a, slope;
        activate2<ACT, true>(words(g[2 * i], g[2 * i + 1]), a, slope);
        h[i] = pack2<T>(mul2(a, up));
        du[i] = pack2<T>(mul2(d, a));
        dg[i] = pack2<T>(mul2(mul2(d, up), slope));
    }
}

// A staged tile into one of the scratch matrices (rows past the live ones, inside the matrix, may be written: nobody
// reads them).
__device__ __forceinline__ void send_tile(const CUtensorMap* map, uint32_t buf, int col0, int row0, int lane)
{
    fence_async_smem();
    __syncwarp();
    if (lane == 0) {
        tma_store_2d(map, buf, col0, row0);
        bulk_commit();
    }
}
// Before a warp stages into a buffer again: all but the last KEEP tiles it sent have been read.
template <int KEEP> __device__ __forceinline__ void wait_sent(int lane)
{
    if (lane == 0)
        bulk_wait_read<KEEP>();
    __syncwarp();
}

struct Tile {
    int m, n, z, s;
};
__device__ __forceinline__ Tile tile_at(int t, const Plan& p, int mTiles)
{
    Tile r;
    r.z = r.s = 0;
    if (p.batch * p.splits > 1) {
        const int plane = mTiles * p.nTiles, q = t / plane;
        t -= q * plane;
        r.s = q / p.batch, r.z = q - r.s * p.batch;
    }
    uint32_t group, inside;
    p.perGroup.divmod((uint32_t)t, group, inside);
    const int rows = mTiles - (int)group * kGroupM;
    if (rows >= kGroupM) {
        r.n = (int)(inside / kGroupM), r.m = (int)(group * kGroupM + inside % kGroupM);
    } else {        // the last group
        r.n = (int)inside / rows, r.m = (int)group * kGroupM + (int)inside - r.n * rows;
    }
    return r;
}

// A_MN / B_MN: the operand's reduction runs along its rows' pitch, not along its rows.
template <typename T, bool A_MN, bool B_MN, int EPI, int BN>
__global__ void __launch_bounds__(kGemmThreads<EPI>, 1) gemm_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Plan p)
{
    constexpr int S = kStages<EPI, BN>, W = kEpiWarps<EPI>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem = (smem_u32(smem_raw) + 1023) & ~1023u;
    const uint32_t staging = smem + S * kStageBytes<BN>;
    const uint32_t bars = staging + kStagingBytes<EPI>;           // full[S], empty[S], accFull[2], accEmpty[2], drain
    const uint32_t full = bars, empty = bars + 8 * S, accFull = bars + 16 * S, accEmpty = accFull + 16, drain = accEmpty + 16;
    __shared__ uint32_t tmemSlot;
    __shared__ int abortFlag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank();      // of this CTA in its pair

    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i)
            mbar_init(full + 8 * i, 1), mbar_init(empty + 8 * i, 1);
        for (int i = 0; i < 2; ++i)
            mbar_init(accFull + 8 * i, 1), mbar_init(accEmpty + 8 * i, 2 * W);
        mbar_init(drain, 1);
        mbar_init_fence();
        abortFlag = 0;
        for (int i = 0; i < 2; ++i)
            prefetch_map(&maps.a[i]), prefetch_map(&maps.b[i]);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(&tmemSlot), 2 * BN);
        tmem_relinquish();
        tc_fence_before();
    }
    __syncthreads();
    cluster_sync();     // the other CTA's barriers are initialised too
    tc_fence_after();
    const uint32_t tmem = *const_cast<volatile uint32_t*>(&tmemSlot);
    volatile int* abort = &abortFlag;
    pdl_wait();
    pdl_launch_dependents();

    const long long rowEnd = live_rows(p.M, p.num_blocks_dev, p.rowsPerBlock);
    const int mTiles = (int)((rowEnd + kTileM - 1) / kTileM);
    const int tiles = mTiles * p.nTiles * p.batch * p.splits;
    const int kAll = p.kIters * p.segs;

    // The two single-thread roles run their loops as whole warps (addresses stay in uniform registers) and let one
    // lane issue.
    if (warp == 0) {
        // ---- producer ----
        // The second CTA's copies are counted on the first CTA's barrier as well: bytes may arrive there before the
        // stage's count has been announced, but a stage is not filled again before both CTAs know it was consumed.
        const uint32_t fullFirst = in_first_cta(full);
        const bool lead = elect_one();
        uint32_t issued = 0;
        bool ok = true;
        for (int t = blockIdx.x >> 1; ok && t < tiles; t += gridDim.x >> 1) {
            const Tile w = tile_at(t, p, mTiles);
            const int k0 = (int)((long long)kAll * w.s / p.splits), k1 = (int)((long long)kAll * (w.s + 1) / p.splits);
            const int row = w.m * kTileM + rank * kCtaM;
            for (int k = k0; k < k1; ++k, ++issued) {
                const uint32_t st = issued % S, turn = issued / S;
                if (turn > 0 && !mbar_wait_warp(empty + 8 * st, (turn - 1) & 1, abort, &g_ffn_timeouts)) {
                    ok = false;
                    break;
                }
                const int seg = p.segs > 1 ? k / p.kIters : 0;
                const int kk = (k - seg * p.kIters) * kStepK;
                const int which = p.segs > 1 ? seg : w.z;
                const uint32_t a = smem + st * kStageBytes<BN>, b = a + kCtaM * kStepK * 2, bar = fullFirst + 8 * st;
                if (lead && EPI == kGrad) {    // segment 0: dY and 64 columns of Wd; segment 1: X and 128 rows of Wg or Wu
                    if (rank == 0)
                        mbar_expect_tx(full + 8 * st, seg == 0 ? 2 * (kCtaM + 64) * kStepK * 2 : 2 * kStageBytes<BN>);
                    tma_load_2d(a, &maps.a[seg], kk, row, bar);
                    if (seg == 0)
                        tma_load_2d(b, &maps.c, w.n * 128 + rank * 64, kk, bar);
                    else
                        tma_load_2d(b, &maps.b[rank], kk, w.n * 128, bar);
                } else if (lead) {
                    if (rank == 0)
                        mbar_expect_tx(full + 8 * st, 2 * kStageBytes<BN>);
                    if (A_MN) {
                        for (int i = 0; i < kCtaM / 64; ++i)
                            tma_load_2d(a + i * 8192, &maps.a[which], row + i * 64, kk, bar);
                    } else {
                        tma_load_2d(a, &maps.a[which], kk, row, bar);
                    }
                    if (EPI == kGate) {     // Wg's rows are the first CTA's half of B, Wu's the second's
                        tma_load_2d(b, &maps.b[rank], kk, w.n * 128, bar);
                    } else if (B_MN) {
                        for (int i = 0; i < BN / 2 / 64; ++i)
                            tma_load_2d(b + i * 8192, &maps.b[which], w.n * BN + rank * (BN / 2) + i * 64, kk, bar);
                    } else {
                        tma_load_2d(b, &maps.b[which], kk, w.n * BN + rank * (BN / 2), bar);
                    }
                }
                __syncwarp();
            }
        }
        if (*abort && rank == 0) {   // shared memory is not given back with copies (of either CTA) in flight
            int own = 0;
            for (uint32_t i = issued > S ? issued - S : 0; i < issued; ++i)
                mbar_wait_bounded(full + 8 * (i % S), (i / S) & 1, &own, &g_ffn_timeouts);
        }
    } else if (warp == 1 && rank == 0) {
        // ---- matrix instructions: the first CTA's, for both ----
        constexpr uint32_t idesc0 = instr_desc<A_MN, B_MN>(0, BN), idesc1 = instr_desc<A_MN, B_MN>(1, BN);
        constexpr uint32_t idesc = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? idesc1 : idesc0;
        const bool lead = elect_one();
        uint32_t used = 0, turn = 0;
        bool ok = true;
        for (int t = blockIdx.x >> 1; ok && t < tiles; t += gridDim.x >> 1, ++turn) {
            const Tile w = tile_at(t, p, mTiles);
            const int k0 = (int)((long long)kAll * w.s / p.splits), k1 = (int)((long long)kAll * (w.s + 1) / p.splits);
            // kGrad: G and U have columns 0 .. 255, dH 256 .. 383 or 384 .. 511 in turn, and one pair of barriers
            const uint32_t acc = EPI == kGrad ? 0 : turn & 1, d = EPI == kGrad ? tmem + 256 + 128 * (turn & 1) : tmem + acc * BN;
            if (EPI != kGrad && turn > 1 && !mbar_wait_warp(accEmpty + 8 * acc, ((turn >> 1) - 1) & 1, abort, &g_ffn_timeouts))
                break;
            tc_fence_after();
            for (int k = k0; k < k1; ++k, ++used) {
                const uint32_t st = used % S;
                if (!mbar_wait_warp(full + 8 * st, (used / S) & 1, abort, &g_ffn_timeouts)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t a = smem + st * kStageBytes<BN>;
                if constexpr (EPI == kGrad) {
                    // dH of the next tile is multiplied while the epilogue still reads G and U of this one
                    if (k == p.kIters) {
                        if (turn > 0 && !mbar_wait_warp(accEmpty, (turn - 1) & 1, abort, &g_ffn_timeouts)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                    }
                    constexpr int format = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
                    if (lead) {
                        const uint64_t da = operand_desc<false>(a);
                        if (k < p.kIters) {
                            const uint64_t db = operand_desc<true>(a + kCtaM * kStepK * 2);
#pragma unroll
                            for (int j = 0; j < kStepK / 16; ++j)
                                mma_f16(d, da + j * kDescStep<false>, db + j * kDescStep<true>, instr_desc<false, true>(format, 128), k > 0 || j > 0);
                        } else {
                            const uint64_t db = operand_desc<false>(a + kCtaM * kStepK * 2);
#pragma unroll
                            for (int j = 0; j < kStepK / 16; ++j)
                                mma_f16(tmem, da + j * kDescStep<false>, db + j * kDescStep<false>, instr_desc<false, false>(format, 256),
                                        k > p.kIters || j > 0);
                        }
                        mma_commit_pair(empty + 8 * st);
                    }
                    __syncwarp();
                    continue;
                }
                const uint64_t da = operand_desc<A_MN>(a), db = operand_desc<B_MN>(a + kCtaM * kStepK * 2);
                if (lead) {
#pragma unroll
                    for (int j = 0; j < kStepK / 16; ++j)
                        mma_f16(d, da + j * kDescStep<A_MN>, db + j * kDescStep<B_MN>, idesc, k > k0 || j > 0);
                    mma_commit_pair(empty + 8 * st);
                }
                __syncwarp();
            }
            if (ok && lead)
                mma_commit_pair(accFull + 8 * acc);
            __syncwarp();
        }
        if (*abort) {
            int own = 0;
            if (lead)
                mma_commit_pair(drain);
            mbar_wait_bounded(drain, 0, &own, &g_ffn_timeouts);
        }
    } else if (warp >= 2) {
        // ---- epilogue: warp w may touch TMEM lanes 32 (w % 4) ..; W / 4 warps share each quarter and split its columns ----
        const int quarter = warp & 3, share = (warp - 2) >> 2;
        const uint32_t buf0 = staging + (warp - 2) * (kStaged<EPI> * 2048), buf1 = buf0 + 2048, buf2 = buf0 + 4096;
        const uint32_t accEmptyFirst = in_first_cta(accEmpty);
        uint32_t turn = 0, sent = 0;
        // kKept: copies this warp's 32 rows x 32 columns of G and U, from column c of its share of a tile.  What lies outside
        // the matrix is copied in whole 16-byte pieces or not at all; it only reaches results that are not stored
        constexpr int kKeptCols = BN * 4 / W;
        auto keptAhead = [&](uint32_t slot, const Tile& w, int c) {
            const long long row = (long long)w.m * kTileM + rank * kCtaM + quarter * 32 + (lane >> 2);
            const int col = w.n * BN + share * kKeptCols + c + (lane & 3) * 4;
            const float *g = p.gate + row * p.ldo + col, *u = p.up + row * p.ldo + col;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    if (row + 8 * i < rowEnd && col + 16 * k < p.N) {
                        const uint32_t dst = piece(slot + k * 4096, i * 8 + (lane >> 2), lane & 3);
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(g + 8 * i * p.ldo + 16 * k) : "memory");
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + 2048), "l"(u + 8 * i * p.ldo + 16 * k) : "memory");
                    }
        };
        if (EPI == kKept && (int)(blockIdx.x >> 1) < tiles) {
            keptAhead(buf0, tile_at(blockIdx.x >> 1, p, mTiles), 0);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        for (int t = blockIdx.x >> 1; t < tiles; t += gridDim.x >> 1, ++turn) {
            const Tile w = tile_at(t, p, mTiles);
            const uint32_t acc = EPI == kGrad ? 0 : turn & 1, d = tmem + acc * BN + ((uint32_t)(quarter * 32) << 16);
            if (!mbar_wait_warp(accFull + 8 * acc, (EPI == kGrad ? turn : turn >> 1) & 1, abort, &g_ffn_timeouts))
                break;
            tc_fence_after();
            const long long row0 = (long long)w.m * kTileM + rank * kCtaM + quarter * 32;
            // after the last read of the accumulator: the next tile may be multiplied into it
            auto release = [&] {
                tc_fence_before();
                if (lane == 0)
                    mbar_arrive_cluster(accEmptyFirst + 8 * acc);
                __syncwarp();
            };
            if (p.splits > 1) {
                float* part = p.partials + ((long long)w.s * p.batch + w.z) * p.mTiles * kTileM * (p.nTiles * BN) +
                              (row0 + lane) * (p.nTiles * BN) + w.n * BN + share * (BN * 4 / W);
#pragma unroll 1
                for (int c = 0; c < BN * 4 / W; c += 32) {
                    uint32_t v[32];
                    tmem_load32(d + share * (BN * 4 / W) + c, v);
                    tmem_wait_load();
                    if (c + 32 == BN * 4 / W)
                        release();
                    if (row0 + lane < rowEnd)
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        *reinterpret_cast<uint4*>(part + c + 4 * i) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                }
            } else if (EPI == kGate) {
#pragma unroll 1
                for (int c = share * (512 / W); c < (share + 1) * (512 / W); c += 32) {
                    uint32_t g[32], u[32], h[16];
                    tmem_load32(d + c, g);
                    tmem_load32(d + 128 + c, u);
                    tmem_wait_load();
                    if (c + 32 == (share + 1) * (512 / W))
                        release();
                    if (p.act == kSilu)
                        gate_chunk<T, kSilu>(g, u, h);
                    else if (p.act == kGelu)
                        gate_chunk<T, kGelu>(g, u, h);
                    else
                        gate_chunk<T, kRelu>(g, u, h);
                    const int col = w.n * 128 + c;
                    wait_sent<1>(lane);     // the two buffers in turn
                    stage_rows(sent & 1 ? buf1 : buf0, lane, h);
                    send_tile(&maps.out, sent++ & 1 ? buf1 : buf0, col, (int)row0, lane);
                    if (p.gate != nullptr) {        // 16 columns of fp32 are as wide as 32 of 16 bits
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t* v = (i < 2 ? g : u) + 16 * (i & 1);
                            wait_sent<1>(lane);
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                sts128(piece(sent & 1 ? buf1 : buf0, lane, k), make_uint4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]));
                            send_tile(i < 2 ? &maps.g : &maps.u, sent++ & 1 ? buf1 : buf0, col + 16 * (i & 1), (int)row0, lane);
                        }
                    }
                }
            } else if (EPI == kGrad) {     // one chunk of 32 columns a warp: TMEM is free again after three loads
                const int c = share * 32;
#pragma unroll
                for (int i = 0; i < 2; ++i) {       // 16 columns at a time: 32 of all three would not fit the registers
                    uint32_t dh[16], g[16], u[16], h[8], dg[8], du[8];
                    tmem_load16(d + c + 16 * i, g);
                    tmem_load16(d + 128 + c + 16 * i, u);
                    tmem_load16(d + 256 + 128 * (turn & 1) + c + 16 * i, dh);
                    tmem_wait_load();
                    if (i == 1)
                        release();
                    if (p.act == kSilu)
                        grad_chunk<T, kSilu>(dh, g, u, h, dg, du);
                    else if (p.act == kGelu)
                        grad_chunk<T, kGelu>(dh, g, u, h, dg, du);
                    else
                        grad_chunk<T, kRelu>(dh, g, u, h, dg, du);
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        sts128(piece(buf0, lane, 2 * i + q), make_uint4(h[4 * q], h[4 * q + 1], h[4 * q + 2], h[4 * q + 3]));
                        sts128(piece(buf1, lane, 2 * i + q), make_uint4(dg[4 * q], dg[4 * q + 1], dg[4 * q + 2], dg[4 * q + 3]));
                        sts128(piece(buf2, lane, 2 * i + q), make_uint4(du[4 * q], du[4 * q + 1], du[4 * q + 2], du[4 * q + 3]));
                    }
                }
                __syncwarp();
                const Spot at = spot(p.ldo, row0, rowEnd, w.n * 128 + c, p.N, lane);
                store_tile<T>(p.hid, at, true, buf0, lane);
                store_tile<T>(p.dgate, at, true, buf1, lane);
                store_tile<T>(p.dup, at, true, buf2, lane);
                __syncwarp();
            } else if (EPI == kKept) {      // 32 columns at a time from one of two slots, the next 32 copying into the other
#pragma unroll 1
                for (int c = 0; c < kKeptCols; c += 32, ++sent) {
                    const uint32_t slot = buf0 + (sent & 1) * 8192;       // G and U of 16 columns, then of the next 16
                    if (c + 32 < kKeptCols)
                        keptAhead(buf0 + (~sent & 1) * 8192, w, c + 32);
                    else if (t + (int)(gridDim.x >> 1) < tiles)
                        keptAhead(buf0 + (~sent & 1) * 8192, tile_at(t + (gridDim.x >> 1), p, mTiles), 0);
                    asm volatile("cp.async.commit_group;" ::: "memory");
                    asm volatile("cp.async.wait_group 1;" ::: "memory");
                    __syncwarp();
                    uint32_t h[16], dg[16], du[16];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        uint32_t dh[16], g[16], u[16], hh[8], gg[8], uu[8];
                        tmem_load16(d + share * kKeptCols + c + 16 * i, dh);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint4 a = lds128(piece(slot + i * 4096, lane, k)), b = lds128(piece(slot + i * 4096 + 2048, lane, k));
                            g[4 * k] = a.x, g[4 * k + 1] = a.y, g[4 * k + 2] = a.z, g[4 * k + 3] = a.w;
                            u[4 * k] = b.x, u[4 * k + 1] = b.y, u[4 * k + 2] = b.z, u[4 * k + 3] = b.w;
                        }
                        // column N of an odd N is padding, whatever it holds, and silu shares a reciprocal between columns N - 1
                        // and N: zero, as the recomputing form has it
                        const int past = p.N - (w.n * BN + share * kKeptCols + c + 16 * i);
                        if (p.N & 1)
#pragma unroll
                            for (int k = 1; k < 16; k += 2)
                                g[k] = k == past ? 0 : g[k];
                        tmem_wait_load();
                        if (c + 16 * i + 16 == kKeptCols)
                            release();
                        if (p.act == kSilu)
                            grad_chunk<T, kSilu>(dh, g, u, hh, gg, uu);
                        else if (p.act == kGelu)
                            grad_chunk<T, kGelu>(dh, g, u, hh, gg, uu);
                        else
                            grad_chunk<T, kRelu>(dh, g, u, hh, gg, uu);
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            h[8 * i + k] = hh[k], dg[8 * i + k] = gg[k], du[8 * i + k] = uu[k];
                    }
                    __syncwarp();       // the slot has been read: the results are staged in it
                    const Spot at = spot(p.ldo, row0, rowEnd, w.n * BN + share * kKeptCols + c, p.N, lane);
                    stage_rows(slot, lane, h);
                    stage_rows(slot + 2048, lane, dg);
                    stage_rows(slot + 4096, lane, du);
                    __syncwarp();
                    store_tile<T>(p.hid, at, true, slot, lane);
                    store_tile<T>(p.dgate, at, true, slot + 2048, lane);
                    store_tile<T>(p.dup, at, true, slot + 4096, lane);
                    __syncwarp();       // before the slot is copied into again
                }
            } else {
                T* out = static_cast<T*>(p.out[w.z]);
                const bool wide = ((p.ldo & 7) == 0) && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
#pragma unroll 1
                for (int c = share * (BN * 4 / W); c < (share + 1) * (BN * 4 / W); c += 32) {
                    uint32_t v[32], h[16];
                    tmem_load32(d + c, v);
                    tmem_wait_load();
                    if (c + 32 == (share + 1) * (BN * 4 / W))
                        release();
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        h[i] = pack2<T>(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
                    stage_rows(buf0, lane, h);
                    __syncwarp();
                    store_tile<T>(out, spot(p.ldo, row0, rowEnd, w.n * BN + c, p.N, lane), wide, buf0, lane);
                    __syncwarp();
                }
            }
        }
        if (EPI == kKept)
            asm volatile("cp.async.wait_all;" ::: "memory");     // none is left but after a wait that gave up
        if (EPI == kGate && lane == 0)
            bulk_wait_all();     // shared memory is read until then
    }
    // every role's waits are bounded, so both CTAs get here; neither frees TMEM or leaves while the other may still
    // signal its barriers or multiply out of its shared memory
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_free(tmem, 2 * BN);
    }
}

// Adds the partial sums of a split reduction in the order of the pieces and finishes the elements as the epilogue
// would have.  A thread takes four neighbouring columns of a row; blocks of 32 x 8 threads cover 128 columns x 8 rows.
__device__ __forceinline__ float4 sum_pieces(const float* q, long long step, int pieces)
{
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = 0; s < pieces; ++s) {
        const float4 w = *reinterpret_cast<const float4*>(q + s * step);
        v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
    }
    return v;
}
template <typename T> __device__ __forceinline__ void store4(T* dst, float4 v, int n, bool wide)
{
    if (wide && n >= 4) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
        return;
    }
    const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < n)
            dst[i] = T(e[i]);
}
template <typename T, int EPI> __global__ void __launch_bounds__(256) finish_kernel(const __grid_constant__ Plan p, int bn)
{
    pdl_wait();
    pdl_launch_dependents();
    const long long rowEnd = live_rows(p.M, p.num_blocks_dev, p.rowsPerBlock);
    const long long pitch = (long long)p.nTiles * bn, plane = (long long)p.mTiles * kTileM * pitch;
    const int col = blockIdx.x * 128 + threadIdx.x * 4, z = blockIdx.z, n = p.N - col;
    if (n <= 0)
        return;
    T* out = static_cast<T*>(p.out[z]);
    const bool wide = (p.ldo & 3) == 0 && (reinterpret_cast<uintptr_t>(out) & 7) == 0;
    for (long long row = (long long)blockIdx.y * 8 + threadIdx.y; row < rowEnd; row += (long long)gridDim.y * 8) {
        if (EPI == kGate) {
            const float* q = p.partials + row * pitch + (col >> 7) * 256 + (col & 127);
            const float4 g = sum_pieces(q, plane, p.splits), u = sum_pieces(q + 128, plane, p.splits);
            float4 h;
            auto gated = [&](float a, float b) { return activate_any(p.act, a) * b; };
            h.x = gated(g.x, u.x), h.y = gated(g.y, u.y), h.z = gated(g.z, u.z), h.w = gated(g.w, u.w);
            store4<T>(out + row * p.ldo + col, h, n, wide);
            if (p.gate != nullptr) {        // the pitch is a multiple of 8
                *reinterpret_cast<float4*>(p.gate + row * p.ldo + col) = g;
                *reinterpret_cast<float4*>(p.up + row * p.ldo + col) = u;
            }
        } else {
            const float4 v = sum_pieces(p.partials + z * plane + row * pitch + col, p.batch * plane, p.splits);
            store4<T>(out + row * p.ldo + col, v, n, wide);
        }
    }
}

// Copies matrices of 16-bit elements to another pitch (a multiple of 8), all of a call's in one launch: grid.y is the
// matrix, a warp takes a row.
constexpr int kMaxRepack = 5;
struct Repack {
    const uint16_t* src[kMaxRepack];
    uint16_t* dst[kMaxRepack];
    long long rows[kMaxRepack];
    int cols[kMaxRepack], ld[kMaxRepack];
};
__global__ void __launch_bounds__(256) repack_kernel(const __grid_constant__ Repack r)
{
    pdl_wait();
    pdl_launch_dependents();
    const int m = blockIdx.y, lane = threadIdx.x & 31, cols = r.cols[m];
    for (long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); row < r.rows[m]; row += (long long)gridDim.x * 8) {
        const uint16_t* src = r.src[m] + row * cols;
        uint16_t* dst = r.dst[m] + row * r.ld[m];
#pragma unroll 4
        for (int c = lane; c < cols; c += 32)
            dst[c] = src[c];
    }
}

// ---- host side -------------------------------------------------------------------------------------------
// Column tile of a plain product: 256 wide unless the matrix is narrow.
int tile_n(int N) { return N <= 128 ? 128 : 256; }

// Pieces of the reduction: what a small model of the two kernels' times says is quickest.  A round of tiles over the
// pairs of SMs costs 0.35 us a stage (tensor cores under the power cap; a stage's B from HBM takes as long) and 1.5 us
// to fill and drain; adding up pieces costs a launch, 4 us, and the partial sums' way to memory and back at 2.5 TB/s.
int split_count(long long rows, long long N, long long tiles, int kIters)
{
    const int pairs = sm_count() / 2;
    int best = 1;
    double least = 1e30;
    for (int s = 1; s <= 64 && (s == 1 || kIters / s >= 4); ++s) {
        const double rounds = (double)((tiles * s + pairs - 1) / pairs);
        double t = rounds * ((double)((kIters + s - 1) / s) * 0.35 + 1.5);
        if (s > 1)
            t += 4 + 8e-6 * (double)s * (double)rows * (double)N / 2.5;
        if (t < least * 0.97)
            least = t, best = s;
    }
    return best;
}

template <typename T, bool A_MN, bool B_MN, int EPI, int BN>
cudaError_t launch_maps(const Maps& maps, Plan& p, cudaStream_t stream)
{
    auto kernel = gemm_kernel<T, A_MN, B_MN, EPI, BN>;
    static std::atomic<bool> done[64] = {};
    if (cudaError_t e = allow_smem(kernel, kGemmSmem<EPI, BN>, done))
        return e;
    const long long tiles = (long long)p.mTiles * p.nTiles * p.batch * p.splits;
    p.perGroup = FastDiv((uint32_t)(kGroupM * p.nTiles));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * (unsigned)std::min<long long>(tiles, sm_count() / 2)), cfg.blockDim = dim3(kGemmThreads<EPI>);
    cfg.dynamicSmemBytes = kGemmSmem<EPI, BN>, cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = options().pdl ? 2 : 1;
    if (cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, maps, p))
        return e;
    if (p.splits == 1)
        return cudaSuccess;
    const dim3 fgrid((unsigned)ceil_div(p.N, 128), (unsigned)std::min<long long>((p.M + 7) / 8, 65535), (unsigned)p.batch);
    if constexpr (EPI == kStore || EPI == kGate)
        return launch_pdl(finish_kernel<T, EPI>, fgrid, dim3(32, 8), 0, stream, p, BN);
    return cudaErrorInvalidValue;
}

template <typename T, bool A_MN, bool B_MN, int EPI, int BN>
cudaError_t launch_gemm(const Matrix (&a)[2], const Matrix (&b)[2], Plan& p, cudaStream_t stream)
{
    Maps maps;
    const int n = std::max(p.batch, p.segs);
    for (int i = 0; i < n; ++i)
        if (cudaError_t e = encode(a[i], A_MN ? kStepK : kCtaM, &maps.a[i]))
            return e;
    for (int i = 0; i < (EPI == kGate ? 2 : n); ++i) {
        if (i > 0 && b[i].ptr == b[0].ptr)
            maps.b[i] = maps.b[0];
        else if (cudaError_t e = encode(b[i], B_MN ? kStepK : BN / 2, &maps.b[i]))
            return e;
    }
    if (n == 1)     // the kernel never reads the second map, but prefetches both
        maps.a[1] = maps.a[0];
    if (n == 1 && EPI != kGate)
        maps.b[1] = maps.b[0];
    if (EPI == kGate && p.splits == 1)
    {
        if (cudaError_t e = encode({p.out[0], p.M, p.N, p.ldo}, 32, &maps.out, 32))
            return e;
        if (p.gate != nullptr) {
            if (cudaError_t e = encode({p.gate, p.M, p.N, p.ldo}, 32, &maps.g, 16, 4))
                return e;
            if (cudaError_t e = encode({p.up, p.M, p.N, p.ldo}, 32, &maps.u, 16, 4))
                return e;
        }
    }
    return launch_maps<T, A_MN, B_MN, EPI, BN>(maps, p, stream);
}

// Hidden gradients.
template <typename T>
cudaError_t launch_grad(const Matrix& dy, const Matrix& x, const Matrix& wd, const Matrix& wg, const Matrix& wu, Plan& p, cudaStream_t stream)
{
    Maps maps;
    if (cudaError_t e = encode(dy, kCtaM, &maps.a[0]))
        return e;
    if (cudaError_t e = encode(x, kCtaM, &maps.a[1]))
        return e;
    if (cudaError_t e = encode(wg, 128, &maps.b[0]))
        return e;
    if (cudaError_t e = encode(wu, 128, &maps.b[1]))
        return e;
    if (cudaError_t e = encode(wd, kStepK, &maps.c))
        return e;
    return launch_maps<T, false, false, kGrad, 256>(maps, p, stream);
}

// A plain product D[m,n] of one or two products (batch) or segments.
template <typename T, bool A_MN, bool B_MN>
cudaError_t product(const Matrix (&a)[2], const Matrix (&b)[2], int batch, int segs, long long M, int N, long long K,
                    void* out0, void* out1, float* partials, const FfnArgs& f, bool rowsOfX, cudaStream_t stream)
{
    Plan p = {};
    const int bn = tile_n(N);
    p.mTiles = ceil_div(M, kTileM), p.nTiles = ceil_div(N, bn), p.batch = batch, p.segs = segs;
    p.kIters = ceil_div(K, kStepK);
    p.splits = split_count(M, (long long)N * batch, (long long)p.mTiles * p.nTiles * batch, p.kIters * segs);
    p.N = N, p.M = M, p.out[0] = out0, p.out[1] = out1, p.ldo = N, p.partials = partials;
    if (rowsOfX)
        p.num_blocks_dev = f.num_blocks_dev, p.rowsPerBlock = f.rowsPerBlock;
    return bn == 128 ? launch_gemm<T, A_MN, B_MN, kStore, 128>(a, b, p, stream)
                     : launch_gemm<T, A_MN, B_MN, kStore, 256>(a, b, p, stream);
}
size_t product_partials(int batch, int segs, long long M, int N, long long K)
{
    const int bn = tile_n(N);
    const long long mT = ceil_div(M, kTileM), nT = ceil_div(N, bn);
    const int s = split_count(M, (long long)N * batch, mT * nT * batch, ceil_div(K, kStepK) * segs);
    return s == 1 ? 0 : sizeof(float) * s * batch * mT * kTileM * nT * bn;
}
size_t gate_partials(long long R, int F, int C)
{
    const long long mT = ceil_div(R, kTileM), nT = ceil_div(F, 128);
    const int s = split_count(R, 2ll * F, mT * nT, ceil_div(C, kStepK));
    return s == 1 ? 0 : sizeof(float) * s * mT * kTileM * nT * 256;
}

// Hands out the caller's workspace in 256-byte aligned pieces; without a base it only counts.
struct Bump {
    uint8_t* base;
    size_t used;
    void* take(size_t bytes)
    {
        void* p = base == nullptr ? nullptr : base + used;
        used += (bytes + 255) & ~(size_t)255;
        return p;
    }
};
int padded(int n) { return (n + 7) & ~7; }

struct Layout {
    Bump bump;
    bool aligned;      // base addresses are multiples of 16
    // pitch at which a [rows, cols] input is read, and room for a copy where that is not its own pitch
    Matrix plan(const void* src, long long rows, int cols)
    {
        Matrix m = {src, rows, cols, cols};
        const bool fits = cols % 8 == 0 && (bump.base == nullptr ? aligned : (reinterpret_cast<uintptr_t>(src) & 15) == 0);
        if (!fits) {
            m.ld = padded(cols);
            m.ptr = bump.take((size_t)rows * m.ld * 2);
        }
        return m;
    }
};
struct Repacks {
    Repack r = {};
    int n = 0;
    long long most = 0;
    void add(const void* src, const Matrix& m)
    {
        if (m.ptr == src)
            return;
        r.src[n] = static_cast<const uint16_t*>(src), r.dst[n] = static_cast<uint16_t*>(const_cast<void*>(m.ptr));
        r.rows[n] = m.rows, r.cols[n] = m.cols, r.ld[n] = (int)m.ld;
        most = std::max(most, m.rows), ++n;
    }
    cudaError_t run(cudaStream_t stream) const
    {
        if (n == 0)
            return cudaSuccess;
        const unsigned grid = (unsigned)std::min<long long>((most + 7) / 8, (long long)sm_count() * 8);
        return launch_pdl(repack_kernel, dim3(grid, n), dim3(256), 0, stream, r);
    }
};

#define SBNET_TRY(call)                  \
    do {                                 \
        if (cudaError_t e_ = (call))     \
            return e_;                   \
    } while (0)

// run == false: only counts the workspace.
template <typename T> cudaError_t forward(const FfnArgs& f, Layout& l, bool run, cudaStream_t stream)
{
    const long long R = f.rows;
    const int C = f.C, F = f.F, Fp = padded(F);
    const Matrix x = l.plan(f.x, R, C), wg = l.plan(f.w_gate, F, C), wu = l.plan(f.w_up, F, C), wd = l.plan(f.w_down, C, F);
    const bool fused = f.kept == nullptr && ffn_fused_suits(R, C);      // needs neither H nor partial sums
    const Matrix h = {fused ? nullptr : l.bump.take((size_t)R * Fp * 2), R, F, Fp};
    float* parts = fused ? nullptr : static_cast<float*>(l.bump.take(std::max(gate_partials(R, F, C), product_partials(1, 1, R, C, F))));
    if (!run)
        return cudaSuccess;
    bool taken = false;
    if (!fused)
        SBNET_TRY(launch_ffn_few<T>(f, const_cast<void*>(h.ptr), stream, &taken));
    if (taken)
        return cudaSuccess;
    note_site("gated_ffn repack");
    Repacks copies;
    copies.add(f.x, x), copies.add(f.w_gate, wg), copies.add(f.w_up, wu), copies.add(f.w_down, wd);
    SBNET_TRY(copies.run(stream));
    if (fused)
        return launch_ffn_fused<T>(f, x, wg, wu, wd, stream);
    note_site("gated_ffn projections");
    Plan p = {};
    p.mTiles = ceil_div(R, kTileM), p.nTiles = ceil_div(F, 128), p.batch = 1, p.segs = 1, p.kIters = ceil_div(C, kStepK);
    p.splits = split_count(R, 2ll * F, (long long)p.mTiles * p.nTiles, p.kIters);
    p.N = F, p.M = R, p.num_blocks_dev = f.num_blocks_dev, p.rowsPerBlock = f.rowsPerBlock, p.act = f.act;
    p.out[0] = const_cast<void*>(h.ptr), p.ldo = Fp, p.partials = parts;
    p.gate = f.kept, p.up = f.kept == nullptr ? nullptr : f.kept + (size_t)R * Fp;
    SBNET_TRY((launch_gemm<T, false, false, kGate, 256>({x, x}, {wg, wu}, p, stream)));
    note_site("gated_ffn output");
    return product<T, false, false>({h, h}, {wd, wd}, 1, 1, R, C, F, f.y, nullptr, parts, f, true, stream);
}

template <typename T> cudaError_t backward(const FfnArgs& f, Layout& l, bool run, cudaStream_t stream)
{
    const long long R = f.rows;
    const int C = f.C, F = f.F, Fp = padded(F);
    const Matrix x = l.plan(f.x, R, C), dy = l.plan(f.dy, R, C), wg = l.plan(f.w_gate, F, C), wu = l.plan(f.w_up, F, C),
                 wd = l.plan(f.w_down, C, F);
    const size_t mid = (size_t)R * Fp * 2;
    const Matrix dg = {l.bump.take(mid), R, F, Fp}, du = {l.bump.take(mid), R, F, Fp}, h = {l.bump.take(mid), R, F, Fp};
    float* parts = static_cast<float*>(l.bump.take(std::max(
        product_partials(1, 2, R, C, F), std::max(product_partials(2, 1, F, C, R), product_partials(1, 1, C, F, R)))));
    if (!run)
        return cudaSuccess;
    note_site("gated_ffn_grad repack");
    Repacks copies;
    copies.add(f.x, x), copies.add(f.dy, dy), copies.add(f.w_gate, wg), copies.add(f.w_up, wu), copies.add(f.w_down, wd);
    SBNET_TRY(copies.run(stream));
    note_site("gated_ffn_grad hidden gradients");
    Plan p = {};
    p.mTiles = ceil_div(R, kTileM), p.nTiles = ceil_div(F, 128), p.batch = 1, p.segs = 2, p.kIters = ceil_div(C, kStepK);
    p.splits = 1, p.N = F, p.M = R, p.act = f.act;
    p.hid = const_cast<void*>(h.ptr), p.dgate = const_cast<void*>(dg.ptr), p.dup = const_cast<void*>(du.ptr), p.ldo = Fp;
    if (f.kept == nullptr) {
        SBNET_TRY(launch_grad<T>(dy, x, wd, wg, wu, p, stream));
    } else {
        p.nTiles = ceil_div(F, 256), p.segs = 1;
        p.gate = f.kept, p.up = f.kept + (size_t)R * Fp;
        SBNET_TRY((launch_gemm<T, false, true, kKept, 256>({dy, dy}, {wd, wd}, p, stream)));
    }
    if (f.dx != nullptr) {
        note_site("gated_ffn_grad dx");
        SBNET_TRY((product<T, false, true>({dg, du}, {wg, wu}, 1, 2, R, C, F, f.dx, nullptr, parts, f, false, stream)));
    }
    if (f.dw_gate != nullptr) {
        note_site("gated_ffn_grad dw_gate, dw_up");
        SBNET_TRY((product<T, true, true>({dg, du}, {x, x}, 2, 1, F, C, R, f.dw_gate, f.dw_up, parts, f, false, stream)));
    }
    if (f.dw_down != nullptr) {
        note_site("gated_ffn_grad dw_down");
        SBNET_TRY((product<T, true, true>({dy, dy}, {h, h}, 1, 1, C, F, R, f.dw_down, nullptr, parts, f, false, stream)));
    }
    return cudaSuccess;
}

} // namespace

size_t gated_ffn_workspace(long long rows, int C, int F, bool grad, bool keep, bool aligned)
{
    static float kept;      // only its being there matters
    FfnArgs f = {};
    f.rows = rows, f.C = C, f.F = F, f.kept = keep ? &kept : nullptr;
    Layout l = {{nullptr, 0}, aligned};
    if (grad)
        backward<__half>(f, l, false, nullptr);
    else
        forward<__half>(f, l, false, nullptr);
    return l.bump.used;
}

// Tensor maps are encoded by a driver call, which wants the device's context current on the calling thread; a thread
// that has made no runtime call yet (a fresh autograd thread) has none.  cudaSetDevice binds it.
static cudaError_t bind_context()
{
    int device = 0;
    if (cudaError_t e = cudaGetDevice(&device))
        return e;
    return cudaSetDevice(device);
}

cudaError_t launch_gated_ffn(const FfnArgs& f, int dtype, cudaStream_t stream)
{
    note_site("gated_ffn context");
    SBNET_TRY(bind_context());
    Layout l = {{static_cast<uint8_t*>(f.workspace), 0}, true};
    return dtype == 1 ? forward<__half>(f, l, true, stream) : forward<__nv_bfloat16>(f, l, true, stream);
}

cudaError_t launch_gated_ffn_grad(const FfnArgs& f, int dtype, cudaStream_t stream)
{
    note_site("gated_ffn_grad context");
    SBNET_TRY(bind_context());
    Layout l = {{static_cast<uint8_t*>(f.workspace), 0}, true};
    return dtype == 1 ? backward<__half>(f, l, true, stream) : backward<__nv_bfloat16>(f, l, true, stream);
}

cudaError_t read_ffn_wait_timeouts(unsigned int* out)
{
    unsigned int fused = 0;
    cudaError_t e = cudaMemcpyFromSymbol(out, g_ffn_timeouts, sizeof(*out));
    if (e == cudaSuccess)
        e = read_ffn_fused_wait_timeouts(&fused);
    *out += fused;
    return e;
}

} // namespace sbnet
