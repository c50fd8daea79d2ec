// Losses of a linear head over a large vocabulary, z = scale * H W^T, without
// z in memory: softmax cross entropy against labels and the divergence from a
// teacher's top logits, with the gradients of H and W. H [T][D] and W [V][D]
// are bf16, products accumulate in f32 in tensor memory (tcgen05).
//
//   plan      rows with a target are packed: their hidden states are copied
//             to an aligned, zero-padded matrix and their count stays on the
//             device, where every later kernel reads it. Rows without a
//             target therefore cost no products, and an infinity or NaN in
//             one cannot reach the others through 0 * NaN. Targets become
//             lists of (vocabulary entry, share) sorted by entry; a label is
//             a list of one.
//   forward   one GEMM over all of V. The epilogue keeps, per row and
//             64-column strip, the maximum and the sum of exp(z - maximum),
//             and stores z where a list names the column; the strips are
//             then folded into log-sum-exp and loss. (A few rows go to
//             linear_score.cuh instead, without packing or tensor cores.)
//   backward  for each piece of the vocabulary: the logits again (summed as
//             the forward pass sums them, by the same kernels), whose
//             epilogue turns them into the slopes
//             G = scale * grad_loss * (exp(z - lse) - share) in bf16 (of up
//             to 64 rows in two bf16 summands); then
//             dH += G W_piece and dW_piece = G^T H, at the same time on a
//             part of the SMs each where that is faster.
//
// Every reduction has a fixed order, so equal inputs give equal bits.
//
// The GEMM has the roles of the one in gemm.cu: per CTA one TMA producer
// lane, one MMA lane, 8 or 16 epilogue warps, and two accumulators of 256
// columns, so that the exponentials of tile i overlap the MMAs of tile i + 1.
// Past 128 rows CTA pairs (cta_group::2) work on tiles of 256 x up to 256, up
// to there single CTAs on 128 x up to 256. Two more warps look up the targets
// of the next tiles' rows. Every wait is bounded: on expiry the CTA raises bit 4 of
// the status word, waits for its MMAs and for the copies in flight (a pair's
// leader for those of both), frees TMEM and returns.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <string>

#include "common.hpp"
#include "exponential.cuh"
#include "linear_loss.hpp"
#include "linear_score.cuh"
#include "loss_parts.cuh"
#include "loss_status.hpp"
#include "tensor_core.cuh"

namespace thb::linear_loss {
namespace {

using namespace thb::tc;

constexpr uint32_t kBM = 128, kBN = 256, kBK = 64;
constexpr uint32_t kListWarps = 2;  // that look up the targets of a tile's rows ahead of its read-out
constexpr uint32_t kTmemCols = 512;
// Products of a logit that the tensor cores sum before the read-out adds: 1024.
// They cut each addition, towards zero. Over 4096 products lse was 1.3e-6 of
// itself off, over 1024 4e-7. The slopes add up their logits the same way, bit
// for bit those that lse was made of: exp(z - lse) of a well-known label is 1
// less a small rest, which a z with roundings of its own would drown (4096
// products, logits around 40: off by 2e-4 where 1e-4 was right).
constexpr uint32_t kBlocksPerSum = 16;
constexpr uint32_t kABytes = kBM * kBK * 2;

enum : int {
    kEpiLse = 0,    // running (max, sum) of each row's strip, z at the listed columns
    kEpiSlope = 1,  // bf16 slopes of the loss
    kEpiTwin = 2,   // the same of few rows, and behind them what their rounding left
    kEpiSlopeSums = 3,  // both of logits that take more than one accumulator's sum
    kEpiTwinSums = 4,
    kEpiAcc = 5,    // f32, stored or added to C
    kEpiOut = 6,    // bf16, rows optionally scattered by a map
};

constexpr bool givesTwins(int epilogue) { return epilogue == kEpiTwin || epilogue == kEpiTwinSums; }
constexpr bool givesSlopes(int epilogue) { return epilogue == kEpiSlope || epilogue == kEpiSlopeSums || givesTwins(epilogue); }
constexpr bool usesLists(int epilogue) { return epilogue == kEpiLse || givesSlopes(epilogue); }
constexpr bool sumsLogits(int epilogue) {
    return epilogue == kEpiLse || epilogue == kEpiSlopeSums || epilogue == kEpiTwinSums;
}

// Epilogue warps: two per TMEM lane quadrant, which split the tile's columns;
// four for logits that are summed, whose part of a row then fits in 64
// registers. (lse: a 1024 x 37888 pass 33.5 -> 29.3 us at a width of 256, 68 ->
// 66.5 at 1024. Slopes of one accumulator are read out faster by two: gradients
// of 64 rows, 32768 x 1024, 65 us against 68. Those of several, with 128 sums a
// thread of which most lie in local memory, are not: 2048 rows, 65536 x 2048,
// 1235 us by two, 1146 by four.)
constexpr uint32_t epilogueWarps(int epilogue) { return sumsLogits(epilogue) ? 16 : 8; }
constexpr uint32_t partsFor(int epilogue) { return epilogueWarps(epilogue) / 4; }
constexpr uint32_t partColumns(int epilogue) { return kBN / partsFor(epilogue); }
constexpr uint32_t threadsFor(int epilogue) {
    return 64 + 32 * (epilogueWarps(epilogue) + (usesLists(epilogue) ? kListWarps : 0));
}
constexpr uint32_t kLogitParts = partsFor(kEpiLse);  // at most
// Strips of a row in a tile of lse.
__host__ __device__ constexpr uint32_t stripsOf(uint32_t tileN) {
    return (tileN + kBN / kLogitParts - 1) / (kBN / kLogitParts);
}

// Rows of the read-out's staging blocks: 64 bytes and a shift of the banks, or
// (four warps a quadrant, whose blocks must leave the ring its stages) 32 bytes.
constexpr uint32_t kStageLd = 80, kSlopeStageLd = 32;
constexpr uint32_t stageLdFor(int epilogue) {
    if (epilogue == kEpiLse || epilogue == kEpiAcc) return 0;
    return sumsLogits(epilogue) ? kSlopeStageLd : kStageLd;
}

// What the read-out of a logits tile needs of its rows: the list's place and,
// for each part of the columns, its first entry there.
struct TileRows {
    uint32_t at[kLogitParts][kBM], next[kLogitParts][kBM], row[kBM];
    float minusLse[kBM], scale[kBM];  // scale: scale * grad_loss
};

template <bool PAIR, int EPI>
struct Geometry {
    static constexpr int stages = PAIR ? 6 : 4;
    static constexpr uint32_t bRows = PAIR ? kBN / 2 : kBN;
    static constexpr uint32_t bBytes = bRows * kBK * 2;
    static constexpr uint32_t stageBytes = kABytes + bBytes;
    static constexpr uint32_t tileM = PAIR ? 2 * kBM : kBM;
    static constexpr uint32_t blockBytes = epilogueWarps(EPI) * 32 * stageLdFor(EPI);
    static constexpr uint32_t smemBytes =
        stages * stageBytes + blockBytes + (usesLists(EPI) ? 2 * sizeof(TileRows) : 0) + 1024;
    static_assert(smemBytes + 512 <= 232448, "shared memory");
};

// f32 accumulator, bf16 operands, N = tileN, M = 128 (one CTA) or 256 (a pair).
template <bool A_MN, bool B_MN, bool PAIR>
__device__ __forceinline__ uint32_t instrDesc(uint32_t tileN) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(A_MN) << 15) |
           (static_cast<uint32_t>(B_MN) << 16) | ((tileN >> 3) << 17) | (((PAIR ? 2 * kBM : kBM) >> 4) << 24);
}

struct Params {
    // C[m][n] = sum over k. The count of packed rows replaces m (countIsM) or k
    // (countIsK, unless k says how many there are where there are any).
    const uint32_t* count;
    uint32_t countIsM, countIsK;
    uint32_t m, n, k;
    uint32_t nTiles, splits, blocksPerSplit;  // k blocks of a split (splits > 1 only with a fixed k)
    uint32_t blocksPerSum;                    // sumsLogits: k blocks that one accumulator sums
    uint32_t aRows;                           // rows of a loaded block of A (K-major A; fewer than 128: the rest is not used)
    uint32_t tileN;                           // columns of a tile (K-major B): 32 to 256, a multiple of 32
    uint32_t group;                           // m blocks per raster group
    uint32_t bFirstN, bFirstK;                // offsets of B's coordinates (the vocabulary piece)
    // kEpiLse, kEpiSlope
    float scale;
    uint32_t entries;
    const uint32_t* rowMap;  // packed row -> row (also kEpiOut, where null keeps the order)
    const uint32_t* ids;     // [row][entries], ascending, kNoEntry behind the last
    const float* shares;     // [row][entries], null: 1
    float* listed;           // z of each list entry, [row][entries]
    float2* strips;          // [strip][stripLd] (maximum, sum)
    uint64_t stripLd;
    // kEpiLse with few rows: each CTA folds its tiles into one strip, and the
    // last to finish joins the strips.
    uint32_t* finished;  // null: joinStrips does
    const float* entropy;
    float* loss;
    float* lse;
    const float* rowLse;     // packed
    const float* rowScale;   // packed: scale * grad_loss
    uint32_t twin;           // kEpiTwin: rows from a slope to what its rounding left
    // outputs
    void* c;
    uint64_t ldc;
    uint64_t splitStride;  // kEpiAcc: elements between the splits' C
    uint32_t accumulate;
    uint32_t* status;
    uint32_t spins;  // tries of a wait
};

// An arrival that orders no memory: what it hands over are TMEM columns whose
// reads are complete. A release at cluster scope would wait for the thread's
// global stores of the tile.
__device__ __forceinline__ void mbarArriveClusterRelaxed(uint32_t clusterAddress) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(clusterAddress) : "memory");
}

// Whether the loads that were issued have landed, when a wait has run out,
// whoever's (all roles have ended). The full barriers count those of `here` and of `peer` k blocks (a CTA alone: the
// same), of which `bytes` each; this CTA has armed its own blocks' barriers for
// both CTAs. A block that one of the two did not come to is armed for the other's
// bytes, or counted down by its own missing ones. Blocks further back than the
// ring were consumed.
template <uint32_t STAGES>
__device__ bool landed(uint64_t* full, uint32_t here, uint32_t peer, uint32_t bytes) {
    const uint32_t end = max(here, peer);
    bool all = true;
    for (uint32_t i = end > STAGES ? end - STAGES : 0u; i < end; ++i) {
        uint64_t* bar = &full[i % STAGES];
        if (i >= here) mbarExpect(bar, bytes);
        else if (i >= peer) mbarComplete(bar, bytes);
        all &= mbarWait(bar, i / STAGES % 2u);
    }
    return all;
}

// Groups of p.group m blocks, walked down m within each n block.
__device__ __forceinline__ void tileCoords(uint32_t tile, uint32_t mTiles, const Params& p, uint32_t& mb, uint32_t& nb) {
    const uint32_t perGroup = p.group * p.nTiles;
    const uint32_t first = tile / perGroup * p.group;
    const uint32_t size = min(mTiles - first, p.group);
    const uint32_t local = tile % perGroup;
    mb = first + local % size;
    nb = local / size;
}

// How many of eight entries of an ascending list, from `first` on `stride`
// apart, lie before `column`; the eight loads are one step of a search.
__device__ __forceinline__ uint32_t probesBefore(const uint32_t* ids, uint32_t first, uint32_t stride, uint32_t entries,
                                                 uint32_t column) {
    uint32_t id[8], count = 0;
#pragma unroll
    for (uint32_t k = 0; k < 8; ++k) id[k] = first + k * stride < entries ? ids[first + k * stride] : kNoEntry;
#pragma unroll
    for (uint32_t k = 0; k < 8; ++k) count += id[k] < column;
    return count;
}

// v[j] by five rounds of selects, so that v stays in registers.
__device__ __forceinline__ float pick(const uint32_t (&v)[32], uint32_t j) {
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = j & 16u ? v[i + 16] : v[i];
#pragma unroll
    for (int width = 8; width >= 1; width >>= 1) {
#pragma unroll
        for (int i = 0; i < width; ++i) w[i] = j & static_cast<uint32_t>(width) ? w[i + width] : w[i];
    }
    return __uint_as_float(w[0]);
}

// A warp's 32 x 32 block of results, lane by row, to bf16 rows in memory:
// through shared memory, so that a store instruction writes whole sectors (8
// rows of 64 bytes; rows that do not start at 16-byte boundaries 32 elements
// of one row) instead of 16 bytes of 32 rows. `row` is the lane's destination
// row; `left` columns lie inside the matrix. (A 64-row step over a 32768 x
// 2048 head: its weight gradient, 134 MB, took 67 us without.)
// SCATTER: row r of the block goes to rows' own destinations (`row` of lane
// r), else to row0 + r. `rows` of the block are written.
template <bool SCATTER>
__device__ __forceinline__ void storeBf16Block(uint8_t* stage, __nv_bfloat16* c, uint64_t ldc, uint64_t row, uint32_t rows,
                                               uint32_t col, const float (&v)[32], uint32_t left, uint32_t lane) {
    __syncwarp();  // the block before has been read
    uint4* mine = reinterpret_cast<uint4*>(stage + lane * kStageLd);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        uint4 packed;
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&packed);
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = __floats2bfloat162_rn(v[q * 8 + 2 * e], v[q * 8 + 2 * e + 1]);
        mine[q] = packed;
    }
    __syncwarp();
    const uint64_t row0 = SCATTER ? 0u : row - lane;
    const bool vectors = left >= 32 && ldc % 8 == 0 && reinterpret_cast<uintptr_t>(c) % 16 == 0;
    if (vectors) {
        __nv_bfloat16* to = c + (row0 + lane / 4) * ldc + col + lane % 4 * 8;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t r = i * 8 + lane / 4;
            const uint4 packed = *reinterpret_cast<const uint4*>(stage + r * kStageLd + lane % 4 * 16);
            if constexpr (SCATTER) to = c + __shfl_sync(0xffffffffu, row, r) * ldc + col + lane % 4 * 8;
            if (r < rows) *reinterpret_cast<uint4*>(to) = packed;
            to += 8 * ldc;
        }
    } else {
        __nv_bfloat16* to = c + row0 * ldc + col + lane;
#pragma unroll 8
        for (uint32_t r = 0; r < 32; ++r) {
            const __nv_bfloat16 x = reinterpret_cast<const __nv_bfloat16*>(stage + r * kStageLd)[lane];
            if constexpr (SCATTER) to = c + __shfl_sync(0xffffffffu, row, r) * ldc + col + lane;
            if (r < rows && lane < left) *to = x;
            to += ldc;
        }
    }
}

// The same of 16 columns of slopes, whose rows lie at 32-byte boundaries: a
// store instruction writes 16 sectors. The halves of a staged row change places
// every four rows, so that eight rows' halves meet every bank once.
__device__ __forceinline__ void storeSlopes(uint8_t* stage, __nv_bfloat16* c, uint64_t ldc, uint32_t row, uint32_t rows,
                                            uint32_t col, const float (&v)[16], uint32_t lane) {
    uint4* block = reinterpret_cast<uint4*>(stage);
    __syncwarp();  // the block before has been read
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
        uint4 packed;
        __nv_bfloat162* pairs = reinterpret_cast<__nv_bfloat162*>(&packed);
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) pairs[e] = __floats2bfloat162_rn(v[h * 8 + 2 * e], v[h * 8 + 2 * e + 1]);
        block[lane * 2 + (h ^ (lane / 4 % 2))] = packed;
    }
    __syncwarp();
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        const uint32_t r = i * 16 + lane / 2, h = lane % 2;
        const uint4 packed = block[r * 2 + (h ^ (r / 4 % 2))];
        if (r < rows) *reinterpret_cast<uint4*>(c + static_cast<uint64_t>(row - lane + r) * ldc + col + h * 8) = packed;
    }
}

// The same of 32 columns, through rows of kStageLd.
__device__ __forceinline__ void storeSlopes(uint8_t* stage, __nv_bfloat16* c, uint64_t ldc, uint32_t row, uint32_t rows,
                                            uint32_t col, const float (&v)[32], uint32_t lane) {
    storeBf16Block<false>(stage, c, ldc, row, rows, col, v, 32u, lane);
}

// The tiles first, first + step, ... of one matrix of products, by a CTA or a
// pair.
template <bool A_MN, bool B_MN, int EPI, bool PAIR>
__device__ __forceinline__ void products(const CUtensorMap& mapA, const CUtensorMap& mapB, const Params& p,
                                         const uint32_t first, const uint32_t step) {
    using G = Geometry<PAIR, EPI>;
    constexpr uint32_t kWarps = epilogueWarps(EPI), kParts = partsFor(EPI), kStrip = partColumns(EPI);
    (void)kParts;
    extern __shared__ uint8_t dynamicSmem[];
    __shared__ __align__(8) uint64_t full[G::stages], empty[G::stages], tmemFull[2], tmemEmpty[2], mmaDone;
    __shared__ __align__(8) uint64_t rowsFull[2], rowsEmpty[2];
    __shared__ uint32_t tmemSlot;
    __shared__ uint32_t issuedHere, issuedByPeer;  // k blocks whose loads were issued; by the other CTA of a pair (leader)
    __shared__ volatile int abortFlag;
    __shared__ float2 parts[kLogitParts][32];  // of the rows' strips, and
    __shared__ bool lastOne;                 // whether this CTA joins them (finished)
    (void)parts;
    (void)lastOne;

    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dynamicSmem) + 1023) & ~uintptr_t(1023));
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t rank = PAIR ? clusterRank() : 0u;

    if (threadIdx.x == 0) {
        abortFlag = 0;
        for (int s = 0; s < G::stages; ++s) {
            mbarInit(&full[s], 1);
            mbarInit(&empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbarInit(&tmemFull[a], 1);
            mbarInit(&tmemEmpty[a], (PAIR ? 2 : 1) * 32 * kWarps);
            mbarInit(&rowsFull[a], 32 * kListWarps);
            mbarInit(&rowsEmpty[a], 32 * kWarps);
        }
        mbarInit(&mmaDone, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem(&tmemSlot)),
                         "r"(kTmemCols)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem(&tmemSlot)),
                         "r"(kTmemCols)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    fenceBefore();
    __syncthreads();
    if constexpr (PAIR) clusterSync();
    fenceAfter();
    const uint32_t tmemBase = tmemSlot;

    // The next kernel's CTAs may take the place of this one's as they leave;
    // they wait for all of this kernel, as this one does here for the one
    // before it. Everything above overlaps that kernel's end.
    gridDependencyLaunch();
    gridDependencyWait();
    const uint32_t count = p.count ? *p.count : 0u;
    const uint32_t m = p.countIsM ? count : p.m;
    const uint32_t k = !p.countIsK || (p.k && count) ? p.k : count;
    const uint32_t mTiles = (m + G::tileM - 1) / G::tileM;
    const uint32_t kBlocks = (k + kBK - 1) / kBK;
    const uint32_t perSplit = p.splits > 1 ? p.blocksPerSplit : kBlocks;
    const uint32_t plane = mTiles * p.nTiles;
    const uint32_t tiles = plane * p.splits;
    const uint32_t tileN = B_MN ? kBN : p.tileN;
    TileRows* tileRows = reinterpret_cast<TileRows*>(base + G::stages * G::stageBytes + G::blockBytes);
    (void)tileRows;
    const uint32_t loadBytes = (A_MN ? kBM : p.aRows) * kBK * 2 + tileN / (PAIR ? 2 : 1) * kBK * 2;  // of a CTA and stage

    if (warp == 0 && lane == 0) {
        // ---- TMA producer ----
        uint32_t stage = 0, phase = 0, issued = 0;
        for (uint32_t tile = first; tile < tiles && !abortFlag; tile += step) {
            uint32_t mb, nb;
            tileCoords(tile % plane, mTiles, p, mb, nb);
            const uint32_t kb0 = tile / plane * perSplit, kb1 = min(kb0 + perSplit, kBlocks);
            const int32_t row0 = static_cast<int32_t>(mb * G::tileM + rank * kBM);
            const int32_t col0 = static_cast<int32_t>(p.bFirstN + nb * tileN + rank * (tileN / 2));
            for (uint32_t kb = kb0; kb < kb1; ++kb) {
                if (!mbarWait(&empty[stage], phase ^ 1u, &abortFlag, p.spins)) { abortFlag = 1; break; }
                uint8_t* a = base + stage * G::stageBytes;
                uint8_t* b = a + kABytes;
                const int32_t ka = static_cast<int32_t>(kb * kBK);
                const int32_t kB = static_cast<int32_t>(p.bFirstK + kb * kBK);
                if constexpr (PAIR) {
                    if (rank == 0) mbarExpect(&full[stage], 2 * loadBytes);
                    const uint32_t bar = pairAddress(&full[stage], 0);
                    if constexpr (A_MN) {
                        tmaLoad2dPair(a, &mapA, row0, ka, bar);
                        tmaLoad2dPair(a + kABytes / 2, &mapA, row0 + 64, ka, bar);
                    } else {
                        tmaLoad2dPair(a, &mapA, ka, row0, bar);
                    }
                    if constexpr (B_MN) {
#pragma unroll
                        for (uint32_t j = 0; j < G::bRows / 64; ++j)
                            tmaLoad2dPair(b + j * (64 * kBK * 2), &mapB, col0 + 64 * j, kB, bar);
                    } else {
                        tmaLoad2dPair(b, &mapB, kB, col0, bar);
                    }
                } else {
                    mbarExpect(&full[stage], loadBytes);
                    if constexpr (A_MN) {
                        tmaLoad2d(a, &mapA, row0, ka, &full[stage]);
                        tmaLoad2d(a + kABytes / 2, &mapA, row0 + 64, ka, &full[stage]);
                    } else {
                        tmaLoad2d(a, &mapA, ka, row0, &full[stage]);
                    }
                    if constexpr (B_MN) {
#pragma unroll
                        for (uint32_t j = 0; j < G::bRows / 64; ++j)
                            tmaLoad2d(b + j * (64 * kBK * 2), &mapB, col0 + 64 * j, kB, &full[stage]);
                    } else {
                        tmaLoad2d(b, &mapB, kB, col0, &full[stage]);
                    }
                }
                ++issued;
                if (++stage == G::stages) { stage = 0; phase ^= 1u; }
            }
        }
        if (rank == 0) issuedHere = issued;
        else storeCluster(pairAddress(&issuedByPeer, 0), issued);
    } else if (warp == 1 && lane == 0) {
        // ---- MMA issuer (of a pair: the leader, for both CTAs) ----
        if (!PAIR || rank == 0) {
            const uint32_t idesc = instrDesc<A_MN, B_MN, PAIR>(tileN);
            constexpr uint32_t atom = 64 * kBK * 2;  // MN-major operands: 64-element atoms
            auto commit = [](uint64_t* bar) {
                if constexpr (PAIR) mmaCommitPair(bar);
                else mmaCommit(bar);
            };
            uint32_t stage = 0, phase = 0, acc = 0, accPhase = 0;
            // The tensor cores hold a few instructions only, so that every
            // cycle of this thread between two k blocks counts: descriptors
            // are those of stage 0 plus an offset (in units of 16 bytes),
            // and whether the next block has arrived is looked up between
            // the instructions of this one. (8192 rows, 131072 x 4096:
            // 21.6 -> 21.0 ms a step under the power cap, 18.95 -> 18.35
            // from idle.)
            const uint64_t da0 = A_MN ? ummaDesc(smem(base), atom, 1024u) : ummaDesc(smem(base), 16u, 1024u);
            const uint64_t db0 =
                B_MN ? ummaDesc(smem(base) + kABytes, atom, 1024u) : ummaDesc(smem(base) + kABytes, 16u, 1024u);
            uint32_t offset = 0;
            bool ready = false;
            for (uint32_t tile = first; tile < tiles && !abortFlag; tile += step) {
                const uint32_t kb0 = tile / plane * perSplit, kb1 = min(kb0 + perSplit, kBlocks);
                bool ok = true;
                uint32_t kb = kb0;
                do {  // one accumulator: the whole k range, or blocksPerSum of it
                    const uint32_t end = sumsLogits(EPI) ? min(kb + p.blocksPerSum, kb1) : kb1;
                    if (!mbarWait(&tmemEmpty[acc], accPhase ^ 1u, &abortFlag, p.spins)) { abortFlag = 1; ok = false; break; }
                    fenceAfter();
                    const uint32_t d = tmemBase + acc * kBN;
                    for (const uint32_t begin = kb; kb < end; ++kb) {
                        if (!ready && !mbarWait(&full[stage], phase, &abortFlag, p.spins)) { abortFlag = 1; ok = false; break; }
                        fenceAfter();
                        const uint32_t next = stage + 1 == G::stages ? 0u : stage + 1;
                        const uint32_t nextPhase = next ? phase : phase ^ 1u;
                        const uint64_t da = da0 + offset, db = db0 + offset;
#pragma unroll
                        for (uint32_t ks = 0; ks < kBK / 16; ++ks) {
                            const uint32_t more = kb != begin || ks != 0 ? 1u : 0u;
                            const uint64_t a = da + ks * (A_MN ? 128u : 2u), b = db + ks * (B_MN ? 128u : 2u);
                            if constexpr (PAIR) mmaPair(d, a, b, idesc, more);
                            else mma(d, a, b, idesc, more);
                            if (ks == 1) ready = mbarTest(&full[next], nextPhase);
                        }
                        commit(&empty[stage]);
                        offset = next ? offset + G::stageBytes / 16 : 0u;
                        stage = next;
                        phase = nextPhase;
                    }
                    if (!ok) break;
                    commit(&tmemFull[acc]);
                    if (++acc == 2) { acc = 0; accPhase ^= 1u; }
                } while (kb < kb1);
                if (!ok) break;
            }
            commit(&mmaDone);
            if (!mbarWait(&mmaDone, 0)) abortFlag = 1;
        }
    } else if (warp >= 2 + kWarps) {
        // ---- the targets of the tiles' rows, two tiles ahead at most ----
        if constexpr (usesLists(EPI)) {
            uint32_t buf = 0, phase = 0;
            for (uint32_t tile = first; tile < tiles; tile += step) {
                uint32_t mb, nb;
                tileCoords(tile % plane, mTiles, p, mb, nb);
                if (!mbarWait(&rowsEmpty[buf], phase ^ 1u, &abortFlag, p.spins)) abortFlag = 1;
                if (__any_sync(0xffffffffu, abortFlag)) break;
                TileRows& out = tileRows[buf];
                constexpr uint32_t kRows = kBM / (32 * kListWarps);  // of a thread
                const uint32_t me = (warp - 2 - kWarps) * 32 + lane;
                const uint32_t row0 = mb * G::tileM + rank * kBM;
                uint32_t to[kRows];
                uint64_t list[kRows];
                bool live[kRows];
#pragma unroll
                for (uint32_t i = 0; i < kRows; ++i) {
                    const uint32_t r = i * 32 * kListWarps + me, row = row0 + r;
                    live[i] = row < m;
                    to[i] = live[i] ? p.rowMap[row] : 0u;
                    list[i] = static_cast<uint64_t>(to[i]) * p.entries;
                    out.row[r] = to[i];
                    if constexpr (givesSlopes(EPI)) {
                        out.minusLse[r] = live[i] ? -p.rowLse[row] : 0.0f;
                        out.scale[r] = live[i] ? p.rowScale[row] : 0.0f;
                    }
                }
                // The first entry at or behind the tile's first column: eight
                // loads a step, the rows side by side, since these warps must
                // keep up with tiles of few k blocks. (4000 rows, 20000 x 328,
                // lists of 50: 399 us a step with binary searches for every
                // part, 376 so.)
                const uint32_t column = p.bFirstN + nb * tileN;
                uint32_t lo[kRows] = {};
                for (uint32_t bound = p.entries > 8 ? p.entries : 0u; bound;) {
                    const uint32_t stride = (bound + 7) / 8;
#pragma unroll
                    for (uint32_t i = 0; i < kRows; ++i)
                        lo[i] += stride * probesBefore(p.ids + list[i], lo[i] + stride - 1, stride, p.entries, column);
                    bound = stride - 1;
                }
                // The parts' first entries are among the next eight as a rule
                // (of lists up to eight, always).
#pragma unroll
                for (uint32_t i = 0; i < kRows; ++i) {
                    const uint32_t r = i * 32 * kListWarps + me;
                    uint32_t window[8];
#pragma unroll
                    for (uint32_t k = 0; k < 8; ++k)
                        window[k] = live[i] && lo[i] + k < p.entries ? p.ids[list[i] + lo[i] + k] : kNoEntry;
#pragma unroll 1
                    for (uint32_t h = 0; h < kParts; ++h) {
                        uint32_t at = lo[i], next = kNoEntry;
#pragma unroll
                        for (uint32_t k = 0; k < 8; ++k) {
                            const bool before = window[k] < column + h * kStrip;
                            at += before;
                            next = min(next, before ? kNoEntry : window[k]);
                        }
                        while (at - lo[i] >= 8 && at < p.entries && (next = p.ids[list[i] + at]) < column + h * kStrip) ++at;
                        if (at >= p.entries) next = kNoEntry;
                        out.at[h][r] = at;
                        out.next[h][r] = next;
                    }
                }
                mbarArrive(&rowsFull[buf]);
                if (++buf == 2) { buf = 0; phase ^= 1u; }
            }
        }
    } else if (warp >= 2) {
        // ---- epilogue ----
        const uint32_t quadrant = warp % 4;  // TMEM lanes 32 * quadrant .. + 31
        const uint32_t part = (warp - 2) / 4;
        uint32_t acc = 0, accPhase = 0;
        uint8_t* stage = base + G::stages * G::stageBytes + (warp - 2) * 32 * stageLdFor(EPI);
        (void)stage;
        uint32_t rowsBuf = 0, rowsPhase = 0;
        float runningTop = -INFINITY, runningSum = 0.0f;
        (void)runningTop;
        (void)runningSum;
        const uint32_t releaseAddress = PAIR ? pairAddress(&tmemEmpty[0], 0) : 0u;
        for (uint32_t tile = first; tile < tiles; tile += step) {
            uint32_t mb, nb;
            tileCoords(tile % plane, mTiles, p, mb, nb);
            const uint32_t split = tile / plane;
            const uint32_t row = mb * G::tileM + rank * kBM + quadrant * 32 + lane;
            const uint32_t col0 = nb * tileN + part * kStrip;  // within C
            // Columns of this warp.
            const uint32_t width = tileN > part * kStrip ? min(tileN - part * kStrip, kStrip) : 0u;
            const bool live = row < m;
            // Rows of this warp that exist.
            const uint32_t rowsHere = row - lane < m ? min(m - (row - lane), 32u) : 0u;
            const uint32_t* ids = nullptr;
            uint64_t list = 0;
            uint32_t at = 0, next = kNoEntry;
            float rowScale = 0.0f, minusLse = 0.0f;
            uint64_t outRow = row;
            if constexpr (usesLists(EPI)) {
                if (!mbarWait(&rowsFull[rowsBuf], rowsPhase, &abortFlag, p.spins)) abortFlag = 1;
                if (__any_sync(0xffffffffu, abortFlag)) break;  // the warp leaves together
                const TileRows& in = tileRows[rowsBuf];
                const uint32_t r = quadrant * 32 + lane;
                list = static_cast<uint64_t>(in.row[r]) * p.entries;
                ids = p.ids + list;
                at = in.at[part][r];
                next = in.next[part][r];
                if constexpr (givesSlopes(EPI)) {
                    rowScale = in.scale[r];
                    minusLse = in.minusLse[r];
                }
                mbarArrive(&rowsEmpty[rowsBuf]);
                if (++rowsBuf == 2) { rowsBuf = 0; rowsPhase ^= 1u; }
            }
            if constexpr (EPI == kEpiOut) {
                if (live && p.rowMap) outRow = p.rowMap[row];
            }
            // Frees the accumulator once its columns are in registers.
            auto release = [&] {
                fenceBefore();
                if (PAIR && rank != 0) mbarArriveClusterRelaxed(releaseAddress + acc * static_cast<uint32_t>(sizeof(uint64_t)));
                else mbarArrive(&tmemEmpty[acc]);
                if (++acc == 2) { acc = 0; accPhase ^= 1u; }
            };
            // Logits of a row, from `col` of C on, to slopes in memory.
            auto giveSlopes = [&](auto& v, uint32_t col) {
                constexpr uint32_t kWidth = sizeof(v) / sizeof(v[0]);
                const float2 slope2 = make_float2(rowScale, rowScale), scale2 = make_float2(p.scale, p.scale);
#pragma unroll
                for (uint32_t j = 0; j < kWidth; j += 2) {
                    const float2 e = mul2(slope2, pow2Shifted(mul2(make_float2(v[j], v[j + 1]), scale2), minusLse, kLog2e));
                    v[j] = e.x;
                    v[j + 1] = e.y;
                }
                while (next < p.bFirstN + col + kWidth) {
                    const float share = rowScale * (p.shares ? p.shares[list + at] : 1.0f);
                    const uint32_t j0 = next - (p.bFirstN + col);
#pragma unroll
                    for (uint32_t j = 0; j < kWidth; ++j) v[j] = __fsub_rn(v[j], j0 == j ? share : 0.0f);
                    next = ++at < p.entries ? ids[at] : kNoEntry;
                }
                // Rows and columns behind the last are operands of the next
                // products (whole k blocks): zeros.
                const uint32_t left = p.n > col ? p.n - col : 0u;  // columns of v inside C
                if (rowsHere < 32 || left < kWidth) {
#pragma unroll
                    for (uint32_t j = 0; j < kWidth; ++j)
                        if (!live || j >= left) v[j] = 0.0f;
                }
                // The slopes are rounded to bf16, the tensor cores' operand
                // type: as much as the gradients' own rounding, so that a
                // gradient is off by 0.0024 of its norm, of any number of
                // rows, where f32 slopes leave 0.0017. Where the rows fill
                // half a tile at most, what the rounding left follows as rows
                // of its own in the other half, whose products add to the
                // same sums: 0.0017 for little (64 rows, 32768 x 2048: 148 us
                // a step instead of 140), while more rows would need as many
                // tiles again.
                __nv_bfloat16* c = static_cast<__nv_bfloat16*>(p.c);
                if constexpr (!givesTwins(EPI)) {
                    storeSlopes(stage, c, p.ldc, row, 32u, col, v, lane);
                } else {
                    uint32_t to = row, end = p.twin;
#pragma unroll 1
                    for (;;) {
                        if (row - lane < end) storeSlopes(stage, c, p.ldc, to, min(end - (row - lane), 32u), col, v, lane);
                        if (to != row) break;
#pragma unroll
                        for (uint32_t j = 0; j < kWidth; ++j) v[j] -= __bfloat162float(__float2bfloat16_rn(v[j]));
                        to = row + p.twin;
                        end = kBM - p.twin;
                    }
                }
            };
            (void)giveSlopes;
            if constexpr (sumsLogits(EPI)) {
                // The strip of a row, in registers. The tensor cores cut each
                // addition to f32, which over a long k drifts towards zero;
                // sums over blocksPerSum k blocks are added here, rounded.
                uint32_t raw[kStrip / 32][32];
                auto z = [&](uint32_t j) { return __uint_as_float(raw[j / 32][j % 32]); };
                auto arrived = [&] {  // (The warp leaves together.)
                    if (!mbarWait(&tmemFull[acc], accPhase, &abortFlag, p.spins)) abortFlag = 1;
                    if (__any_sync(0xffffffffu, abortFlag)) return false;
                    fenceAfter();
                    return true;
                };
                const uint32_t columns = tmemBase + ((quadrant * 32u) << 16) + part * kStrip;
                if (!arrived()) break;
#pragma unroll
                for (uint32_t q = 0; q < kStrip / 32; ++q) tmemFetch32(columns + acc * kBN + q * 32u, raw[q]);
#pragma unroll
                for (uint32_t q = 0; q < kStrip / 32; ++q) tmemArrived(raw[q]);
                release();
                bool ok = true;
                for (uint32_t kb = p.blocksPerSum; kb < kBlocks; kb += p.blocksPerSum) {
                    if (!(ok = arrived())) break;
#pragma unroll
                    for (uint32_t q = 0; q < kStrip / 16; ++q) {
                        uint32_t r[16];
                        tmemLoad16(columns + acc * kBN + q * 16u, r);
#pragma unroll
                        for (uint32_t j = 0; j < 16; ++j) {
                            uint32_t& sum = raw[q / 2][q % 2 * 16 + j];
                            sum = __float_as_uint(__uint_as_float(sum) + __uint_as_float(r[j]));
                        }
                    }
                    release();
                }
                if (!ok) break;
                if constexpr (givesSlopes(EPI)) {
#pragma unroll
                    for (uint32_t q = 0; q < kStrip / 16; ++q) {
                        const uint32_t col = col0 + q * 16;
                        if (q * 16 >= width || col >= p.ldc) break;
                        float v[16];
#pragma unroll
                        for (uint32_t j = 0; j < 16; ++j) v[j] = z(q * 16 + j);
                        giveSlopes(v, col);
                    }
                    continue;
                }
                if (!live || width == 0) continue;
                const uint32_t left = p.n > col0 ? min(p.n - col0, width) : 0u;  // columns of the strip in the vocabulary
                if (left < kStrip) {
#pragma unroll
                    for (uint32_t j = 0; j < kStrip; ++j)
                        if (j >= left) raw[j / 32][j % 32] = __float_as_uint(-INFINITY);
                }
                float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (uint32_t j = 0; j < kStrip; ++j) tops[j % 4] = fmaxf(tops[j % 4], z(j));
                const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
                // (A strip of nothing but -inf takes any finite maximum.)
                const float c = p.scale * kLog2e, minusTop = top == -INFINITY ? 0.0f : -top;
                float2 sums[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                for (uint32_t j = 0; j < kStrip / 2; ++j)
                    sums[j % 2] = add2(sums[j % 2], pow2Shifted(make_float2(z(2 * j), z(2 * j + 1)), minusTop, c));
                const float2 sum = add2(sums[0], sums[1]);
                if (p.finished)
                    fold(runningTop, runningSum, top, sum.x + sum.y, c);
                else
                    p.strips[static_cast<uint64_t>(nb * stripsOf(tileN) + part) * p.stripLd + row] =
                        make_float2(top, sum.x + sum.y);
#pragma unroll
                for (uint32_t q = 0; q < kStrip / 32; ++q) {
                    while (next < col0 + min((q + 1) * 32, width)) {
                        p.listed[list + at] = pick(raw[q], next - (col0 + q * 32)) * p.scale;
                        next = ++at < p.entries ? ids[at] : kNoEntry;
                    }
                }
                continue;
            }
            if (!mbarWait(&tmemFull[acc], accPhase, &abortFlag, p.spins)) abortFlag = 1;
            if (__any_sync(0xffffffffu, abortFlag)) break;
            fenceAfter();
            // 32 columns at a time, the next ones on their way meanwhile.
            const uint32_t limit = givesSlopes(EPI) ? static_cast<uint32_t>(p.ldc) : p.n;
            const uint32_t chunks = col0 < limit ? min(width, limit - col0 + 31) / 32 : 0u;
            const uint32_t columns = tmemBase + ((quadrant * 32u) << 16) + acc * kBN + part * kStrip;
            uint32_t r[32];
            if (chunks) tmemFetch32(columns, r);
            else release();
#pragma unroll 1
            for (uint32_t chunk = 0; chunk < chunks; ++chunk) {
                const uint32_t col = col0 + chunk * 32;
                __syncwarp();
                tmemArrived(r);
                float v[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
                if (chunk + 1 < chunks) tmemFetch32(columns + (chunk + 1) * 32u, r);
                else release();
                const uint32_t left = p.n > col ? p.n - col : 0u;  // columns of the chunk inside C
                if constexpr (givesSlopes(EPI)) {
                    giveSlopes(v, col);
                } else {
                    if (kBlocks == 0) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = 0.0f;  // no MMA has written the accumulator
                    }
                    if constexpr (EPI == kEpiOut) {
                        __nv_bfloat16* c = static_cast<__nv_bfloat16*>(p.c);
                        if (p.rowMap) storeBf16Block<true>(stage, c, p.ldc, outRow, rowsHere, col, v, left, lane);
                        else storeBf16Block<false>(stage, c, p.ldc, row, rowsHere, col, v, left, lane);
                    } else if (live) {
                        {
                            float* dst = static_cast<float*>(p.c) + split * p.splitStride + outRow * p.ldc + col;
                            if (left >= 32) {  // ldc is a multiple of 4
#pragma unroll
                                for (int q = 0; q < 8; ++q) {
                                    float4 w = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
                                    if (p.accumulate) {
                                        const float4 old = *reinterpret_cast<const float4*>(dst + 4 * q);
                                        w.x += old.x;
                                        w.y += old.y;
                                        w.z += old.z;
                                        w.w += old.w;
                                    }
                                    *reinterpret_cast<float4*>(dst + 4 * q) = w;
                                }
                            } else {
#pragma unroll
                                for (uint32_t j = 0; j < 32; ++j)
                                    if (j < left) dst[j] = p.accumulate ? dst[j] + v[j] : v[j];
                            }
                        }
                    }
                }
            }
        }
        if constexpr (EPI == kEpiLse) {
            if (p.finished && quadrant == 0) parts[part][lane] = make_float2(runningTop, runningSum);
        }
    }
    __syncthreads();
    if (threadIdx.x == 0 && abortFlag) atomicOr(p.status, kWaitStatus);
    if constexpr (EPI == kEpiLse) {
        if (p.finished) {
            // The CTA's tiles in one strip a row, stored strip-fastest. (The
            // z of its list entries are stored too, by the warps above.)
            __threadfence();
            __syncthreads();
            const float c = p.scale * kLog2e;
            if (warp == 0) {
                float top = -INFINITY, sum = 0.0f;
#pragma unroll
                for (uint32_t k = 0; k < kParts; ++k) fold(top, sum, parts[k][lane].x, parts[k][lane].y, c);
                if (lane < m) p.strips[lane * step + first] = make_float2(top, sum);
                __threadfence();
                __syncwarp();
                if (lane == 0) lastOne = atomicAdd(p.finished, 1u) == step - 1;
                __threadfence();
            }
            __syncthreads();
            if (lastOne) {
                // A warp a row: its lanes fold the CTAs' strips in a fixed order.
                for (uint32_t row = warp; row < m; row += threadsFor(EPI) / 32) {
                    const uint64_t to = p.rowMap[row];
                    float top = -INFINITY, sum = 0.0f, target = 0.0f;
                    for (uint32_t s = lane; s < step; s += 32) {
                        const float2 x = __ldcg(p.strips + row * step + s);
                        fold(top, sum, x.x, x.y, c);
                    }
                    for (uint32_t e = lane; e < p.entries; e += 32) {
                        if (p.ids[to * p.entries + e] == kNoEntry) break;  // the list is sorted
                        const float share = p.shares ? p.shares[to * p.entries + e] : 1.0f;
                        // A share of nothing takes nothing, whatever z is.
                        if (share != 0.0f) target += share * __ldcg(p.listed + to * p.entries + e);
                    }
                    __syncwarp();
#pragma unroll
                    for (uint32_t o = 1; o < 32; o *= 2) {
                        const float otherTop = __shfl_xor_sync(0xffffffffu, top, o);
                        const float otherSum = __shfl_xor_sync(0xffffffffu, sum, o);
                        fold(top, sum, otherTop, otherSum, c);
                        target += __shfl_xor_sync(0xffffffffu, target, o);
                    }
                    if (lane == 0) closeRow(to, top, sum, p.scale, target, p.entropy, p.loss, p.lse);
                }
            }
        }
    }
    // A pair stays resident until both CTAs are done: the leader's MMAs read
    // the peer's shared memory, the peer arrives on the leader's barriers, and
    // loads in flight, which both CTAs count there, land before either leaves.
    if constexpr (PAIR) {
        clusterSync();
        if (rank == 0 && threadIdx.x == 0 && (abortFlag || issuedHere != issuedByPeer) &&
            !landed<G::stages>(full, issuedHere, issuedByPeer, loadBytes))
            atomicOr(p.status, kWaitStatus | kDrainStatus);
        clusterSync();
    } else if (threadIdx.x == 0 && abortFlag && !landed<G::stages>(full, issuedHere, issuedHere, loadBytes)) {
        atomicOr(p.status, kDrainStatus);
    }
    if (warp == 1) {
        fenceAfter();
        if constexpr (PAIR)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmemBase), "r"(kTmemCols) : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmemBase), "r"(kTmemCols) : "memory");
    }
}

template <bool A_MN, bool B_MN, int EPI, bool PAIR>
__global__ void __launch_bounds__(threadsFor(EPI), 1)
    lossGemm(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB, const Params p) {
    constexpr uint32_t unit = PAIR ? 2 : 1;
    products<A_MN, B_MN, EPI, PAIR>(mapA, mapB, p, blockIdx.x / unit, gridDim.x / unit);
}

// Both gradients at the same time: the first `hidden` CTAs (pairs) work on dH,
// which reads the weights, the others on dW, which writes as much. planGradients
// says when.
template <bool PAIR>
__global__ void __launch_bounds__(threadsFor(kEpiOut), 1)
    bothGradients(const __grid_constant__ CUtensorMap slopesK, const __grid_constant__ CUtensorMap weightMN,
                  const __grid_constant__ CUtensorMap slopesMN, const __grid_constant__ CUtensorMap hiddenMN,
                  const Params h, const Params w, const uint32_t hidden) {
    static_assert(threadsFor(kEpiOut) == threadsFor(kEpiAcc));
    constexpr uint32_t unit = PAIR ? 2 : 1;
    const uint32_t i = blockIdx.x / unit;
    if (i < hidden)
        products<false, true, kEpiAcc, PAIR>(slopesK, weightMN, h, i, hidden);
    else
        products<true, true, kEpiOut, PAIR>(slopesMN, hiddenMN, w, i - hidden, gridDim.x / unit - hidden);
}

// ---- plan ----------------------------------------------------------------

__device__ __forceinline__ float teacherLogit(const void* s, bool bf16, uint64_t i) {
    return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(s)[i]) : static_cast<const float*>(s)[i];
}

// ---- copies of unaligned rows ----
//
// Rows of bf16 that start off a 16-byte boundary are read in the aligned
// vectors that hold them (each holds at least one of the row's elements) and
// shifted into place between neighbouring lanes.

// Elements 8 i .. 8 i + 7 of a row that starts `off` elements into vector 0,
// from vector i and the one behind it; elements from `dim` on are zeros.
__device__ __forceinline__ uint4 shifted(const uint4& a, const uint4& b, uint32_t off, uint32_t i, uint32_t dim) {
    uint32_t w[4];
    auto shift = [&](uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, uint32_t w4) {
        const uint32_t bits = off % 2 * 16;
        w[0] = __funnelshift_r(w0, w1, bits);
        w[1] = __funnelshift_r(w1, w2, bits);
        w[2] = __funnelshift_r(w2, w3, bits);
        w[3] = __funnelshift_r(w3, w4, bits);
    };
    switch (off / 2) {
    case 0: shift(a.x, a.y, a.z, a.w, b.x); break;
    case 1: shift(a.y, a.z, a.w, b.x, b.y); break;
    case 2: shift(a.z, a.w, b.x, b.y, b.z); break;
    default: shift(a.w, b.x, b.y, b.z, b.w); break;
    }
    if (i * 8 + 8 > dim) {
#pragma unroll
        for (uint32_t q = 0; q < 4; ++q) {
            const uint32_t e = i * 8 + 2 * q;
            if (e >= dim) w[q] = 0;
            else if (e + 1 >= dim) w[q] &= 0xffffu;
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// The next lane's vector; lane 31 gets lane 0's `wrapped`.
__device__ __forceinline__ uint4 nextLane(const uint4& mine, const uint4& wrapped, uint32_t lane) {
    const uint4 give = lane == 0 ? wrapped : mine;
    return make_uint4(__shfl_sync(0xffffffffu, give.x, (lane + 1) % 32), __shfl_sync(0xffffffffu, give.y, (lane + 1) % 32),
                      __shfl_sync(0xffffffffu, give.z, (lane + 1) % 32), __shfl_sync(0xffffffffu, give.w, (lane + 1) % 32));
}

__device__ __forceinline__ uint32_t elementsOff(const __nv_bfloat16* p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) % 16 / 2);
}

// A warp copies one row (zeros when src is null), padded with zeros from
// `dim` to `width`.
__device__ __forceinline__ void copyRow(__nv_bfloat16* dst, const __nv_bfloat16* src, uint32_t dim, uint32_t width,
                                        uint32_t lane) {
    if (reinterpret_cast<uintptr_t>(dst) % 16 || width % 8) {
        for (uint32_t i = lane; i < width; i += 32) dst[i] = src && i < dim ? src[i] : __float2bfloat16_rn(0.0f);
        return;
    }
    uint4* to = reinterpret_cast<uint4*>(dst);
    const uint32_t vectors = width / 8, off = elementsOff(src);
    const uint4 zero = make_uint4(0, 0, 0, 0);
    if (!src || (off == 0 && width == dim)) {
        const uint4* from = reinterpret_cast<const uint4*>(src);
        for (uint32_t i0 = lane; i0 < vectors; i0 += 256) {
            uint4 mine[8];
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) mine[k] = src && i0 + 32 * k < vectors ? __ldcs(from + i0 + 32 * k) : zero;
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k)
                if (i0 + 32 * k < vectors) to[i0 + 32 * k] = mine[k];
        }
        return;
    }
    const uint4* from = reinterpret_cast<const uint4*>(src - off);
    const uint32_t there = (off + dim + 7) / 8;  // aligned vectors that hold the row
    // Four vectors of a lane on their way at a time.
    for (uint32_t i0 = 0; i0 < vectors; i0 += 128) {
        uint4 mine[5];
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            const uint32_t i = i0 + 32 * k + lane;
            mine[k] = i < there ? __ldcs(from + i) : zero;
        }
        mine[4] = lane == 0 && i0 + 128 < there ? __ldcs(from + i0 + 128) : zero;
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            const uint32_t i = i0 + 32 * k + lane;
            const uint4 behind = nextLane(mine[k], mine[k + 1], lane);
            if (i < vectors) to[i] = shifted(mine[k], behind, off, i, dim);
        }
    }
}

// Weights whose rows TMA cannot address, copied to 16-byte rows by the blocks
// behind `firstBlock` of the call's first kernel, a warp a row.
struct Align {
    uint32_t firstBlock = UINT32_MAX;
    const __nv_bfloat16* src = nullptr;
    uint64_t ld = 0, vocab = 0;
    uint32_t dim = 0, width = 0;
    __nv_bfloat16* dst = nullptr;
};

__device__ __forceinline__ void alignWeights(const Align& p) {
    const uint32_t lane = threadIdx.x % 32, warps = blockDim.x / 32;
    const uint64_t step = static_cast<uint64_t>(gridDim.x - p.firstBlock) * warps;
    uint64_t v = static_cast<uint64_t>(blockIdx.x - p.firstBlock) * warps + threadIdx.x / 32;
    constexpr uint32_t kRows = 4;
    if (p.dim <= 31 * 8) {
        // Rows that one vector a lane holds, at any offset: four at a time
        // (126737 rows of 234 elements: 54 us one at a time).
        const uint4 zero = make_uint4(0, 0, 0, 0);
        for (; v < p.vocab; v += kRows * step) {
            uint4 mine[kRows];
#pragma unroll
            for (uint32_t k = 0; k < kRows; ++k) {
                const __nv_bfloat16* src = p.src + (v + k * step) * p.ld;
                const uint32_t off = elementsOff(src);
                mine[k] = v + k * step < p.vocab && lane < (off + p.dim + 7) / 8
                              ? __ldcs(reinterpret_cast<const uint4*>(src - off) + lane)
                              : zero;
            }
#pragma unroll
            for (uint32_t k = 0; k < kRows; ++k) {
                const uint4 behind = nextLane(mine[k], zero, lane);
                if (v + k * step < p.vocab && lane < p.width / 8)
                    reinterpret_cast<uint4*>(p.dst + (v + k * step) * p.width)[lane] =
                        shifted(mine[k], behind, elementsOff(p.src + (v + k * step) * p.ld), lane, p.dim);
            }
        }
        return;
    }
    for (; v < p.vocab; v += step) copyRow(p.dst + v * p.width, p.src + v * p.ld, p.dim, p.width, lane);
}

// One warp per row: the teacher's distribution over the row's entries, sorted
// by vocabulary entry (each entry's place is the number of entries before it:
// entries^2 / 32 compares per lane, small beside the row's products). Equal
// ids keep their order and stay separate entries.
constexpr uint32_t kTeacherWarps = 4;
__global__ void __launch_bounds__(32 * kTeacherWarps)
    teacherLists(const int64_t* ids, const void* logits, uint32_t bf16, uint64_t rows,
                 uint32_t entries, uint64_t vocab, float scale, uint32_t* outIds,
                 float* outShares, float* entropy, uint8_t* state,
                 uint32_t* status, const Align align) {
    extern __shared__ uint32_t teacherSmem[];
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    uint32_t* key = teacherSmem + warp * 2 * entries;
    float* s = reinterpret_cast<float*>(key + entries);
    gridDependencyLaunch();
    gridDependencyWait();
    if (blockIdx.x >= align.firstBlock) {
        alignWeights(align);
        return;
    }
    const uint64_t row = static_cast<uint64_t>(blockIdx.x) * kTeacherWarps + warp;
    if (row < rows) {
        const uint64_t list = row * entries;
        float top = -INFINITY;
        bool bad = false, nan = false;
        for (uint32_t e = lane; e < entries; e += 32) {
            const int64_t id = ids[list + e];
            const float x = teacherLogit(logits, bf16, list + e) * scale;
            const bool there = id >= 0 && x != -INFINITY;
            bad |= id >= static_cast<int64_t>(vocab);
            nan |= there && x != x;
            key[e] = there && id < static_cast<int64_t>(vocab) ? static_cast<uint32_t>(id) : kNoEntry;
            s[e] = there ? x : -INFINITY;
            if (there) top = fmaxf(top, x);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        bad = __any_sync(0xffffffffu, bad);
        nan = __any_sync(0xffffffffu, nan);
        const bool live = (top != -INFINITY || nan) && !bad;
        const float shift = top == -INFINITY ? 0.0f : top;
        float total = 0.0f, weighted = 0.0f;
        __syncwarp();
        for (uint32_t e = lane; e < entries; e += 32) {
            const float x = s[e] - shift;
            const float w = expf(x);
            total += w;
            if (w != 0.0f) weighted += w * x;  // w == 0: its share is 0, and x may be -inf
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            total += __shfl_xor_sync(0xffffffffu, total, o);
            weighted += __shfl_xor_sync(0xffffffffu, weighted, o);
        }
        for (uint32_t e = lane; e < entries; e += 32) {
            const uint32_t mine = key[e];
            uint32_t place = 0;
            for (uint32_t f = 0; f < entries; ++f) place += key[f] < mine || (key[f] == mine && f < e);
            outIds[list + place] = mine;
            outShares[list + place] = mine == kNoEntry || !live ? 0.0f : expf(s[e] - shift) / total;
        }
        if (lane == 0) {
            // sum q log q with log q = x - log(total).
            entropy[row] = live ? weighted / total - logf(total) : 0.0f;
            state[row] = bad ? kBad : live ? kLive : kDead;
            if (bad) atomicOr(status, loss::kBoundsStatus);
        }
    }
}

struct PlanParams {
    uint64_t rows, vocab;
    uint32_t dim, ldPacked;
    const __nv_bfloat16* hidden;
    uint64_t ldHidden;
    const int64_t* labels;  // null: `state` says which rows live
    int64_t ignore;
    uint8_t* state;
    __nv_bfloat16* packed;
    uint32_t* count;
    uint32_t* rowMap;
    uint32_t* ids;       // labels only
    float* loss;         // forward
    float* lse;          // forward: written for dead rows; backward: read
    float* rowScale;     // backward
    float* rowLse;       // backward
    const float* gradLoss;
    float scale;
    __nv_bfloat16* gradHidden;
    uint64_t ldGradHidden;
    uint32_t twin;       // a second copy of the packed rows, so many rows on
    uint32_t* status;
};

constexpr uint32_t kPlanThreads = 256;

__device__ __forceinline__ uint8_t rowState(const PlanParams& p, uint64_t row) {
    return p.labels ? labelState(p.labels[row], p.ignore, p.vocab) : p.state[row];
}

// Packs the live rows. Each CTA takes a run of rows and counts the live ones
// before it for itself, which needs no second launch but reads every row's
// label (8 bytes, or a state of 1) in every CTA, up to 4 an SM: 4.7 KB of L2
// reads a row. At 8192 rows that is 39 MB, a few us; at a million rows of a
// narrow head the largest part of the call (1048576 rows, 1000 x 64: 770 us of
// 1900).
__global__ void __launch_bounds__(kPlanThreads) planRows(const PlanParams p, uint32_t blocks, const Align align) {
    __shared__ uint32_t warpSums[2][kPlanThreads / 32];
    __shared__ uint32_t places[kPlanThreads];
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    gridDependencyLaunch();
    gridDependencyWait();
    if (blockIdx.x >= align.firstBlock) {
        alignWeights(align);
        return;
    }
    const uint64_t run = (p.rows + blocks - 1) / blocks;
    const uint64_t lo = min(p.rows, run * blockIdx.x), hi = min(p.rows, lo + run);
    uint32_t before = 0, total = 0;
    for (uint64_t i = threadIdx.x; i < p.rows; i += kPlanThreads) {
        const uint32_t live = rowState(p, i) == kLive;
        total += live;
        before += i < lo ? live : 0u;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        before += __shfl_xor_sync(0xffffffffu, before, o);
        total += __shfl_xor_sync(0xffffffffu, total, o);
    }
    if (lane == 0) {
        warpSums[0][warp] = before;
        warpSums[1][warp] = total;
    }
    __syncthreads();
    before = total = 0;
    for (uint32_t w = 0; w < kPlanThreads / 32; ++w) {
        before += warpSums[0][w];
        total += warpSums[1][w];
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        p.count[0] = total;
        p.count[1] = 0;  // CTAs that have finished (lossGemm)
    }
    for (uint64_t batch = lo; batch < hi; batch += kPlanThreads) {
        const uint64_t row = batch + threadIdx.x;
        const uint8_t state = row < hi ? rowState(p, row) : kDead;
        const uint32_t votes = __ballot_sync(0xffffffffu, state == kLive);
        __syncthreads();  // warpSums and places of the previous round are read
        if (lane == 0) warpSums[0][warp] = __popc(votes);
        __syncthreads();
        uint32_t place = before + __popc(votes & ((1u << lane) - 1u));
        uint32_t all = 0;
        for (uint32_t w = 0; w < kPlanThreads / 32; ++w) {
            if (w < warp) place += warpSums[0][w];
            all += warpSums[0][w];
        }
        places[threadIdx.x] = state == kLive ? place : kNoEntry;
        if (row < hi) {
            if (state == kLive) {
                p.rowMap[place] = static_cast<uint32_t>(row);
                if (p.labels) p.ids[row] = static_cast<uint32_t>(p.labels[row]);
                if (p.gradLoss) {
                    p.rowScale[place] = p.gradLoss[row] * p.scale;
                    p.rowLse[place] = p.lse[row];
                }
            } else if (!p.gradLoss) {
                p.loss[row] = p.lse[row] = state == kBad ? NAN : 0.0f;
            }
            if (state == kBad && p.labels) atomicOr(p.status, loss::kBoundsStatus);
        }
        before += all;
        __syncthreads();
        const uint32_t rowsHere = static_cast<uint32_t>(min(hi - batch, static_cast<uint64_t>(kPlanThreads)));
        for (uint32_t r = warp; r < rowsHere; r += kPlanThreads / 32) {
            const uint32_t to = places[r];
            if (to != kNoEntry) {
                const __nv_bfloat16* from = p.hidden + (batch + r) * p.ldHidden;
                copyRow(p.packed + static_cast<uint64_t>(to) * p.ldPacked, from, p.dim, p.ldPacked, lane);
                if (p.twin) copyRow(p.packed + static_cast<uint64_t>(to + p.twin) * p.ldPacked, from, p.dim, p.ldPacked, lane);
            } else if (p.gradHidden)
                copyRow(p.gradHidden + (batch + r) * p.ldGradHidden, nullptr, p.dim, p.dim, lane);
        }
    }
    // dW's products run over whole k blocks of packed rows: the rows behind
    // the last are zeros.
    if (p.gradLoss) {
        const uint32_t end = ((p.twin ? 2 * p.twin : total) + kBK - 1) / kBK * kBK;
        for (uint32_t r = total + blockIdx.x * (kPlanThreads / 32) + warp; r < end; r += blocks * (kPlanThreads / 32)) {
            if (p.twin && r >= p.twin && r < p.twin + total) continue;
            copyRow(p.packed + static_cast<uint64_t>(r) * p.ldPacked, nullptr, p.ldPacked, p.ldPacked, lane);
        }
    }
}

// ---- join ------------------------------------------------------------------

// kJoinRows packed rows per CTA; 64 threads fold the strips of a row (stored
// row-fastest: eight rows are 64 bytes) and share its list, first within a
// warp, then over the warps in order. One thread closes the loss
//   lse = scale maximum + log(sum),  loss = sum q log q - sum q z + lse.
constexpr uint32_t kJoinRows = 8, kJoinThreads = 512;

__global__ void __launch_bounds__(kJoinThreads)
    joinStrips(const float2* strips, uint64_t stripLd, uint32_t stripCount, const uint32_t* count, const uint32_t* rowMap,
               const uint32_t* ids, const float* shares, const float* listed, const float* entropy, uint32_t entries,
               float scale, float* loss, float* lse) {
    constexpr uint32_t kWarps = kJoinThreads / 32, kGroups = kJoinThreads / kJoinRows;
    __shared__ float tops[kWarps][kJoinRows], sums[kWarps][kJoinRows], targets[kWarps][kJoinRows];
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const uint32_t mine = threadIdx.x % kJoinRows, group = threadIdx.x / kJoinRows;
    gridDependencyLaunch();
    gridDependencyWait();
    const uint32_t row = blockIdx.x * kJoinRows + mine;
    const bool live = row < *count;
    const float c = scale * kLog2e;
    float top = -INFINITY, sum = 0.0f, target = 0.0f;
    uint64_t to = 0;
    if (live) {
        to = rowMap[row];
#pragma unroll 4
        for (uint32_t s = group; s < stripCount; s += kGroups) {
            const float2 x = strips[s * stripLd + row];
            fold(top, sum, x.x, x.y, c);
        }
        for (uint32_t e = group; e < entries; e += kGroups) {
            if (ids[to * entries + e] == kNoEntry) break;  // the list is sorted
            const float share = shares ? shares[to * entries + e] : 1.0f;
            // A share of nothing takes nothing, whatever z is.
            if (share != 0.0f) target += share * listed[to * entries + e];
        }
    }
#pragma unroll
    for (uint32_t o = kJoinRows; o < 32; o *= 2) {
        fold(top, sum, __shfl_xor_sync(0xffffffffu, top, o), __shfl_xor_sync(0xffffffffu, sum, o), c);
        target += __shfl_xor_sync(0xffffffffu, target, o);
    }
    if (lane < kJoinRows) {
        tops[warp][mine] = top;
        sums[warp][mine] = sum;
        targets[warp][mine] = target;
    }
    __syncthreads();
    if (threadIdx.x < kJoinRows && live) {
        for (uint32_t w = 1; w < kWarps; ++w) {
            fold(top, sum, tops[w][mine], sums[w][mine], c);
            target += targets[w][mine];
        }
        closeRow(to, top, sum, scale, target, entropy, loss, lse);
    }
}

// grad_hidden of the packed rows: the splits' sums (and those of the twin rows,
// twinStride on) added in a fixed order, rounded once, and scattered to their rows. GROUPS threads share the splits
// of four elements.
template <uint32_t GROUPS, bool TWIN>
__global__ void __launch_bounds__(256)
    finishHidden(const float* acc, uint64_t splitStride, uint32_t splits, uint64_t twinStride, uint32_t ld, uint32_t dim,
                 const uint32_t* count, const uint32_t* rowMap, __nv_bfloat16* out, uint64_t ldOut) {
    constexpr uint32_t kAcross = 256 / GROUPS;  // groups of four elements a CTA works on
    __shared__ float4 sums[GROUPS][kAcross];
    gridDependencyLaunch();
    gridDependencyWait();
    const uint32_t rows = *count;
    const uint32_t vectors = (dim + 3) / 4;
    const uint64_t all = static_cast<uint64_t>(rows) * vectors;
    const uint32_t group = threadIdx.x / kAcross, mine = threadIdx.x % kAcross;
    for (uint64_t first = static_cast<uint64_t>(blockIdx.x) * kAcross; first < all;
         first += static_cast<uint64_t>(gridDim.x) * kAcross) {
        const uint64_t i = first + mine;
        const uint32_t row = static_cast<uint32_t>(i / vectors), col = static_cast<uint32_t>(i % vectors) * 4;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (i < all) {
            const float* src = acc + static_cast<uint64_t>(row) * ld + col;
#pragma unroll 4
            for (uint32_t s = group; s < splits; s += GROUPS) {
                float4 w = __ldcs(reinterpret_cast<const float4*>(src + s * splitStride));
                if constexpr (TWIN) {
                    const float4 t = __ldcs(reinterpret_cast<const float4*>(src + s * splitStride + twinStride));
                    w.x += t.x;
                    w.y += t.y;
                    w.z += t.z;
                    w.w += t.w;
                }
                v.x += w.x;
                v.y += w.y;
                v.z += w.z;
                v.w += w.w;
            }
        }
        if constexpr (GROUPS > 1) {
            sums[group][mine] = v;
            __syncthreads();
            if (group == 0) {
#pragma unroll
                for (uint32_t g = 1; g < GROUPS; ++g) {
                    const float4 w = sums[g][mine];
                    v.x += w.x;
                    v.y += w.y;
                    v.z += w.z;
                    v.w += w.w;
                }
            }
            __syncthreads();
        }
        if (group == 0 && i < all) {
            __nv_bfloat16* dst = out + rowMap[row] * ldOut + col;
            if (col + 4 <= dim && reinterpret_cast<uintptr_t>(dst) % 8 == 0) {
                uint2 packed;
                __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&packed);
                h[0] = __floats2bfloat162_rn(v.x, v.y);
                h[1] = __floats2bfloat162_rn(v.z, v.w);
                *reinterpret_cast<uint2*>(dst) = packed;
            } else {
                const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j)
                    if (col + j < dim) dst[j] = __float2bfloat16_rn(e[j]);
            }
        }
    }
}

// ---- host ------------------------------------------------------------------

bool weightAligned(const Problem& q) {
    return q.ldWeight % 8 == 0 && reinterpret_cast<uintptr_t>(q.weight) % 16 == 0;
}

uint64_t roundUp(uint64_t x, uint64_t to) { return (x + to - 1) / to * to; }

// Launches with programmatic stream serialization: the kernel's prologue may
// overlap the tail of the kernel before it in the stream, and it waits
// (griddepcontrol.wait) before it touches memory.
template <class... Formal, class... Actual>
cudaError_t launch(void (*kernel)(Formal...), uint32_t grid, uint32_t block, uint32_t smemBytes, cudaStream_t stream,
                   uint32_t cluster, Actual&&... args) {
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(grid);
    config.blockDim = dim3(block);
    config.dynamicSmemBytes = smemBytes;
    config.stream = stream;
    cudaLaunchAttribute attributes[2]{};
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attributes;
    config.numAttrs = 1;
    if (cluster > 1) {
        attributes[1].id = cudaLaunchAttributeClusterDimension;
        attributes[1].val.clusterDim.x = cluster;
        attributes[1].val.clusterDim.y = 1;
        attributes[1].val.clusterDim.z = 1;
        config.numAttrs = 2;
    }
    return cudaLaunchKernelEx(&config, kernel, static_cast<Formal>(args)...);
}

constexpr int kKnownDevices = 64;  // what is remembered of a device, is of the first 64

// Clusters of two that fit on the current device at once (SMs left over by the
// GPC layout, which differs from one GPU to the next, cannot host a pair);
// asked once a device (`known`), a query that failed again with the next call.
template <class Kernel>
uint32_t residentPairs(Kernel kernel, uint32_t threads, uint32_t smemBytes, int smCount,
                       std::atomic<uint32_t> (&known)[kKnownDevices]) {
    const uint32_t fallback = static_cast<uint32_t>(smCount) / 2;
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return fallback;
    if (device < kKnownDevices)
        if (const uint32_t pairs = known[device].load(std::memory_order_relaxed)) return pairs;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(2);
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smemBytes;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = 2;
    attribute.val.clusterDim.y = 1;
    attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    int clusters = 0;
    if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &config) != cudaSuccess) {
        (void)cudaGetLastError();
        return fallback;
    }
    if (clusters < 1) return fallback;
    if (device < kKnownDevices) known[device].store(static_cast<uint32_t>(clusters), std::memory_order_relaxed);
    return static_cast<uint32_t>(clusters);
}

// Lets the kernel use its shared memory, once a device (`ready`).
template <class Kernel>
cudaError_t allowShared(Kernel kernel, uint32_t smemBytes, std::atomic<uint64_t>& ready) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const uint64_t bit = device < kKnownDevices ? 1ull << device : 0;
    if (!bit || !(ready.load(std::memory_order_acquire) & bit)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smemBytes));
        if (e != cudaSuccess) return e;
        ready.fetch_or(bit, std::memory_order_release);
    }
    return cudaSuccess;
}

template <bool A_MN, bool B_MN, int EPI, bool PAIR>
cudaError_t launchTyped(const CUtensorMap& a, const CUtensorMap& b, const Params& p, uint64_t maxTiles, int smCount,
                        cudaStream_t stream) {
    auto kernel = lossGemm<A_MN, B_MN, EPI, PAIR>;
    constexpr uint32_t smemBytes = Geometry<PAIR, EPI>::smemBytes;
    static std::atomic<uint64_t> ready{0};
    const cudaError_t e = allowShared(kernel, smemBytes, ready);
    if (e != cudaSuccess) return e;
    uint32_t slots = static_cast<uint32_t>(smCount);
    if constexpr (PAIR) {
        static std::atomic<uint32_t> pairs[kKnownDevices]{};
        const uint32_t resident = residentPairs(kernel, threadsFor(EPI), smemBytes, smCount, pairs);
        slots = std::min(resident, static_cast<uint32_t>(smCount) / 2);
    }
    const uint32_t grid = static_cast<uint32_t>(std::min<uint64_t>(maxTiles, slots)) * (PAIR ? 2u : 1u);
    return launch(kernel, grid, threadsFor(EPI), smemBytes, stream, PAIR ? 2u : 1u, a, b, p);
}

// Rows of a K-major A that a tile loads: fewer than 128 when there are fewer,
// in whole swizzle atoms.
uint32_t blockRows(uint64_t m) { return static_cast<uint32_t>(std::min<uint64_t>(kBM, roundUp(m, 8))); }

// Columns of a tile for n columns of logits: tiles of the same width in whole
// waves over the SMs. A narrower tile reads A more often, which counts as 16
// more columns a tile (a 64-row pass over 32768 x 2048 weights in one wave of
// 147 tiles of 224 columns instead of 128 of 256; a small vocabulary in tiles
// of 32 on as many SMs as it has).
uint32_t tileColumns(uint64_t mTiles, uint64_t n, uint64_t slots) {
    uint32_t best = kBN;
    uint64_t least = UINT64_MAX;
    for (uint32_t w = kBN; w >= 32; w -= 32) {
        const uint64_t waves = (mTiles * ((n + w - 1) / w) + slots - 1) / slots;
        if (waves * (w + 16) < least) {
            least = waves * (w + 16);
            best = w;
        }
    }
    return best;
}

template <bool A_MN, bool B_MN, int EPI>
cudaError_t gemm(const CUtensorMap& a, const CUtensorMap& b, Params& p, uint64_t maxM, bool pair, int smCount,
                 cudaStream_t stream) {
    const uint64_t tileM = pair ? 2 * kBM : kBM;
    // Slopes are written for whole k blocks of the products that read them.
    const uint32_t n = givesSlopes(EPI) ? static_cast<uint32_t>(roundUp(p.n, kBK)) : p.n;
    if (B_MN) p.tileN = kBN;
    p.aRows = blockRows(maxM);
    p.nTiles = (n + p.tileN - 1) / p.tileN;
    p.group = 16;
    const uint64_t tiles = (maxM + tileM - 1) / tileM * p.nTiles * p.splits;
    if (tiles > UINT32_MAX / 2) return cudaErrorInvalidValue;
    if constexpr (!givesTwins(EPI)) {  // (its rows fit half a CTA's)
        if (pair) return launchTyped<A_MN, B_MN, EPI, true>(a, b, p, tiles, smCount, stream);
    }
    return launchTyped<A_MN, B_MN, EPI, false>(a, b, p, tiles, smCount, stream);
}

template <bool PAIR>
cudaError_t launchBoth(const CUtensorMap& slopesK, const CUtensorMap& weightMN, const CUtensorMap& slopesMN,
                       const CUtensorMap& hiddenMN, Params& h, Params& w, uint64_t maxRows, uint32_t hidden, int smCount,
                       cudaStream_t stream) {
    auto kernel = bothGradients<PAIR>;
    constexpr uint32_t smemBytes = Geometry<PAIR, kEpiOut>::smemBytes;
    static_assert(smemBytes >= Geometry<PAIR, kEpiAcc>::smemBytes);
    static std::atomic<uint64_t> ready{0};
    const cudaError_t e = allowShared(kernel, smemBytes, ready);
    if (e != cudaSuccess) return e;
    uint32_t units = static_cast<uint32_t>(smCount);
    if constexpr (PAIR) {
        static std::atomic<uint32_t> pairs[kKnownDevices]{};
        const uint32_t resident = residentPairs(kernel, threadsFor(kEpiOut), smemBytes, smCount, pairs);
        units = std::max(2u, std::min(resident, static_cast<uint32_t>(smCount) / 2));
    }
    if ((w.m + kBM - 1ull) / kBM * ((w.n + kBN - 1ull) / kBN) > UINT32_MAX / 2) return cudaErrorInvalidValue;
    h.aRows = w.aRows = blockRows(maxRows);
    h.tileN = w.tileN = kBN;
    h.nTiles = w.nTiles = (h.n + kBN - 1) / kBN;
    h.group = w.group = 16;
    return launch(kernel, units * (PAIR ? 2u : 1u), threadsFor(kEpiOut), smemBytes, stream, PAIR ? 2u : 1u, slopesK, weightMN,
                  slopesMN, hiddenMN, h, w, std::min(hidden, units - 1));
}

// CTA pairs need at least one full 128-row block for each CTA to pay.
bool pairFor(uint64_t m) { return m > kBM; }

// Sizes of one problem and where each part of the workspace lies.
struct Layout {
    uint64_t rowsPad, dimPad;
    uint32_t tileN, pieceTileN;  // columns of a logits tile: over the vocabulary, over a piece
    uint64_t stripCount;
    uint64_t piece, pieces;  // vocabulary columns of a piece (a multiple of 256)
    uint32_t splits;         // of dH's products
    uint32_t twin;           // rows of slopes, and behind them as many of what their rounding left; 0: one
    bool direct;             // dH in one go, straight to its rows
    uint32_t hiddenUnits;    // CTAs or pairs for dH, dW on the others; 0: one after the other
    uint32_t scoreCtas;      // of scoreFew, both passes; 0: the logits go to the tensor cores
    uint64_t count, rowMap, rowScale, rowLse, state, ids, shares, entropy, packed, weights;
    uint64_t strips, listed;  // forward
    uint64_t slopes, acc;     // backward (shares the forward's place)
    uint64_t bytes;
};

// Columns of a vocabulary piece: 2^28 slopes (512 MB), so that dH's f32
// accumulator is read and written a few times only, but no piece under 4096
// columns, where that traffic would catch up with the piece's products.
constexpr uint64_t kPieceElements = 1ull << 28, kMinPiece = 4096;
constexpr uint64_t kMaxSplits = 128;

// How dH and dW share the SMs. dH has few tiles and a long k (the piece): it
// is split over k, the splits' sums joined afterwards. In us: 0.27 a k block
// of a tile and 10 blocks' worth to begin and end it; the partial sums,
// written and read at about 5 TB/s; 3 for the launch that joins them, 5 for
// another product's.
//
// One after the other, dH takes at least the time to read the weights and dW
// to write as much (6.5 and 3.7 TB/s); a tile of dW at least 1.6 to read out,
// 4 where rows are no whole vectors. At the same time, on a part of the SMs
// each, both take at least that of the mixed traffic (4.5 to 5 TB/s is what
// this kernel reaches, short of the 6.5 of a copy); few
// SMs read less than they compute, 0.5 us a k block of a single CTA; and
// products that fill the SMs lose about a tenth to shorter waves. So this wins
// where launches and memory count (the gradients' call: 64 rows, 32768 x 2048
// 107 -> 96 us; 512 rows, 32768 x 1024 111 -> 100; 1024 rows, 4096 x 512 60 ->
// 46) and not where the products do (2048 rows, 65536 x 2048: 1190 apart,
// 1290 to 1340 together, the power cap moving either by a tenth).
void planGradients(Layout& l, uint64_t rows, uint64_t width, uint64_t dim, uint64_t mTiles, uint64_t slots, bool pair) {
    const uint64_t nTiles = (dim + kBN - 1) / kBN, tiles = mTiles * nTiles, blocks = (width + kBK - 1) / kBK;
    const auto over = [](uint64_t a, uint64_t b) { return (a + b - 1) / b; };
    const double block = 0.27, partial = static_cast<double>(rows * dim * 8) * 2e-7;
    double hidden = 0.0;
    for (uint64_t s = 1; s <= kMaxSplits && (s == 1 || 2 * s <= blocks); ++s) {
        const double cost = block * static_cast<double>(over(tiles * s, slots) * (over(blocks, s) + 10)) +
                            (s > 1 || l.pieces > 1 ? 3.0 + static_cast<double>(s) * partial : 0.0);
        if (s == 1 || cost < hidden) {
            hidden = cost;
            l.splits = static_cast<uint32_t>(s);
        }
    }
    l.hiddenUnits = 0;
    if (l.pieces > 1 || slots < 4) return;
    const uint64_t weightTiles = over(width, pair ? 2 * kBM : kBM) * nTiles;
    const double weightTile = std::max(block * static_cast<double>(over(rows, kBK)) + 0.3, dim % 8 ? 4.0 : 1.6);
    const double bytes = static_cast<double>(width * dim * 2);
    const double apart = std::max(hidden, bytes / 6.5e6) + 5.0 +
                         std::max(static_cast<double>(over(weightTiles, slots)) * weightTile, bytes / 3.7e6);
    double least = apart;
    for (uint64_t waves = 1; waves <= 2; ++waves) {
        for (uint64_t s = 1; s <= kMaxSplits && (s == 1 || 2 * s <= blocks) && over(tiles * s, waves) <= slots / 2; ++s) {
            const uint64_t units = over(tiles * s, waves);
            const double work =
                std::max((pair ? block : 0.5) * static_cast<double>(waves * (over(blocks, s) + 10)) +
                             static_cast<double>(s) * partial,
                         static_cast<double>(over(weightTiles, slots - units)) * weightTile);
            const double cost = 3.0 + std::max(1.1 * work, 2.0 * bytes / 5e6);
            if (cost < least) {
                least = cost;
                l.splits = static_cast<uint32_t>(s);
                l.hiddenUnits = static_cast<uint32_t>(units);
            }
        }
    }
}

// CTAs of scoreFew, 0 where the tensor cores do better: more than 8 rows; more
// than 4 over more than 2^21 weights (4 MB) that need no copy first
// (linear_score.cuh has the figures); rows too long for shared memory. One a
// SM, but no warp without a row of weights, and one for each class of them.
uint32_t scoreCtas(uint64_t rows, uint64_t vocab, uint64_t dim, bool aligned, int smCount) {
    if (rows > kScoreRows || (rows > 4 && aligned && vocab * dim > (1ull << 21)) ||
        scoreHeight(rows) * scoreLd(dim) * 4 > kScoreShared || smCount < 8)
        return 0;
    return static_cast<uint32_t>(std::clamp<uint64_t>((vocab + kScoreWarps - 1) / kScoreWarps, 8, smCount));
}

Layout layoutFor(uint64_t rows, uint64_t vocab, uint64_t dim, uint64_t entries, bool backward, bool aligned, int smCount) {
    Layout l{};
    if (rows == 0) return l;
    l.rowsPad = roundUp(rows, 256);
    l.dimPad = roundUp(dim, 8);
    const uint64_t most = std::max(kMinPiece, kPieceElements / l.rowsPad / kBN * kBN);
    l.pieces = (vocab + most - 1) / most;
    l.piece = roundUp((vocab + l.pieces - 1) / l.pieces, kBN);
    l.pieces = (vocab + l.piece - 1) / l.piece;
    const bool pair = pairFor(rows);
    const uint64_t tileM = pair ? 256 : 128, slots = pair ? smCount / 2 : smCount;
    const uint64_t mTiles = (rows + tileM - 1) / tileM;
    l.tileN = tileColumns(mTiles, vocab, slots);
    l.pieceTileN = tileColumns(mTiles, std::min(l.piece, vocab), slots);
    l.stripCount = (vocab + l.tileN - 1) / l.tileN * stripsOf(l.tileN);
    l.splits = 1;
    if (backward) planGradients(l, rows, std::min(l.piece, vocab), dim, mTiles, slots, pair);
    l.scoreCtas = scoreCtas(rows, vocab, dim, aligned, smCount);
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) {
        const uint64_t here = at;
        at = roundUp(at + bytes, 1024);
        return here;
    };
    l.count = take(8);  // live rows; CTAs that have finished
    l.rowMap = take(l.rowsPad * 4);
    l.rowScale = take(l.rowsPad * 4);
    l.rowLse = take(l.rowsPad * 4);
    l.state = take(rows);
    l.ids = take(rows * entries * 4);
    l.shares = take(rows * entries * 4);
    l.entropy = take(rows * 4);
    l.packed = take(l.rowsPad * l.dimPad * 2);
    l.weights = take(aligned || (l.scoreCtas && !backward) ? 0 : vocab * l.dimPad * 2);
    const uint64_t shared = at;
    l.strips = take(l.stripCount * l.rowsPad * 8);  // more than scoreFew's, at most 8 a 16 rows of weights
    l.listed = take(rows * entries * 4);
    l.bytes = at;
    if (backward) {
        at = shared;
        l.slopes = take(l.rowsPad * l.piece * 2);
        l.twin = rows <= kBM / 2 ? static_cast<uint32_t>(roundUp(rows, 8)) : 0;
        l.direct = l.pieces == 1 && l.splits == 1 && !l.hiddenUnits && !l.twin;
        l.acc = take(l.direct ? 0 : l.splits * l.rowsPad * l.dimPad * 4);
        l.bytes = std::max(l.bytes, at);
    }
    return l;
}

template <class T>
T* place(const Problem& q, uint64_t offset) {
    return reinterpret_cast<T*>(static_cast<uint8_t*>(q.workspace) + offset);
}

void requireWorkspace(const Problem& q, const Layout& l) {
    if (q.workspaceBytes < l.bytes)
        fail(Category::Validation, "GPU-LOSS-WORKSPACE", "the workspace has " + std::to_string(q.workspaceBytes) +
                                                             " bytes, this call needs " + std::to_string(l.bytes));
}

uint64_t entriesOf(const Problem& q) { return q.labels ? 1 : q.entries; }

cudaError_t teacher(const Problem& q, const Layout& l, const Align& align, uint32_t alignBlocks, uint32_t* status,
                    cudaStream_t stream) {
    return launch(teacherLists, static_cast<uint32_t>((q.rows + kTeacherWarps - 1) / kTeacherWarps) + alignBlocks,
                  32 * kTeacherWarps, static_cast<uint32_t>(kTeacherWarps * 8 * q.entries), stream, 1, q.teacherIds,
                  q.teacherLogits, q.teacherBf16 ? 1u : 0u, q.rows, static_cast<uint32_t>(q.entries), q.vocab, q.scale,
                  place<uint32_t>(q, l.ids), place<float>(q, l.shares), place<float>(q, l.entropy),
                  place<uint8_t>(q, l.state), status, align);
}

// The lists, the packed rows and, where needed, the aligned weights, in one
// launch for labels and two for a teacher.
cudaError_t plan(const Problem& q, const Layout& l, bool backward, int smCount, uint32_t* status, cudaStream_t stream,
                 const void*& weight, uint64_t& ldWeight) {
    cudaError_t e = cudaSuccess;
    weight = q.weight;
    ldWeight = q.ldWeight;
    Align align;
    uint32_t alignBlocks = 0;
    if (!weightAligned(q)) {
        align.src = static_cast<const __nv_bfloat16*>(q.weight);
        align.ld = q.ldWeight;
        align.vocab = q.vocab;
        align.dim = static_cast<uint32_t>(q.dim);
        align.width = static_cast<uint32_t>(l.dimPad);
        align.dst = place<__nv_bfloat16>(q, l.weights);
        alignBlocks = static_cast<uint32_t>(std::min<uint64_t>((q.vocab + 7) / 8, smCount * 8ull));
        weight = align.dst;
        ldWeight = l.dimPad;
    }
    const Align none;
    if (!q.labels) {
        align.firstBlock = static_cast<uint32_t>((q.rows + kTeacherWarps - 1) / kTeacherWarps);
        // (Blocks of half the threads: twice as many.)
        e = teacher(q, l, align, 2 * alignBlocks, status, stream);
        if (e != cudaSuccess) return e;
        alignBlocks = 0;
        align = none;
    }
    PlanParams p{};
    p.rows = q.rows;
    p.vocab = q.vocab;
    p.dim = static_cast<uint32_t>(q.dim);
    p.ldPacked = static_cast<uint32_t>(l.dimPad);
    p.hidden = static_cast<const __nv_bfloat16*>(q.hidden);
    p.ldHidden = q.ldHidden;
    p.labels = q.labels;
    p.ignore = q.ignore;
    p.state = place<uint8_t>(q, l.state);
    p.packed = place<__nv_bfloat16>(q, l.packed);
    p.count = place<uint32_t>(q, l.count);
    p.rowMap = place<uint32_t>(q, l.rowMap);
    p.ids = place<uint32_t>(q, l.ids);
    p.loss = q.loss;
    p.lse = q.lse;
    p.rowScale = place<float>(q, l.rowScale);
    p.rowLse = place<float>(q, l.rowLse);
    p.gradLoss = backward ? q.gradLoss : nullptr;
    p.scale = q.scale;
    p.gradHidden = backward ? static_cast<__nv_bfloat16*>(q.gradHidden) : nullptr;
    p.ldGradHidden = q.ldGradHidden;
    p.twin = l.twin;
    p.status = status;
    const uint32_t blocks = static_cast<uint32_t>(std::min<uint64_t>((q.rows + 7) / 8, smCount * 4ull));
    if (alignBlocks) align.firstBlock = blocks;
    e = launch(planRows, blocks + alignBlocks, kPlanThreads, 0, stream, 1, p, blocks, align);
    return e;
}

template <uint32_t T, bool SLOPES>
cudaError_t launchScoreRows(const ScoreParams& p, uint32_t ctas, cudaStream_t stream) {
    static std::atomic<uint64_t> ready{0};
    const cudaError_t e = allowShared(scoreFew<T, SLOPES>, kScoreShared, ready);
    if (e != cudaSuccess) return e;
    return launch(scoreFew<T, SLOPES>, ctas, kScoreThreads, static_cast<uint32_t>(T * scoreLd(p.dim) * 4), stream, 1, p);
}

template <bool SLOPES>
cudaError_t launchScore(const ScoreParams& p, uint32_t ctas, cudaStream_t stream) {
    switch (scoreHeight(p.rows)) {
    case 1: return launchScoreRows<1, SLOPES>(p, ctas, stream);
    case 2: return launchScoreRows<2, SLOPES>(p, ctas, stream);
    case 4: return launchScoreRows<4, SLOPES>(p, ctas, stream);
    default: return launchScoreRows<8, SLOPES>(p, ctas, stream);
    }
}

// What both passes of a few rows share.
ScoreParams scoreParams(const Problem& q, const Layout& l, uint32_t* status) {
    ScoreParams p{};
    p.weight = static_cast<const __nv_bfloat16*>(q.weight);
    p.ldWeight = q.ldWeight;
    p.rows = static_cast<uint32_t>(q.rows);
    p.vocab = static_cast<uint32_t>(q.vocab);
    p.dim = static_cast<uint32_t>(q.dim);
    p.entries = static_cast<uint32_t>(entriesOf(q));
    p.classes = 8;
    while (p.classes > 1 && q.ldWeight * p.classes / 2 % 8 == 0) p.classes /= 2;
    p.scale = q.scale;
    p.ids = place<uint32_t>(q, l.ids);
    p.shares = q.labels ? nullptr : place<float>(q, l.shares);
    p.status = status;
    return p;
}

cudaError_t score(const Problem& q, const Layout& l, uint32_t* status, cudaStream_t stream) {
    cudaError_t e = cudaSuccess;
    if (!q.labels) e = teacher(q, l, Align{}, 0, status, stream);
    if (e != cudaSuccess) return e;
    ScoreParams p = scoreParams(q, l, status);
    p.hidden = static_cast<const __nv_bfloat16*>(q.hidden);
    p.ldHidden = q.ldHidden;
    p.labels = q.labels;
    p.ignore = q.ignore;
    p.state = place<uint8_t>(q, l.state);
    p.entropy = place<float>(q, l.entropy);
    p.strips = place<float2>(q, l.strips);
    p.listed = place<float>(q, l.listed);
    p.loss = q.loss;
    p.lse = q.lse;
    e = launchScore<false>(p, l.scoreCtas, stream);
    if (e != cudaSuccess) return e;
    return launch(closeFew, p.rows, kCloseThreads, 0, stream, 1, p, l.scoreCtas);
}

} // namespace

std::uint64_t workspaceBytes(std::uint64_t rows, std::uint64_t vocab, std::uint64_t dim, std::uint64_t entries,
                             bool backward, bool aligned, int smCount) {
    return layoutFor(rows, vocab, dim, entries, backward, aligned, smCount).bytes;
}

cudaError_t forward(const Problem& q, int smCount, std::uint32_t* status, cudaStream_t stream) {
    if (q.rows == 0) return cudaSuccess;
    const uint64_t entries = entriesOf(q);
    const Layout l = layoutFor(q.rows, q.vocab, q.dim, entries, false, weightAligned(q), smCount);
    requireWorkspace(q, l);
    if (l.scoreCtas) return score(q, l, status, stream);
    const void* weight = nullptr;
    uint64_t ldWeight = 0;
    cudaError_t e = plan(q, l, false, smCount, status, stream, weight, ldWeight);
    if (e != cudaSuccess) return e;
    const bool pair = pairFor(q.rows) && smCount >= 2;
    CUtensorMap a, b;
    if (!makeMap(&a, place<void>(q, l.packed), l.dimPad, l.rowsPad, l.dimPad, blockRows(q.rows)) ||
        !makeMap(&b, weight, q.dim, q.vocab, ldWeight, pair ? l.tileN / 2 : l.tileN))
        return cudaErrorInvalidValue;
    Params p{};
    p.count = place<uint32_t>(q, l.count);
    p.countIsM = 1;
    p.n = static_cast<uint32_t>(q.vocab);
    p.k = static_cast<uint32_t>(q.dim);
    p.splits = 1;
    p.tileN = l.tileN;
    p.blocksPerSum = kBlocksPerSum;
    p.scale = q.scale;
    p.entries = static_cast<uint32_t>(entries);
    p.rowMap = place<uint32_t>(q, l.rowMap);
    p.ids = place<uint32_t>(q, l.ids);
    p.listed = place<float>(q, l.listed);
    p.shares = q.labels ? nullptr : place<float>(q, l.shares);
    p.strips = place<float2>(q, l.strips);
    p.stripLd = l.rowsPad;
    p.status = status;
    p.spins = waitSpins();
    // Rows that the last CTA of the products joins by itself, saving a launch
    // where a call is little more than its launches. (128 rows would take it
    // 37 us instead of the 5 of joinStrips.)
    constexpr uint64_t kFewRows = 32;
    const bool few = q.rows <= kFewRows;
    if (few) {
        p.finished = place<uint32_t>(q, l.count) + 1;
        p.entropy = q.labels ? nullptr : place<float>(q, l.entropy);
        p.loss = q.loss;
        p.lse = q.lse;
    }
    e = gemm<false, false, kEpiLse>(a, b, p, q.rows, pair, smCount, stream);
    if (e != cudaSuccess || few) return e;
    return launch(joinStrips, static_cast<uint32_t>((q.rows + kJoinRows - 1) / kJoinRows), kJoinThreads, 0, stream, 1,
                  p.strips, p.stripLd, static_cast<uint32_t>(l.stripCount), p.count, p.rowMap, p.ids, p.shares, p.listed,
                  q.labels ? nullptr : place<float>(q, l.entropy), p.entries, q.scale, q.loss, q.lse);
}

cudaError_t backward(const Problem& q, int smCount, std::uint32_t* status, cudaStream_t stream) {
    if (q.rows == 0)
        return cudaMemset2DAsync(q.gradWeight, q.ldGradWeight * 2, 0, q.dim * 2, q.vocab, stream);
    const uint64_t entries = entriesOf(q);
    const Layout l = layoutFor(q.rows, q.vocab, q.dim, entries, true, weightAligned(q), smCount);
    requireWorkspace(q, l);
    const void* weight = nullptr;
    uint64_t ldWeight = 0;
    cudaError_t e = plan(q, l, true, smCount, status, stream, weight, ldWeight);
    if (e != cudaSuccess) return e;
    const bool pair = pairFor(q.rows) && smCount >= 2;
    const bool pairW = pairFor(q.vocab) && smCount >= 2;
    void* packed = place<void>(q, l.packed);
    void* slopes = place<void>(q, l.slopes);
    const uint64_t slopeRows = l.twin ? 2 * l.twin : q.rows;
    CUtensorMap hiddenK, weightK, slopesK, weightMN, slopesMN, hiddenMN;
    if (!makeMap(&hiddenK, packed, l.dimPad, l.rowsPad, l.dimPad, blockRows(q.rows)) ||
        !makeMap(&weightK, weight, q.dim, q.vocab, ldWeight, pair ? l.pieceTileN / 2 : l.pieceTileN) ||
        !makeMap(&slopesK, slopes, l.piece, l.rowsPad, l.piece, blockRows(slopeRows)) ||
        !makeMap(&weightMN, weight, q.dim, q.vocab, ldWeight, 64) ||
        // (scoreFew writes the rows of both summands; those behind are read as zeros.)
        !makeMap(&slopesMN, slopes, l.piece, l.scoreCtas ? slopeRows : l.rowsPad, l.piece, 64) ||
        !makeMap(&hiddenMN, packed, l.dimPad, l.rowsPad, l.dimPad, 64))
        return cudaErrorInvalidValue;
    Params base{};
    base.count = place<uint32_t>(q, l.count);
    base.splits = 1;
    base.status = status;
    base.spins = waitSpins();
    for (uint64_t i = 0; i < l.pieces; ++i) {
        const uint64_t first = i * l.piece, width = std::min(l.piece, q.vocab - first);
        Params s = base;
        s.countIsM = 1;
        s.n = static_cast<uint32_t>(width);
        s.k = static_cast<uint32_t>(q.dim);
        s.tileN = l.pieceTileN;
        s.bFirstN = static_cast<uint32_t>(first);
        s.scale = q.scale;
        s.entries = static_cast<uint32_t>(entries);
        s.rowMap = place<uint32_t>(q, l.rowMap);
        s.ids = place<uint32_t>(q, l.ids);
        s.shares = q.labels ? nullptr : place<float>(q, l.shares);
        s.rowLse = place<float>(q, l.rowLse);
        s.rowScale = place<float>(q, l.rowScale);
        s.twin = l.twin;
        s.c = slopes;
        s.ldc = l.piece;
        s.blocksPerSum = kBlocksPerSum;
        if (l.scoreCtas) {  // (up to kScoreRows rows: their twins are as many on)
            ScoreParams f = scoreParams(q, l, status);
            f.hidden = static_cast<const __nv_bfloat16*>(packed);
            f.ldHidden = l.dimPad;
            f.weight += first * q.ldWeight;
            f.vocab = static_cast<uint32_t>(width);
            f.first = static_cast<uint32_t>(first);
            f.count = base.count;
            f.rowMap = s.rowMap;
            f.rowLse = s.rowLse;
            f.rowScale = s.rowScale;
            f.slopes = static_cast<__nv_bfloat16*>(slopes);
            f.ldSlopes = l.piece;
            e = launchScore<true>(f, l.scoreCtas, stream);
        } else if (q.dim <= kBlocksPerSum * kBK)
            e = l.twin ? gemm<false, false, kEpiTwin>(hiddenK, weightK, s, q.rows, false, smCount, stream)
                       : gemm<false, false, kEpiSlope>(hiddenK, weightK, s, q.rows, pair, smCount, stream);
        else
            e = l.twin ? gemm<false, false, kEpiTwinSums>(hiddenK, weightK, s, q.rows, false, smCount, stream)
                       : gemm<false, false, kEpiSlopeSums>(hiddenK, weightK, s, q.rows, pair, smCount, stream);
        if (e != cudaSuccess) return e;
        Params h = base;
        h.countIsM = !l.twin;
        h.m = static_cast<uint32_t>(slopeRows);
        h.n = static_cast<uint32_t>(q.dim);
        h.k = static_cast<uint32_t>(width);
        h.bFirstK = static_cast<uint32_t>(first);
        if (l.direct) {
            h.rowMap = place<uint32_t>(q, l.rowMap);
            h.c = q.gradHidden;
            h.ldc = q.ldGradHidden;
        } else {
            // A last, narrower piece may have too few k blocks for every split.
            const uint32_t blocks = static_cast<uint32_t>((width + kBK - 1) / kBK);
            h.blocksPerSplit = (blocks + l.splits - 1) / l.splits;
            h.splits = (blocks + h.blocksPerSplit - 1) / h.blocksPerSplit;
            h.c = place<void>(q, l.acc);
            h.ldc = l.dimPad;
            h.splitStride = l.rowsPad * l.dimPad;
            h.accumulate = i > 0;
        }
        Params w = base;
        w.countIsK = 1;
        w.k = 2 * l.twin;
        w.m = static_cast<uint32_t>(width);
        w.n = static_cast<uint32_t>(q.dim);
        w.c = static_cast<__nv_bfloat16*>(q.gradWeight) + first * q.ldGradWeight;
        w.ldc = q.ldGradWeight;
        if (l.hiddenUnits) {
            e = (pair ? launchBoth<true> : launchBoth<false>)(slopesK, weightMN, slopesMN, hiddenMN, h, w, slopeRows,
                                                              l.hiddenUnits, smCount, stream);
        } else {
            e = l.direct ? gemm<false, true, kEpiOut>(slopesK, weightMN, h, slopeRows, pair, smCount, stream)
                         : gemm<false, true, kEpiAcc>(slopesK, weightMN, h, slopeRows, pair, smCount, stream);
            if (e == cudaSuccess) e = gemm<true, true, kEpiOut>(slopesMN, hiddenMN, w, width, pairW, smCount, stream);
        }
        if (e != cudaSuccess) return e;
    }
    if (l.direct) return cudaSuccess;
    const uint32_t firstBlocks = static_cast<uint32_t>((std::min(l.piece, q.vocab) + kBK - 1) / kBK);
    const uint32_t perSplit = (firstBlocks + l.splits - 1) / l.splits;
    const uint32_t used = (firstBlocks + perSplit - 1) / perSplit;  // splits the first piece wrote
    const uint64_t vectors = q.rows * ((q.dim + 3) / 4);
    const bool shared = used >= 8;
    const uint32_t across = shared ? 32 : 256;
    const auto finish = [&](auto kernel) {
        return launch(kernel, static_cast<uint32_t>(std::min<uint64_t>((vectors + across - 1) / across, smCount * 8ull)), 256, 0,
                      stream, 1, place<float>(q, l.acc), l.rowsPad * l.dimPad, used, l.twin * l.dimPad,
                      static_cast<uint32_t>(l.dimPad), static_cast<uint32_t>(q.dim), base.count, place<uint32_t>(q, l.rowMap),
                      static_cast<__nv_bfloat16*>(q.gradHidden), q.ldGradHidden);
    };
    if (l.twin) return shared ? finish(finishHidden<8, true>) : finish(finishHidden<1, true>);
    return shared ? finish(finishHidden<8, false>) : finish(finishHidden<1, false>);
}

} // namespace thb::linear_loss
