// lse and loss of a few rows (a token at a time, a short batch), and their
// slopes: the logits of the linear losses without tensor cores.
//
// Up to kScoreRows rows the products are small beside the weights that they
// read, so that the weights are streamed once through plain loads, each
// element multiplied with the rows' elements from shared memory. A warp takes
// a run of weight rows, four at a time, and keeps a running (maximum, sum) for
// every row. No packing and no copies: rows of weights at any address are read
// in the aligned 16-byte vectors that hold them, against H shifted as far. Rows
// with the same shift are `classes` apart; a CTA takes those of one class.
//
// The slopes of rows that were scored here are computed here too, from the same
// sums: exp(z - lse) of a well-known label is 1 less a small rest, which the
// tensor cores' roundings of z would drown (8 rows of 4096 products, logits
// around 40: off by 5e-5 where 1e-4 was right). They are written as the tensor
// cores' kernel writes those of few rows, in two bf16 summands.
//
// Against the tensor cores' path, us a call in a graph (whose weights stay in
// L2 where they fit): 1 row, 32768 x 1024 11.6 to 17.9, 4 rows 17.7 to 18.3;
// 1 row, 131072 x 4096 166 to 186 (reading the weights at the copy rate is
// 164); 1 row of odd width, 50021 x 1003, 21 to 65, 8 rows 46 to 65; 1 row,
// 4096 x 512 5.8 to 13.1, 8 rows 10.5 to 13.1. Past a row or two the reads of H
// from shared memory bound it. The gradients' call with its slopes from here
// and from the tensor cores: 1 row, 32768 x 1024 64 and 66, 4 rows 75 and 67; 1
// row, 131072 x 4096 687 and 667; 8 rows, 50021 x 1003 176 and 146.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "loss_parts.cuh"
#include "loss_status.hpp"

namespace thb::linear_loss {

constexpr uint32_t kScoreRows = 8, kScoreThreads = 512, kScoreWarps = kScoreThreads / 32;
constexpr uint32_t kScoreAcross = 4;  // weight rows of a warp side by side
constexpr uint32_t kScoreShared = 200 << 10;

struct ScoreParams {
    const __nv_bfloat16* hidden;
    uint64_t ldHidden;
    const __nv_bfloat16* weight;
    uint64_t ldWeight;
    uint32_t rows, vocab, dim, entries;
    uint32_t classes;  // a power of two: rows v and v + classes start equally far from a 16-byte boundary
    float scale;
    const int64_t* labels;  // null: the lists
    int64_t ignore;
    const uint8_t* state;    // of the lists' rows
    const uint32_t* ids;     // [row][entries], ascending, kNoEntry behind the last
    const float* shares;     // [row][entries]
    const float* entropy;    // [row]
    float2* strips;          // [row][CTA] (maximum, sum)
    float* listed;           // z of each list entry, [row][entries]
    float* loss;
    float* lse;
    uint32_t* status;
    // Slopes: `weight` and `vocab` are those of a piece of the vocabulary, from
    // entry `first` (a multiple of 8) on; `hidden` is packed.
    uint32_t first;
    const uint32_t* count;   // packed rows
    const uint32_t* rowMap;  // packed row -> row
    const float* rowLse;     // packed
    const float* rowScale;   // packed: scale * grad_loss
    __nv_bfloat16* slopes;   // [2 kScoreRows][ldSlopes], what the roundings left behind the slopes
    uint64_t ldSlopes;
};

__device__ __forceinline__ uint8_t stateOf(const ScoreParams& p, uint32_t row) {
    return p.labels ? labelState(p.labels[row], p.ignore, p.vocab) : p.state[row];
}

// H in shared memory, f32: its rows (zeros behind the last) and floats a row.
constexpr uint32_t scoreHeight(uint64_t rows) { return rows <= 2 ? static_cast<uint32_t>(rows) : rows <= 4 ? 4 : 8; }
__host__ __device__ constexpr uint64_t scoreLd(uint64_t dim) { return (dim + 14) / 8 * 8; }

// Both halves of a bf16 pair; bf16 is the upper half of f32.
__device__ __forceinline__ float2 widened(uint32_t pair) {
    return make_float2(__uint_as_float(pair << 16), __uint_as_float(pair & 0xffff0000u));
}

// Where place e of a row of H lies in shared memory: the first halves of all
// vectors, then the second ones, so that a warp's 16-byte reads meet every bank
// once.
__device__ __forceinline__ uint32_t placeOf(uint32_t e, uint32_t vectors) {
    return (e % 8 / 4 * vectors + e / 8) * 4 + e % 4;
}

// A row of H, `off` places up, zeros around it (and throughout without `from`).
__device__ __forceinline__ void fillRow(float* h, const __nv_bfloat16* from, uint32_t dim, uint32_t off, uint32_t vectors) {
    if (from && off == 0 && dim % 8 == 0 && reinterpret_cast<uintptr_t>(from) % 16 == 0) {
#pragma unroll 2
        for (uint32_t i = threadIdx.x; i < vectors; i += kScoreThreads) {
            const uint4 raw = reinterpret_cast<const uint4*>(from)[i];
            const float2 a = widened(raw.x), b = widened(raw.y), c = widened(raw.z), d = widened(raw.w);
            reinterpret_cast<float4*>(h)[i] = make_float4(a.x, a.y, b.x, b.y);
            reinterpret_cast<float4*>(h)[vectors + i] = make_float4(c.x, c.y, d.x, d.y);
        }
    } else {
#pragma unroll 4
        for (uint32_t e = threadIdx.x; e < vectors * 8; e += kScoreThreads)
            h[placeOf(e, vectors)] = from && e >= off && e < off + dim ? __bfloat162float(from[e - off]) : 0.0f;
    }
}

// The elements of vector i of a row that starts `off` places into vector 0 and
// has `dim` of them; the others, of neighbouring rows, become 0.
__device__ __forceinline__ uint4 ownPart(uint4 x, uint32_t i, uint32_t off, uint32_t dim) {
    uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (uint32_t k = 0; k < 8; ++k) {
        const uint32_t e = i * 8 + k;
        if (e < off || e >= off + dim) w[k / 2] &= k % 2 ? 0x0000ffffu : 0xffff0000u;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// A lane's part of h[t] . w[r] for T rows of H and R rows of weights (vectors
// that hold them, the first `off` elements of vector 0 not theirs), at
// [t * R + r]. Sums of f32, even and odd elements apart.
template <uint32_t T, uint32_t R>
__device__ __forceinline__ void dots(const uint4* const (&w)[R], const float* h, uint32_t ldh, uint32_t dim, uint32_t off,
                                     uint32_t lane, float (&z)[T * R]) {
    // Vectors of a row that are loaded at once (8 rows of H leave registers for
    // half as many: 50021 x 1003 70 us else, 46 so).
    constexpr uint32_t kAhead = (T == 8 ? 4 : 8) / R;
    const uint32_t vectors = (off + dim + 7) / 8;
    const bool ragged = (off + dim) % 8 != 0;
    float2 sums[T * R];
#pragma unroll
    for (uint32_t i = 0; i < T * R; ++i) sums[i] = make_float2(0.0f, 0.0f);
    for (uint32_t first = lane; first < vectors; first += 32 * kAhead) {
        uint4 x[kAhead][R];
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a) {
            const uint32_t i = first + a * 32;
            if (i < vectors) {
#pragma unroll
                for (uint32_t r = 0; r < R; ++r) x[a][r] = w[r][i];
            }
        }
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a) {
            const uint32_t i = first + a * 32;
            if (i >= vectors) break;
            if ((off && i == 0) || (ragged && i == vectors - 1)) {
#pragma unroll
                for (uint32_t r = 0; r < R; ++r) x[a][r] = ownPart(x[a][r], i, off, dim);
            }
            float2 v[R][4];
#pragma unroll
            for (uint32_t r = 0; r < R; ++r) {
                v[r][0] = widened(x[a][r].x);
                v[r][1] = widened(x[a][r].y);
                v[r][2] = widened(x[a][r].z);
                v[r][3] = widened(x[a][r].w);
            }
#pragma unroll
            for (uint32_t t = 0; t < T; ++t) {
                const float4 lo = *reinterpret_cast<const float4*>(h + t * ldh + i * 4);
                const float4 hi = *reinterpret_cast<const float4*>(h + t * ldh + (vectors + i) * 4);
#pragma unroll
                for (uint32_t r = 0; r < R; ++r) {
                    float2& s = sums[t * R + r];
                    s = fma2(v[r][0], make_float2(lo.x, lo.y), s);
                    s = fma2(v[r][1], make_float2(lo.z, lo.w), s);
                    s = fma2(v[r][2], make_float2(hi.x, hi.y), s);
                    s = fma2(v[r][3], make_float2(hi.z, hi.w), s);
                }
            }
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < T * R; ++i) z[i] = sums[i].x + sums[i].y;
}

// Sums over the warp of N values (a power of two) a lane: lane l returns that
// of value n, the bits of n from the highest being those of l from the lowest.
// One tree whatever N, so that equal products give equal sums.
template <uint32_t N>
__device__ __forceinline__ float warpSums(float (&v)[N], uint32_t lane) {
    uint32_t bit = 1;
#pragma unroll
    for (uint32_t width = N / 2; width >= 1; width /= 2, bit *= 2) {
        const bool upper = lane & bit;
#pragma unroll
        for (uint32_t i = 0; i < width; ++i) {
            const float send = upper ? v[i] : v[i + width], keep = upper ? v[i + width] : v[i];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, send, bit);
        }
    }
#pragma unroll
    for (uint32_t o = N; o < 32; o *= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    return v[0];
}

// The bits of x below `below` (a power of two) in reverse.
template <uint32_t BELOW>
__device__ __forceinline__ uint32_t reversed(uint32_t x) {
    uint32_t y = 0;
#pragma unroll
    for (uint32_t bit = 1; bit < BELOW; bit *= 2) y = y * 2 + (x & bit ? 1 : 0);
    return y;
}

// The running maximum of a row and the sum of 2^((z - maximum) c); a sum of
// nothing but -inf takes any finite maximum.
struct Running {
    float top = -INFINITY, sum = 0.0f;

    __device__ __forceinline__ void take(float z, float c) {
        if (z > top) {
            sum *= pow2((top - z) * c);
            top = z;
        }
        sum += pow2((z - (top == -INFINITY ? 0.0f : top)) * c);
    }
};

// What a lane knows of the row of H whose slopes it gives: the place in its
// list from the current entry of the vocabulary on.
struct SlopeRow {
    float lse = 0.0f, scale = 0.0f;
    uint64_t list = 0;
    uint32_t at = 0, next = kNoEntry;
    bool live = false;

    __device__ __forceinline__ void step(const ScoreParams& p) {
        next = ++at < p.entries ? p.ids[list + at] : kNoEntry;
    }

    // The list's first entry from `entry` on.
    __device__ __forceinline__ void begin(const ScoreParams& p, uint32_t row, uint32_t rows, uint32_t entry) {
        live = row < rows;
        if (!live) return;
        lse = p.rowLse[row];
        scale = p.rowScale[row];
        list = static_cast<uint64_t>(p.rowMap[row]) * p.entries;
        uint32_t end = p.entries;
        while (at < end) {
            const uint32_t middle = (at + end) / 2;
            if (p.ids[list + middle] < entry) at = middle + 1;
            else end = middle;
        }
        next = at < p.entries ? p.ids[list + at] : kNoEntry;
    }

    // The slope at z (unscaled) of `entry`, rounded as in the tensor cores' kernel.
    __device__ __forceinline__ float take(const ScoreParams& p, float z, uint32_t entry) {
        float slope = __fmul_rn(scale, pow2(__fmul_rn(__fadd_rn(__fmul_rn(z, p.scale), -lse), kLog2e)));
        while (next < entry) step(p);
        while (next == entry) {
            slope = __fsub_rn(slope, scale * (p.shares ? p.shares[list + at] : 1.0f));
            step(p);
        }
        return slope;
    }
};

// `slope` of packed row `row` in two summands at column v.
__device__ __forceinline__ void giveSlope(const ScoreParams& p, uint32_t row, uint32_t v, float slope) {
    const __nv_bfloat16 high = __float2bfloat16_rn(slope);
    p.slopes[row * p.ldSlopes + v] = high;
    p.slopes[(row + kScoreRows) * p.ldSlopes + v] = __float2bfloat16_rn(slope - __bfloat162float(high));
}

// The slopes behind those of the packed rows are operands of the next products:
// zeros, in rows up to kScoreRows and in columns up to the end of a k block of
// 64. A CTA fills a run of 16-byte vectors in each row.
__device__ __forceinline__ void zeroSlopes(const ScoreParams& p, uint32_t packed) {
    const uint32_t vectors = (p.vocab + 63) / 64 * 8;
    const uint32_t first = static_cast<uint32_t>(static_cast<uint64_t>(vectors) * blockIdx.x / gridDim.x);
    const uint32_t end = static_cast<uint32_t>(static_cast<uint64_t>(vectors) * (blockIdx.x + 1) / gridDim.x);
    for (uint32_t row = packed; row < 2 * kScoreRows; ++row) {
        if (row % kScoreRows < packed) continue;
        uint4* to = reinterpret_cast<uint4*>(p.slopes + row * p.ldSlopes);
        for (uint32_t i = first + threadIdx.x; i < end; i += kScoreThreads) to[i] = make_uint4(0, 0, 0, 0);
    }
    const uint32_t behind = (p.vocab + 63) / 64 * 64 - p.vocab;
    if (blockIdx.x == 0)
        for (uint32_t e = threadIdx.x; e < packed * behind; e += kScoreThreads)
            giveSlope(p, e / behind, p.vocab + e % behind, 0.0f);
}

template <uint32_t T, bool SLOPES>
__global__ void __launch_bounds__(kScoreThreads, 1) scoreFew(const ScoreParams p) {
    extern __shared__ float4 sharedHidden[];
    __shared__ float2 parts[kScoreWarps][T];
    float* h = reinterpret_cast<float*>(sharedHidden);
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t ldh = static_cast<uint32_t>(scoreLd(p.dim));
    // This CTA's weight rows: own, own + classes, ...
    const uint32_t own = blockIdx.x % p.classes;
    const auto rowAt = [&](uint32_t v) { return p.weight + v * p.ldWeight; };
    const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(rowAt(own)) / 2 % 8), vectors = (off + p.dim + 7) / 8;
    const auto vectorsAt = [&](uint32_t v) { return reinterpret_cast<const uint4*>(rowAt(v) - off); };
    gridDependencyLaunch();
    gridDependencyWait();
    // Without a target no row needs the weights.
    const uint32_t packed = SLOPES ? *p.count : 0u;
    if (SLOPES && packed == 0) return;
    const bool mine = !SLOPES && threadIdx.x < p.rows && stateOf(p, threadIdx.x) == kLive;
#pragma unroll
    for (uint32_t t = 0; t < T; ++t)  // (packed rows: zeros behind the last)
        fillRow(h + t * ldh, SLOPES || t < p.rows ? p.hidden + t * p.ldHidden : nullptr, p.dim, off, vectors);
    if (!__syncthreads_or(mine) && !SLOPES) return;

    // A run of them for each warp.
    const uint32_t at = blockIdx.x / p.classes * kScoreWarps + warp;
    const uint32_t of = (gridDim.x - own + p.classes - 1) / p.classes * kScoreWarps;
    const uint64_t count = own < p.vocab ? (p.vocab - own + p.classes - 1) / p.classes : 0u;
    uint32_t i = static_cast<uint32_t>(count * at / of);
    const uint32_t end = static_cast<uint32_t>(count * (at + 1) / of);
    const float c = p.scale * kLog2e;
    // Lane l holds row reversed<T>(l) of H, of weight rows reversed<kScoreAcross>(l / T).
    Running run;
    SlopeRow row;
    const uint32_t t = reversed<T>(lane);
    if constexpr (SLOPES) row.begin(p, t, packed, p.first + own + i * p.classes);
    for (; i + kScoreAcross <= end; i += kScoreAcross) {
        const uint4* w[kScoreAcross];
#pragma unroll
        for (uint32_t r = 0; r < kScoreAcross; ++r) w[r] = vectorsAt(own + (i + r) * p.classes);
        float z[T * kScoreAcross];
        dots<T>(w, h, ldh, p.dim, off, lane, z);
        const float x = warpSums(z, lane);
        if constexpr (SLOPES) {
            const uint32_t v = own + (i + reversed<kScoreAcross>(lane / T)) * p.classes;
            if (lane < T * kScoreAcross && row.live) giveSlope(p, t, v, row.take(p, x, p.first + v));
        } else {
            if (lane < T * kScoreAcross) run.take(x, c);
        }
    }
    for (; i < end; ++i) {
        const uint32_t v = own + i * p.classes;
        const uint4* const w[1] = {vectorsAt(v)};
        float z[T];
        dots<T>(w, h, ldh, p.dim, off, lane, z);
        const float x = warpSums(z, lane);
        if constexpr (SLOPES) {
            if (lane < T && row.live) giveSlope(p, t, v, row.take(p, x, p.first + v));
        } else {
            if (lane < T) run.take(x, c);
        }
    }
    if constexpr (SLOPES) {
        zeroSlopes(p, packed);
        return;
    }
#pragma unroll
    for (uint32_t o = T; o < T * kScoreAcross; o *= 2)
        fold(run.top, run.sum, __shfl_xor_sync(0xffffffffu, run.top, o), __shfl_xor_sync(0xffffffffu, run.sum, o), c);
    if (lane < T) parts[warp][t] = make_float2(run.top, run.sum);

    // z where a list (a label) names an entry of this class, a warp an entry.
    for (uint32_t e = at; e < p.rows * p.entries; e += of) {
        const uint32_t to = e / p.entries;
        if (stateOf(p, to) != kLive) continue;
        const uint32_t id = p.labels ? static_cast<uint32_t>(p.labels[to]) : p.ids[e];
        if (id == kNoEntry || id % p.classes != own) continue;
        const uint4* const w[1] = {vectorsAt(id)};
        float z[1];
        dots<1>(w, h + to * ldh, ldh, p.dim, off, lane, z);
        const float x = warpSums(z, lane);
        if (lane == 0) p.listed[e] = x * p.scale;
    }
    __syncthreads();
    if (threadIdx.x < T && threadIdx.x < p.rows) {
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (uint32_t k = 0; k < kScoreWarps; ++k) fold(top, sum, parts[k][threadIdx.x].x, parts[k][threadIdx.x].y, c);
        p.strips[threadIdx.x * gridDim.x + blockIdx.x] = make_float2(top, sum);
    }
}

// A CTA a row: the strips of scoreFew's `ctas`, the targets, the loss. Rows
// without a target have 0, those with one outside the vocabulary NaN.
constexpr uint32_t kCloseThreads = 128;

__global__ void __launch_bounds__(kCloseThreads) closeFew(const ScoreParams p, uint32_t ctas) {
    constexpr uint32_t kWarps = kCloseThreads / 32;
    __shared__ float tops[kWarps], sums[kWarps], targets[kWarps];
    const uint32_t row = blockIdx.x, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    gridDependencyLaunch();
    gridDependencyWait();
    const uint8_t state = stateOf(p, row);
    if (state != kLive) {
        if (threadIdx.x == 0) {
            p.loss[row] = p.lse[row] = state == kBad ? NAN : 0.0f;
            if (state == kBad && p.labels) atomicOr(p.status, loss::kBoundsStatus);
        }
        return;
    }
    const float c = p.scale * kLog2e;
    float top = -INFINITY, sum = 0.0f, target = 0.0f;
    for (uint32_t s = threadIdx.x; s < ctas; s += kCloseThreads) {
        const float2 x = p.strips[row * ctas + s];
        fold(top, sum, x.x, x.y, c);
    }
    for (uint32_t e = threadIdx.x; e < p.entries; e += kCloseThreads) {
        if (!p.labels && p.ids[row * p.entries + e] == kNoEntry) break;  // the list is sorted
        const float share = p.labels ? 1.0f : p.shares[row * p.entries + e];
        // A share of nothing takes nothing, whatever z is.
        if (share != 0.0f) target += share * p.listed[row * p.entries + e];
    }
#pragma unroll
    for (uint32_t o = 1; o < 32; o *= 2) {
        fold(top, sum, __shfl_xor_sync(0xffffffffu, top, o), __shfl_xor_sync(0xffffffffu, sum, o), c);
        target += __shfl_xor_sync(0xffffffffu, target, o);
    }
    if (lane == 0) {
        tops[warp] = top;
        sums[warp] = sum;
        targets[warp] = target;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (uint32_t w = 1; w < kWarps; ++w) {
            fold(top, sum, tops[w], sums[w], c);
            target += targets[w];
        }
        closeRow(row, top, sum, p.scale, target, p.labels ? nullptr : p.entropy, p.loss, p.lse);
    }
}

} // namespace thb::linear_loss
