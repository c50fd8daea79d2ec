// Distillation from a teacher's top logits, student logits [rows][vocab] in
// memory (bf16 or f32): the loss, and its gradient in the same pass.
//
// The bound is HBM: one read of the logits and one write of their gradient.
// A softmax needs a row twice, so a row stays on chip between. CTAs are
// persistent and take rows in turn; a row passes through a ring of chunks in
// shared memory, kVectors 16-byte vectors a thread and chunk:
//   copy warp   starts bulk copies into chunks as they come free, a row ahead
//               where the ring has room;
//   list warp   rows ahead: the teacher's list and its softmax, the student's
//               logits at the entries, which rows have a target (the others
//               are not read);
//   the others  sum a row's chunks as they arrive (running maximum and sum of
//               exponentials per thread), fold them over the CTA, and go over
//               the row again to write the gradient, from the chunks that
//               the ring still holds and, for rows longer than it, from chunks
//               copied again (from L2: the rows in work on all SMs are a few
//               tens of MB). The teacher's entries then overwrite their places.
// Two CTAs share an SM, so that one's exponentials fill the other's folds and
// waits. The folds have a fixed order: equal inputs give equal bits.
//
// Every wait is bounded. A warp whose wait ran out says so at the next barrier
// of the CTA's computing warps, behind which none of them goes on: a row's list
// names places in memory, and nobody uses one that was not handed over.
//
// When there are fewer rows than CTAs, a cluster of up to 8 shares a row and
// its CTAs send each other their parts by asynchronous stores into
// distributed shared memory.
//
// Rows need not start at 16-byte boundaries (an odd vocabulary): the elements
// before the first boundary and behind the last are the first and the last
// CTA's edges, loaded one by one.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <map>
#include <mutex>
#include <tuple>
#include <type_traits>

#include "distill.hpp"
#include "exponential.cuh"
#include "loss_status.hpp"
#include "tensor_core.cuh"

namespace thb::distill {
namespace {

using namespace thb::tc;

// Vectors of a thread in a chunk. A chunk costs a warp about 50 instructions
// besides its exponentials, and with two CTAs of 8 warps on an SM issue slots
// are nearly as scarce as bytes. 4096 x 65536 bf16 with gradient: 1 vector
// (16 warps) 239 us, 2 (16 warps) 208, 3 (12 warps) 199, 4 (8 warps) 195.
constexpr uint32_t kVectors = 4;
constexpr uint32_t kMaxCluster = 8;
constexpr uint32_t kSmemPerSm = 227 * 1024, kReservedSmem = 3 * 1024;  // static and the system's share of a CTA
constexpr uint32_t kMaxChunks = 16, kMinChunks = 4;
constexpr uint32_t kAhead = 2;   // chunks that a row never keeps from the copies behind it
constexpr uint32_t kLists = 3;   // rows whose lists are kept
constexpr uint32_t kEdges = 16;
constexpr uint32_t kNoEntry = 0x7fffffffu;
constexpr float kLowest = -3.402823466e38f;

enum : int { kScore = 0, kTrain = 1, kBackward = 2 };

struct Params {
    uint64_t rows, vocab, ldLogits, ldGrad;
    const void* logits;
    const int64_t* ids;
    const void* teacher;
    uint32_t teacherBf16;
    uint32_t entries;
    uint32_t cluster;
    uint32_t chunks;  // of the ring
    float scale;
    float* loss;
    float* lse;
    const float* gradLoss;
    void* grad;
    uint32_t* status;
    uint32_t spins;  // tries of a wait
};

// 16-byte vectors of logits as pairs of f32.
template <class T>
struct Vec;
template <>
struct Vec<float> {
    static constexpr uint32_t n = 4;
    static __device__ __forceinline__ void unpack(const uint4& u, float2 (&v)[2]) {
        v[0] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
        v[1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
    }
    static __device__ __forceinline__ uint4 pack(const float2 (&v)[2]) {
        return make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
    }
    // A running maximum over vectors, and its value.
    using Top = float2;
    static __device__ __forceinline__ Top lowest() { return make_float2(-INFINITY, -INFINITY); }
    static __device__ __forceinline__ void raise(Top& top, const uint4& u) {
        top.x = fmaxf(fmaxf(top.x, __uint_as_float(u.x)), __uint_as_float(u.y));
        top.y = fmaxf(fmaxf(top.y, __uint_as_float(u.z)), __uint_as_float(u.w));
    }
    static __device__ __forceinline__ float value(const Top& top) { return fmaxf(top.x, top.y); }
    static __device__ __forceinline__ float get(const float* p) { return *p; }
    static __device__ __forceinline__ float from(float x) { return x; }
};
template <>
struct Vec<__nv_bfloat16> {
    static constexpr uint32_t n = 8;
    static __device__ __forceinline__ void unpack(const uint4& u, float2 (&v)[4]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
    static __device__ __forceinline__ uint4 pack(const float2 (&v)[4]) {
        uint4 u;
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __float22bfloat162_rn(v[i]);
        return u;
    }
    using Top = __nv_bfloat162;
    static __device__ __forceinline__ Top lowest() { return __float2bfloat162_rn(-INFINITY); }
    static __device__ __forceinline__ void raise(Top& top, const uint4& u) {
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
        top = __hmax2(top, __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    }
    static __device__ __forceinline__ float value(const Top& top) {
        return fmaxf(__low2float(top), __high2float(top));
    }
    static __device__ __forceinline__ float get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
    static __device__ __forceinline__ __nv_bfloat16 from(float x) { return __float2bfloat16_rn(x); }
};

__device__ __forceinline__ float warpMax(float x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}
__device__ __forceinline__ float warpSum(float x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

// The part of a row that a CTA holds: head edge | vectors | tail edge.
template <class T>
struct Segment {
    uint64_t first = 0;  // element of its first vector
    uint64_t tail = 0;   // first element of the tail edge
    uint32_t vectors = 0;
    uint32_t headHere = 0, tailHere = 0;  // edge elements of this CTA

    __device__ __forceinline__ Segment() {}
    __device__ __forceinline__ Segment(const T* z, uint64_t vocab, uint32_t cluster, uint32_t rank) {
        constexpr uint32_t N = Vec<T>::n;
        const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(z) % 16 / sizeof(T));
        const uint32_t head = static_cast<uint32_t>(min(static_cast<uint64_t>(off ? N - off : 0u), vocab));
        const uint64_t all = (vocab - head) / N;
        const uint64_t perCta = cluster > 1 ? (all + cluster - 1) / cluster : all;
        const uint64_t v0 = min(all, perCta * rank);
        vectors = static_cast<uint32_t>(min(all, v0 + perCta) - v0);
        first = head + v0 * N;
        tail = head + all * N;
        headHere = rank == 0 ? head : 0u;
        tailHere = rank == cluster - 1 ? static_cast<uint32_t>(vocab - tail) : 0u;
    }
    __device__ __forceinline__ bool holds(uint32_t id) const {
        return (id >= first && id < first + static_cast<uint64_t>(vectors) * Vec<T>::n) || id < headHere ||
               (tailHere && id >= tail);
    }
    __device__ __forceinline__ uint32_t edges() const { return headHere + tailHere; }
    __device__ __forceinline__ uint64_t edge(uint32_t i) const { return i < headHere ? i : tail + (i - headHere); }
};

// Running (maximum, sum of exp(scale (z - maximum))). The maximum starts at
// the lowest finite value, so that -inf adds 0 and the lowest value counts.
struct Running {
    float top = -3.402823466e38f;
    float2 sum = make_float2(0.0f, 0.0f);
    // (All lanes; a vote, since a maximum rises seldom after the first vectors.)
    __device__ __forceinline__ void raise(float to, float c) {
        if (__any_sync(0xffffffffu, to > top)) {
            const float high = fmaxf(to, top), down = pow2((top - high) * c);
            sum = mul2(sum, make_float2(down, down));
            top = high;
        }
    }
};

// Sends four words to the same object in CTA `rank` of the cluster and counts
// their bytes on that CTA's barrier.
__device__ __forceinline__ void sendTo(uint32_t rank, void* to, uint64_t* bar, float4 v) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(
                     pairAddress(to, rank)),
                 "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w), "r"(pairAddress(bar, rank))
                 : "memory");
}

// Bulk copy of `bytes` (a multiple of 16) into shared memory.
__device__ __forceinline__ void bulkLoad(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem(dst)),
                 "l"(src), "r"(bytes), "r"(smem(bar))
                 : "memory");
}

// Whether all that the cluster's CTAs have sent here has landed. Row j is
// counted on barrier j % 2, which this CTA arms when it sends its own part;
// rows before its last were waited for, and no CTA is more than one ahead. After
// an expired wait, parts that were not sent are counted in their place, and
// those of a row that this CTA did not come to are armed.
__device__ bool partsLanded(uint64_t* received, uint32_t here, const uint32_t* by, uint32_t cluster, bool gaveUp) {
    uint32_t missing = 0, ahead = 0;
    for (uint32_t k = 0; k < cluster; ++k) {
        missing += by[k] < here;
        ahead += by[k] > here;
    }
    if (!gaveUp && !missing && !ahead) return true;
    bool all = true;
    if (here) {
        const uint32_t last = here - 1;
        if (missing) mbarComplete(&received[last % 2], 16 * missing);
        all = mbarWait(&received[last % 2], last / 2 % 2);
    }
    if (ahead) {
        mbarExpect(&received[here % 2], 16 * ahead);
        all &= mbarWait(&received[here % 2], here / 2 % 2);
    }
    return all;
}

// A row as the list warp hands it over.
struct RowInfo {
    int state;        // 0: no target, 1: live, 2: an id outside the vocabulary
    uint32_t owned;   // entries in this CTA's segment
    float constant;   // loss less lse: sum q log q - sum q z
    float slope;      // grad_loss * scale
    float lse;        // backward
    float edges[kEdges];
};

// WARPS that compute; two more run ahead.
template <class T, int MODE, uint32_t WARPS>
__global__ void __launch_bounds__(32 * WARPS + 64, WARPS >= 8 ? 2 : 6) distillRows(const Params p) {
    constexpr uint32_t N = Vec<T>::n, kConsumers = 32 * WARPS, kChunk = kConsumers * kVectors;
    extern __shared__ __align__(128) uint8_t dynamicSmem[];
    __shared__ __align__(8) uint64_t full[kMaxChunks], empty[kMaxChunks], listed[kLists], unlisted[kLists], received[2];
    __shared__ __align__(16) float4 records[2][kMaxCluster];
    __shared__ float2 parts[2][WARPS];
    __shared__ RowInfo infos[kLists];
    __shared__ volatile int abortFlag;
    __shared__ uint32_t started, parity;  // bit per slot: a copy was started; its parity
    __shared__ uint32_t sentHere, sentBy[kMaxCluster];  // rows whose part this CTA, each CTA has sent the cluster

    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t rank = p.cluster > 1 ? blockIdx.x % p.cluster : 0u;
    const uint64_t firstRow = blockIdx.x / p.cluster, step = gridDim.x / p.cluster;
    uint4* ring = reinterpret_cast<uint4*>(dynamicSmem);
    // Behind the ring, for each kept row: the entries' ids, shares and logits.
    struct List {
        uint32_t* key;
        float *share, *logit;
    };
    auto listAt = [&](uint32_t i) {
        uint32_t* key = reinterpret_cast<uint32_t*>(ring + p.chunks * kChunk) + i * p.entries * 3;
        return List{key, reinterpret_cast<float*>(key + p.entries), reinterpret_cast<float*>(key + 2 * p.entries)};
    };
    auto logitsOf = [&](uint64_t row) { return static_cast<const T*>(p.logits) + row * p.ldLogits; };
    auto chunksOf = [&](const Segment<T>& seg) { return (seg.vectors + kChunk - 1) / kChunk; };
    // Chunks of a row that stay in the ring between the two passes.
    auto keptOf = [&](uint32_t n) { return MODE == kTrain ? min(n, p.chunks - kAhead) : 0u; };

    if (threadIdx.x == 0) {
        abortFlag = 0;
        sentHere = 0;
        for (uint32_t i = 0; i < kMaxChunks; ++i) {
            mbarInit(&full[i], 1);
            mbarInit(&empty[i], WARPS);
        }
        for (uint32_t i = 0; i < kLists; ++i) {
            mbarInit(&listed[i], 1);
            mbarInit(&unlisted[i], WARPS + 1);
        }
        for (uint32_t i = 0; i < 2; ++i) mbarInit(&received[i], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    if (p.cluster > 1) clusterSync();  // barriers are ready before another CTA sends

    if (warp == WARPS) {
        // ---- copies ----
        if (lane == 0) {
            uint32_t slot = 0, phase = 0, list = 0, listPhase = 0;
            uint32_t begun = 0, phases = 0;  // started, parity
            for (uint64_t row = firstRow; row < p.rows && !abortFlag; row += step) {
                if (!mbarWait(&listed[list], listPhase, &abortFlag, p.spins)) { abortFlag = 1; break; }
                const int state = infos[list].state;
                mbarArrive(&unlisted[list]);
                if (++list == kLists) { list = 0; listPhase ^= 1u; }
                if (state != 1) continue;
                const Segment<T> seg(logitsOf(row), p.vocab, p.cluster, rank);
                const uint4* data = reinterpret_cast<const uint4*>(logitsOf(row) + seg.first);
                const uint32_t n = chunksOf(seg), again = MODE == kTrain ? n - keptOf(n) : 0u;
                for (uint32_t i = 0; i < n + again; ++i) {
                    const uint32_t first = (i < n ? i : i - n) * kChunk;
                    const uint32_t bytes = min(seg.vectors - first, kChunk) * 16;
                    if (!mbarWait(&empty[slot], phase ^ 1u, &abortFlag, p.spins)) { abortFlag = 1; break; }
                    mbarExpect(&full[slot], bytes);
                    bulkLoad(ring + slot * kChunk, data + first, bytes, &full[slot]);
                    begun |= 1u << slot;
                    phases = (phases & ~(1u << slot)) | phase << slot;
                    if (++slot == p.chunks) { slot = 0; phase ^= 1u; }
                }
            }
            started = begun;
            parity = phases;
        }
    } else if (warp == WARPS + 1) {
        // ---- lists ----
        uint32_t at = 0, phase = 0;
        constexpr uint32_t kEarly = 4;  // entries of a lane that are read a row ahead
        int64_t earlyId[kEarly];
        float earlyLogit[kEarly];
        auto idOf = [&](uint64_t row, uint32_t e) { return p.ids[row * p.entries + e]; };
        auto teacherOf = [&](uint64_t row, uint32_t e) {
            const uint64_t i = row * p.entries + e;
            return (p.teacherBf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.teacher)[i])
                                  : static_cast<const float*>(p.teacher)[i]) *
                   p.scale;
        };
        auto readEarly = [&](uint64_t row) {
#pragma unroll
            for (uint32_t k = 0; k < kEarly; ++k) {
                const uint32_t e = lane + 32 * k;
                const bool there = row < p.rows && e < p.entries;
                earlyId[k] = there ? idOf(row, e) : -1;
                earlyLogit[k] = there ? teacherOf(row, e) : -INFINITY;
            }
        };
        readEarly(firstRow);
        for (uint64_t row = firstRow; row < p.rows; row += step) {
            if (!mbarWait(&unlisted[at], phase ^ 1u, &abortFlag, p.spins)) abortFlag = 1;
            if (__any_sync(0xffffffffu, abortFlag)) break;
            const T* z = logitsOf(row);
            const Segment<T> seg(z, p.vocab, p.cluster, rank);
            const List list = listAt(at);
            RowInfo& info = infos[at];
            float top = -INFINITY;
            bool bad = false, nan = false;
            auto take = [&](uint32_t e, int64_t id, float x) {
                if (e >= p.entries) return;
                const bool there = id >= 0 && x != -INFINITY, inside = id < static_cast<int64_t>(p.vocab);
                bad |= !inside;
                nan |= there && x != x;
                list.key[e] = there && inside ? static_cast<uint32_t>(id) : kNoEntry;
                list.share[e] = there ? x : -INFINITY;
                // (Backward, another CTA of the cluster may be writing its part of the row.)
                const bool wanted = there && inside && (MODE != kBackward || seg.holds(static_cast<uint32_t>(id)));
                list.logit[e] = wanted ? Vec<T>::get(z + id) : 0.0f;
                if (there) top = fmaxf(top, x);
            };
#pragma unroll
            for (uint32_t k = 0; k < kEarly; ++k) take(lane + 32 * k, earlyId[k], earlyLogit[k]);
            for (uint32_t e = lane + 32 * kEarly; e < p.entries; e += 32) take(e, idOf(row, e), teacherOf(row, e));
            readEarly(row + step);
            top = warpMax(top);
            bad = __any_sync(0xffffffffu, bad);
            nan = __any_sync(0xffffffffu, nan);
            const int state = bad ? 2 : top != -INFINITY || nan ? 1 : 0;
            if (state == 1) {
                const float shift = top == -INFINITY ? 0.0f : top;
                float total = 0.0f, weighted = 0.0f, target = 0.0f;
                for (uint32_t e = lane; e < p.entries; e += 32) {
                    const float x = list.share[e] - shift, w = expf(x);
                    list.share[e] = w;
                    if (w == 0.0f) continue;  // no share takes nothing, and x or z may be infinite
                    total += w;
                    weighted += w * x;
                    target += w * (list.logit[e] * p.scale);
                }
                total = warpSum(total);
                weighted = warpSum(weighted);
                target = warpSum(target);
                // sum q log q = weighted / total - log(total)
                if (lane == 0) info.constant = (weighted / total - logf(total)) - target / total;
                // The entries in this segment move to the front, in order.
                uint32_t mine = 0;
                for (uint32_t e0 = 0; MODE != kScore && e0 < p.entries; e0 += 32) {
                    const uint32_t e = e0 + lane;
                    const bool inside = e < p.entries;
                    const uint32_t id = inside ? list.key[e] : kNoEntry;
                    const float share = inside ? list.share[e] / total : 0.0f, x = inside ? list.logit[e] : 0.0f;
                    const bool here = id != kNoEntry && seg.holds(id);
                    const uint32_t votes = __ballot_sync(0xffffffffu, here);
                    if (here) {
                        const uint32_t to = mine + __popc(votes & ((1u << lane) - 1u));
                        list.key[to] = id;
                        list.share[to] = share;
                        list.logit[to] = x;
                    }
                    mine += __popc(votes);
                    __syncwarp();
                }
                if (lane < seg.edges()) info.edges[lane] = Vec<T>::get(z + seg.edge(lane));
                if (lane == 0) {
                    info.owned = mine;
                    if constexpr (MODE != kScore) info.slope = p.gradLoss[row] * p.scale;
                    if constexpr (MODE == kBackward) info.lse = p.lse[row];
                }
            }
            if (lane == 0) info.state = state;
            __syncwarp();
            if (lane == 0) mbarArrive(&listed[at]);
            if (++at == kLists) { at = 0; phase ^= 1u; }
        }
    } else {
        // ---- sums and gradients ----
        const float c = p.scale * kLog2e;
        const uint32_t fromLast = kConsumers - 1 - threadIdx.x;  // entries go to the last warps; the first one folds
        uint32_t slot = 0, phase = 0, at = 0, listPhase = 0, turn = 0, recPhase = 0;
        // A wait that runs out ends every later one at once.
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            if (mbarWait(bar, parity, &abortFlag, p.spins)) return true;
            abortFlag = 1;
            return false;
        };
        // A barrier of the computing warps: whether no wait has run out. A warp
        // whose list did not come meets the others at their next barrier, and
        // all leave behind it; those without another row meet it at one behind
        // the loop.
        auto agreed = [&] {
            uint32_t all;
            asm volatile(
                "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.and.pred q, 1, %2, p;\n"
                " selp.u32 %0, 1, 0, q;\n}\n"
                : "=r"(all)
                : "r"(abortFlag ? 0u : 1u), "n"(kConsumers)
                : "memory");
            return all != 0;
        };
        auto advance = [&] {
            if (++slot == p.chunks) { slot = 0; phase ^= 1u; }
        };
        auto release = [&](uint64_t* bar) {
            __syncwarp();
            if (lane == 0) mbarArrive(bar);
        };
        auto fold = [&](float2 part, float& top) {
            top = warpMax(part.x);
            return warpSum(part.y * pow2((part.x - top) * c));
        };
        const float2 none = make_float2(kLowest, 0.0f);

        bool together = true;
        for (uint64_t row = firstRow; row < p.rows; row += step) {
            const Segment<T> seg(logitsOf(row), p.vocab, p.cluster, rank);
            T* grad = MODE == kScore ? nullptr : static_cast<T*>(p.grad) + row * p.ldGrad;
            uint4* gradVectors = reinterpret_cast<uint4*>(grad + seg.first);
            const bool aligned = reinterpret_cast<uintptr_t>(gradVectors) % 16 == 0;
            const bool hasEdge = threadIdx.x < seg.edges();
            auto store = [&](uint32_t v, const float2 (&x)[N / 2]) {
                if (aligned) {
                    __stcs(gradVectors + v, Vec<T>::pack(x));
                } else {
#pragma unroll
                    for (uint32_t j = 0; j < N / 2; ++j) {
                        T* to = grad + seg.first + static_cast<uint64_t>(v) * N + 2 * j;
                        to[0] = Vec<T>::from(x[j].x);
                        to[1] = Vec<T>::from(x[j].y);
                    }
                }
            };
            if (!__all_sync(0xffffffffu, wait(&listed[at], listPhase))) {
                together = agreed();
                break;
            }
            const RowInfo& info = infos[at];
            const int state = info.state;
            if (state != 1) {
                if (threadIdx.x == 0 && rank == 0) {
                    if constexpr (MODE != kBackward) p.loss[row] = p.lse[row] = state == 2 ? NAN : 0.0f;
                    if (state == 2) atomicOr(p.status, loss::kBoundsStatus);
                }
                if constexpr (MODE != kScore) {
                    float2 zeros[N / 2];
#pragma unroll
                    for (uint32_t j = 0; j < N / 2; ++j) zeros[j] = make_float2(0.0f, 0.0f);
                    for (uint32_t v = threadIdx.x; v < seg.vectors; v += kConsumers) store(v, zeros);
                    if (hasEdge) grad[seg.edge(threadIdx.x)] = Vec<T>::from(0.0f);
                }
            } else {
                const float edge = hasEdge ? info.edges[threadIdx.x] : -INFINITY;
                const uint32_t n = chunksOf(seg), kept = keptOf(n);
                float top = 0.0f, sum = 1.0f;
                uint32_t firstKept = 0;
                if constexpr (MODE != kBackward) {
                    // ---- first pass ----
                    Running running;
                    // `whole`: every thread has all its vectors of the chunk.
                    auto take = [&](uint32_t i, auto whole) {
                        const uint4* mine = ring + slot * kChunk + threadIdx.x;
                        const uint32_t v = i * kChunk + threadIdx.x;
                        uint4 raw[kVectors];
                        auto high = Vec<T>::lowest();
#pragma unroll
                        for (uint32_t k = 0; k < kVectors; ++k) {
                            if (!whole && v + k * kConsumers >= seg.vectors) break;
                            raw[k] = mine[k * kConsumers];
                            Vec<T>::raise(high, raw[k]);
                        }
                        running.raise(Vec<T>::value(high), c);
                        const float minusTop = -running.top;
#pragma unroll
                        for (uint32_t k = 0; k < kVectors; ++k) {
                            if (!whole && v + k * kConsumers >= seg.vectors) break;
                            float2 x[N / 2];
                            Vec<T>::unpack(raw[k], x);
#pragma unroll
                            for (uint32_t j = 0; j < N / 2; ++j)
                                running.sum = add2(running.sum, pow2Shifted(x[j], minusTop, c));
                        }
                    };
                    for (uint32_t i = 0; i < n; ++i) {
                        if (i == n - kept) firstKept = slot;
                        wait(&full[slot], phase);
                        if ((i + 1) * kChunk <= seg.vectors) take(i, std::true_type{});
                        else take(i, std::false_type{});
                        if (i < n - kept) release(&empty[slot]);
                        advance();
                    }
                    running.raise(edge, c);  // -inf where there is none: adds 0
                    top = warpMax(running.top);
                    sum = warpSum((running.sum.x + running.sum.y + pow2((edge - running.top) * c)) *
                                  pow2((running.top - top) * c));
                    if (lane == 0) parts[turn][warp] = make_float2(top, sum);
                    if (!(together = agreed())) break;
                    if (p.cluster == 1) {
                        sum = fold(lane < WARPS ? parts[turn][lane] : none, top);
                    } else {
                        if (warp == 0) {
                            sum = fold(lane < WARPS ? parts[turn][lane] : none, top);
                            if (lane == 0) {
                                mbarExpect(&received[turn], 16 * p.cluster);
                                ++sentHere;
                            }
                            if (lane < p.cluster)
                                sendTo(lane, &records[turn][rank], &received[turn], make_float4(top, sum, 0.0f, 0.0f));
                        }
                        wait(&received[turn], recPhase);
                        __syncwarp();
                        const float4 r = lane < p.cluster ? records[turn][lane] : make_float4(kLowest, 0.0f, 0.0f, 0.0f);
                        sum = fold(make_float2(r.x, r.y), top);
                    }
                    if (rank == 0 && threadIdx.x == 0) {
                        const float lse = top * p.scale + logf(sum);
                        p.lse[row] = lse;
                        p.loss[row] = lse + info.constant;
                    }
                    if (++turn == 2) { turn = 0; recPhase ^= 1u; }
                }
                if constexpr (MODE != kScore) {
                    // ---- second pass ----
                    const float slope = info.slope, lse = MODE == kBackward ? info.lse : 0.0f;
                    const float factor = 1.0f / sum, coefficient = slope * factor;
                    auto probability = [&](float x) {
                        if constexpr (MODE == kTrain) return factor * pow2((x - top) * c);
                        else return pow2((x * p.scale - lse) * kLog2e);
                    };
                    auto give = [&](uint32_t i, uint32_t s, auto whole) {
                        const uint4* mine = ring + s * kChunk + threadIdx.x;
                        const uint32_t v = i * kChunk + threadIdx.x;
#pragma unroll
                        for (uint32_t k = 0; k < kVectors; ++k) {
                            if (!whole && v + k * kConsumers >= seg.vectors) break;
                            float2 x[N / 2];
                            Vec<T>::unpack(mine[k * kConsumers], x);
#pragma unroll
                            for (uint32_t j = 0; j < N / 2; ++j) {
                                const float2 e = MODE == kTrain
                                                     ? pow2Shifted(x[j], -top, c)
                                                     : pow2Shifted(mul2(x[j], make_float2(p.scale, p.scale)), -lse, kLog2e);
                                x[j] = mul2(e, make_float2(coefficient, coefficient));
                            }
                            if (whole) __stcs(gradVectors + v + k * kConsumers, Vec<T>::pack(x));
                            else store(v + k * kConsumers, x);
                        }
                    };
                    auto write = [&](uint32_t i, uint32_t s) {
                        if (aligned && (i + 1) * kChunk <= seg.vectors) give(i, s, std::true_type{});
                        else give(i, s, std::false_type{});
                        release(&empty[s]);
                    };
                    for (uint32_t i = n - kept, s = firstKept; i < n && MODE == kTrain; ++i) {
                        write(i, s);
                        if (++s == p.chunks) s = 0;
                    }
                    for (uint32_t i = 0; i < n - kept; ++i) {
                        wait(&full[slot], phase);
                        write(i, slot);
                        advance();
                    }
                    if (hasEdge) grad[seg.edge(threadIdx.x)] = Vec<T>::from(slope * probability(edge));
                    if constexpr (MODE == kBackward) {
                        if (!(together = agreed())) break;
                    } else {
                        asm volatile("barrier.sync 1, %0;" ::"n"(kConsumers) : "memory");  // all agreed on this row
                    }
                    // The entries' places, behind the stores above: p less the
                    // shares of the id, which the first of equal ids writes.
                    const List list = listAt(at);
                    const uint32_t owned = info.owned;
                    for (uint32_t e = fromLast; e < owned; e += kConsumers) {
                        const uint32_t id = list.key[e];
                        float share = 0.0f;
                        bool before = false;
#pragma unroll 4
                        for (uint32_t f = 0; f < owned; ++f) {
                            const bool same = list.key[f] == id;
                            before |= same && f < e;
                            share += same ? list.share[f] : 0.0f;
                        }
                        if (!before) grad[id] = Vec<T>::from(slope * (probability(list.logit[e]) - share));
                    }
                }
            }
            release(&unlisted[at]);
            if (++at == kLists) { at = 0; listPhase ^= 1u; }
        }
        if (together) agreed();
    }
    __syncthreads();
    if (threadIdx.x == 0 && abortFlag) {
        // Whoever gave up: copies in flight land before the CTA leaves.
        bool drained = true;
        for (uint32_t i = 0; i < p.chunks; ++i)
            if (started >> i & 1u) drained &= mbarWait(&full[i], parity >> i & 1u);
        atomicOr(p.status, kWaitStatus | (drained ? 0u : kDrainStatus));
    }
    if (p.cluster > 1) {
        if (threadIdx.x < p.cluster) storeCluster(pairAddress(&sentBy[rank], threadIdx.x), sentHere);
        clusterSync();  // nothing is sent to a CTA that has left
        if (threadIdx.x == 0 && !partsLanded(received, sentHere, sentBy, p.cluster, abortFlag))
            atomicOr(p.status, kWaitStatus | kDrainStatus);
    }
}

cudaLaunchConfig_t configFor(uint32_t grid, uint32_t threads, uint32_t smemBytes, uint32_t cluster,
                             cudaLaunchAttribute& attribute, cudaStream_t stream) {
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(grid);
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smemBytes;
    config.stream = stream;
    attribute = cudaLaunchAttribute{};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = cluster;
    attribute.val.clusterDim.y = 1;
    attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    return config;
}

// Clusters of this shape that fit on the device at once.
cudaError_t residentClusters(void (*kernel)(Params), uint32_t threads, uint32_t cluster, uint32_t smemBytes, int device,
                             uint32_t& out) {
    static std::mutex mutex;
    static std::map<std::tuple<void (*)(Params), int, uint32_t, uint32_t>, uint32_t> known;
    std::lock_guard<std::mutex> lock(mutex);
    auto found = known.find({kernel, device, cluster, smemBytes});
    if (found == known.end()) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             static_cast<int>(kSmemPerSm - kReservedSmem));
        if (e != cudaSuccess) return e;
        cudaLaunchAttribute attribute;
        const cudaLaunchConfig_t config = configFor(cluster, threads, smemBytes, cluster, attribute, nullptr);
        int clusters = 0;
        e = cudaOccupancyMaxActiveClusters(&clusters, kernel, &config);
        if (e != cudaSuccess) return e;
        if (clusters < 1) return cudaErrorInvalidConfiguration;
        if (known.size() > 4096) known.clear();
        found = known.emplace(std::make_tuple(kernel, device, cluster, smemBytes), static_cast<uint32_t>(clusters)).first;
    }
    out = found->second;
    return cudaSuccess;
}

template <class T, int MODE, uint32_t WARPS>
cudaError_t launchTyped(const Problem& q, int smCount, uint32_t* status, cudaStream_t stream) {
    constexpr uint32_t N = Vec<T>::n, kPerSm = WARPS >= 8 ? 2 : 6, kThreads = 32 * WARPS + 64;
    constexpr uint32_t kChunkBytes = 32 * WARPS * kVectors * 16;
    auto kernel = distillRows<T, MODE, WARPS>;
    const uint64_t rowBytes = (q.vocab + N - 1) / N * 16;
    // The ring takes what the lists leave of a CTA's share of an SM, or its
    // least size (fewer CTAs then share the SM).
    const uint32_t lists = kLists * static_cast<uint32_t>(q.entries) * 12, share = kSmemPerSm / kPerSm - kReservedSmem;
    const uint32_t chunks =
        std::min(kMaxChunks, std::max(kMinChunks, share > lists ? (share - lists) / kChunkBytes : 0u));
    uint32_t cluster = 1;
    // A segment much longer than the ring comes from L2 a second time for the
    // most part: past 1.5 rings a row is shared by more CTAs (8192 x 131072
    // bf16 with gradient: 956 us by one CTA, 826 by two; 4096 x 65536, 1.3
    // rings: 208 by one, 241 by two).
    while (MODE == kTrain && cluster < kMaxCluster && rowBytes / cluster * 2 > chunks * kChunkBytes * 3ull) cluster *= 2;
    // Few rows: spread each over more SMs while a segment keeps 4 KB.
    while (cluster < kMaxCluster && q.rows * cluster * 2 <= static_cast<uint64_t>(smCount) * 2 &&
           rowBytes / (cluster * 2) >= 4096)
        cluster *= 2;
    Params p{};
    p.rows = q.rows;
    p.vocab = q.vocab;
    p.ldLogits = q.ldLogits;
    p.ldGrad = q.ldGrad;
    p.logits = q.logits;
    p.ids = q.teacherIds;
    p.teacher = q.teacherLogits;
    p.teacherBf16 = q.teacherBf16 ? 1u : 0u;
    p.entries = static_cast<uint32_t>(q.entries);
    p.cluster = cluster;
    p.scale = q.scale;
    p.loss = q.loss;
    p.lse = q.lse;
    p.gradLoss = q.gradLoss;
    p.grad = q.gradLogits;
    p.status = status;
    p.spins = waitSpins();
    p.chunks = chunks;
    const uint32_t smemBytes = p.chunks * kChunkBytes + lists;
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    uint32_t resident = 0;
    e = residentClusters(kernel, kThreads, cluster, smemBytes, device, resident);
    if (e != cudaSuccess) return e;
    const uint32_t grid = static_cast<uint32_t>(std::min<uint64_t>(q.rows, resident)) * cluster;
    cudaLaunchAttribute attribute;
    const cudaLaunchConfig_t config = configFor(grid, kThreads, smemBytes, cluster, attribute, stream);
    return cudaLaunchKernelEx(&config, kernel, p);
}

// Rows within one chunk of the large CTAs go to small ones, six to an SM.
constexpr uint64_t kShortRow = 16 * 1024;

template <int MODE>
cudaError_t launchMode(const Problem& q, int smCount, uint32_t* status, cudaStream_t stream) {
    if (q.rows == 0) return cudaSuccess;
    const bool small = q.vocab * (q.bf16 ? 2 : 4) <= kShortRow;
    if (q.bf16)
        return small ? launchTyped<__nv_bfloat16, MODE, 4>(q, smCount, status, stream)
                     : launchTyped<__nv_bfloat16, MODE, 8>(q, smCount, status, stream);
    return small ? launchTyped<float, MODE, 4>(q, smCount, status, stream)
                 : launchTyped<float, MODE, 8>(q, smCount, status, stream);
}

} // namespace

cudaError_t forward(const Problem& q, int smCount, std::uint32_t* status, cudaStream_t stream) {
    return q.gradLogits ? launchMode<kTrain>(q, smCount, status, stream) : launchMode<kScore>(q, smCount, status, stream);
}

cudaError_t backward(const Problem& q, int smCount, std::uint32_t* status, cudaStream_t stream) {
    return launchMode<kBackward>(q, smCount, status, stream);
}

} // namespace thb::distill
