// What the kernels of the linear losses share.
#pragma once

#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "exponential.cuh"

namespace thb::linear_loss {

constexpr uint32_t kNoEntry = 0x7fffffffu;  // sorts behind every vocabulary entry

enum RowState : uint8_t { kDead = 0, kLive = 1, kBad = 2 };  // kBad: a target outside the vocabulary

// Of rows with labels; a teacher's lists come with their states.
__device__ __forceinline__ uint8_t labelState(int64_t label, int64_t ignore, uint64_t vocab) {
    if (label == ignore) return kDead;
    return label >= 0 && label < static_cast<int64_t>(vocab) ? kLive : kBad;
}

__device__ __forceinline__ void gridDependencyWait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void gridDependencyLaunch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// (maximum, sum of 2^((z - maximum) c)) of two parts of a row, joined. The
// maxima are logits as they are, since a scaled one, rounded, is off by more
// than an exponential holds once logits pass 2^30.
__device__ __forceinline__ void fold(float& top, float& sum, float otherTop, float otherSum, float c) {
    const float high = fmaxf(top, otherTop);
    const float from = high == -INFINITY ? 0.0f : high;
    sum = sum * pow2((top - from) * c) + otherSum * pow2((otherTop - from) * c);
    top = high;
}

// log-sum-exp of a row and its loss, sum q log q - sum q z + lse. The scaled
// maximum is rounded by itself, as the backward pass rounds the scaled logits
// that it takes lse from: far from 0 the two are then the same value.
__device__ __forceinline__ void closeRow(uint64_t row, float top, float sum, float scale, float target, const float* entropy,
                                         float* loss, float* lse) {
    const float total = __fadd_rn(__fmul_rn(top, scale), logf(sum));
    lse[row] = total;
    loss[row] = (entropy ? entropy[row] : 0.0f) + (total - target);
}

} // namespace thb::linear_loss
