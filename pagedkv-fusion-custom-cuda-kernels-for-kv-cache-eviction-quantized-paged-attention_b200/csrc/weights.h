// What weights.cu and weights_tc.cu know of each other.
#pragma once

#include "cache_mma.cuh"
#include "pkv_internal.h"

namespace pkv {

// Weights meet as integers of 2^-38, so that the order of their arrival changes nothing;
// 2^25 of weight before bit 63, which says that a sum was not finite.
constexpr float kWeightUnit = 274877906944.0f;
constexpr unsigned long long kNotFinite = 1ull << 63;

__device__ __forceinline__ void add_weight(unsigned long long* sum, float v) {
  if (v < 33554432.0f) {
    const unsigned long long u = __float2ull_rn(v * kWeightUnit);
    if (u != 0) atomicAdd(sum, u);
  } else {
    atomicOr(sum, kNotFinite);  // NaN, or lse of other tokens
  }
}

int launch_gather_tc(const ChunkArgs& a, const float* lse, PlanHead* head, PlanSeq* seq,
                     unsigned long long* sums, cudaStream_t stream);

}  // namespace pkv
