// What weights.cu and weights_tc.cu know of each other.
#pragma once

#include "cache_mma.cuh"
#include "pkv_internal.h"

namespace pkv {

// Weights meet as integers of 2^-37, so that the order of their arrival changes nothing;
// the 2^25 rows that a call may have give a token up to 2^62, with the roundings of their
// exponentials, and bit 63 says that a sum was not finite.
constexpr float kWeightUnit = 137438953472.0f;
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
