// What chunk.cu and chunk_tc.cu know of each other.
#pragma once

#include <cuda.h>

#include "cache_mma.cuh"
#include "pkv_internal.h"

namespace pkv {

// A cache as (channel, head, token of all pages); boxes of `channels` codes of one head
// and `tokens` tokens, plain or swizzled within rows of 64 or 128 bytes.  Channels past
// head_dim load as zero.
bool cache_map(CUtensorMap* map, const int8_t* cache, const ChunkArgs& a, int channels, int tokens,
               bool swizzle);

constexpr int kChunkTcCtas = 148;  // one per SM

// Whether the tensor-memory kernel takes this call's shapes.
bool chunk_tc_takes(const ChunkArgs& a);
// Its plan, from one with the call's sizes.
PlanArgs chunk_tc_plan(const PlanArgs& base);
size_t chunk_tc_workspace_size(const ChunkArgs& a);
// The units of a plan in head and seq; with zero_rows also rows outside all sequences.
int launch_chunk_tc(const ChunkArgs& a, PlanHead* head, PlanSeq* seq, uint8_t* ws, bool zero_rows,
                    cudaStream_t stream);

}  // namespace pkv
