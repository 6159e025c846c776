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

// Where launch_chunk left the sequences' rows and lengths (of calls without a V cache).
const PlanSeq* chunk_plan(const ChunkArgs& a, void* workspace);

// A unit that was cut, for the kernel that joins its parts.
struct CutUnit {
  int parts;  // 0: there is none
  int rows, kvh, block, q0;
  int first;  // of the workers that have parts
};

constexpr int kTileUnitRows = 256;
constexpr int kTileKeys = 128;
constexpr int kTileOver = 3;   // tiles that a unit's start and end cost
constexpr int kTileLeast = 6;  // places of a CTA's share

// Work of kernels whose units are 256 query rows of a KV head, in tiles of 128 keys:
// each of `ctas` CTAs has the same share of the plan's places.
struct TileWork {
  const PlanHead* head;
  const PlanSeq* seq;
  int seqs, group, kv_heads, ctas;
};

__device__ __forceinline__ int64_t tile_share(const TileWork& p) {
  return max((p.head->places + p.ctas - 1) / p.ctas, (int64_t)kTileLeast);
}

// A unit, and the part of it that a CTA has.
struct TileUnit {
  PlanSeq seq;
  int s, kvh, block, rows;
  int64_t at;          // first place
  int cta0, parts;
  int tile0, n;        // the CTA's tiles of it
  int tiles[2];        // of each row tile, from tile0 on
  bool dual;           // the row tiles share the rows, and the tiles in turns

  __device__ __forceinline__ void find(const TileWork& p, int64_t place, int64_t share) {
    int unit;
    for (;;) {  // (sequences that are not this kernel's have no places)
      seq = p.seq[s];
      unit = (int)((place - seq.first) / (seq.steps + kTileOver));
      const int64_t next = s + 1 < p.seqs ? p.seq[s + 1].first : p.head->places;
      if (place < next) break;
      ++s;
    }
    at = seq.first + (int64_t)unit * (seq.steps + kTileOver);
    kvh = unit % p.kv_heads;
    block = unit / p.kv_heads;
    rows = (int)min((int64_t)kTileUnitRows, seq.lq * (int64_t)p.group - (int64_t)block * kTileUnitRows);
    cta0 = (int)((at + kTileOver) / share);
    parts = (int)((at + kTileOver + seq.steps - 1) / share) - cta0 + 1;
    dual = rows <= (kTileUnitRows / 2) && seq.steps > 1;
  }
  __device__ __forceinline__ void cut(const TileWork& p, int64_t now, int64_t stop) {
    tile0 = (int)max(now - at - kTileOver, (int64_t)0);
    const int end = (int)max(min((int64_t)seq.steps, stop - at - kTileOver), (int64_t)tile0);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int last = min((x + 1) * (kTileUnitRows / 2), rows) - 1;
      const int keys = last >= x * (kTileUnitRows / 2) || dual ? max(limit(p, min(last, rows - 1)), 0) : 0;
      tiles[x] = max(min((keys + kTileKeys - 1) / kTileKeys, end) - tile0, 0);
    }
    n = max(tiles[0], tiles[1]);
  }
  __device__ __forceinline__ bool empty(int64_t stop) const { return stop <= at + kTileOver; }
  // the keys that row r sees
  __device__ __forceinline__ int limit(const TileWork& p, int r) const {
    return r < rows ? min((int)((uint32_t)(block * kTileUnitRows + r) / (uint32_t)p.group) + 1 + seq.len - seq.lq,
                          seq.len)
                    : 0;
  }
  __device__ __forceinline__ int64_t token(const TileWork& p, int r, int* head) const {
    const uint32_t i = block * kTileUnitRows + r;  // (a call has less than 2^31 rows)
    const uint32_t tok = i / (uint32_t)p.group;
    *head = kvh * p.group + (int)(i - tok * (uint32_t)p.group);
    return seq.q0 + tok;
  }
};

__device__ __forceinline__ float load_if(bool on, const float* p) {
  float v;
  asm volatile(
      "{\n\t.reg .pred on;\n\tsetp.ne.u32 on, %2, 0;\n\tmov.f32 %0, 0f00000000;\n\t"
      "@on ld.global.nc.f32 %0, [%1];\n\t}"
      : "=&f"(v)
      : "l"(p), "r"((uint32_t)on));
  return v;
}

// Query rows of a unit, as tcgen05 operands in shared memory: boxes of 64 fp16 channels,
// rows of 128 bytes in the 128-byte swizzle, BOX bytes from one to the next; for fp32
// queries boxes of hi, then of lo.  They arrive as they are, a warp its 32 rows, all on
// their way at once (a quarter of them at a time through registers took 18,000 clocks of
// a call's first unit, 5 us each), in the places that the row's own thread then writes:
// of 4-byte channels, 32 a box, those 32 i .. are box i / 2, or (odd i) DP / 64 further.
// `mine` is the lane's row, count how many of the warp's there are; the others, and
// channels behind dim, are zero.
template <typename T, int DP, int BOX>
__device__ __forceinline__ void copy_query_rows(uint32_t tile, int row0, const T* any, const T* mine,
                                                int count, int dim) {
  constexpr int kPieces = DP * (int)sizeof(T) / 16;  // of 16 bytes, of a row
  constexpr int kEach = 32 / kPieces;                // rows at once
  const int lane = threadIdx.x & 31, piece = lane % kPieces;
  const int c = piece * (16 / (int)sizeof(T)), box = piece / 8;
  const uint32_t to = tile + (sizeof(T) == 4 ? box / 2 + box % 2 * (DP / 64) : box) * BOX;
#pragma unroll 4
  for (int i = 0; i < kPieces; ++i) {
    const int r = i * kEach + lane / kPieces;
    const T* from = reinterpret_cast<const T*>(
        __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), r));
    const bool on = r < count && c < dim;
    copy16_if(on, to + sw128_offset(row0 + r, piece % 8 * 16), on ? from + c : any);
  }
  copies_commit();
  copies_wait<0>();
  __syncwarp();
}
// The largest magnitude of a row's (infinity or NaN where there is one); nothing for fp16.
template <typename T, int DP, int BOX>
__device__ __forceinline__ float query_row_most(const uint8_t* tile, int row) {
  uint32_t most = 0;
#pragma unroll 4
  for (int i = 0; i < DP * (int)sizeof(T) / 16; ++i) {
    const uint4 w = *reinterpret_cast<const uint4*>(tile + i / 8 * BOX + sw128_offset(row, i % 8 * 16));
    if constexpr (sizeof(T) == 4) {
      constexpr uint32_t kAbs = 0x7fffffffu;
      most = max(most, max(max(w.x & kAbs, w.y & kAbs), max(w.z & kAbs, w.w & kAbs)));
    } else {
      constexpr uint32_t kAbs = 0x7fff7fffu;
      most = __vmaxu2(most, __vmaxu2(__vmaxu2(w.x & kAbs, w.y & kAbs), __vmaxu2(w.z & kAbs, w.w & kAbs)));
    }
  }
  return __uint_as_float(sizeof(T) == 4 ? most : max(most << 16, most & 0xffff0000u));
}
// A row times the power of two `up`, in place (fp16 is as it is).
template <typename T, int DP, int BOX>
__device__ __forceinline__ void split_query_row(uint8_t* tile, int row, float up) {
  const auto at = [&](int box, int piece) {
    return reinterpret_cast<uint4*>(tile + box * BOX + sw128_offset(row, piece * 16));
  };
#pragma unroll 1
  for (int b = 0; b < DP / 64; ++b) {
    if constexpr (sizeof(T) == 4) {
      uint4 w[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = *at(b + i / 8 * (DP / 64), i % 8);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint32_t h[4], l[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint4 x = w[2 * i + e / 2];
          const float f0 = __uint_as_float(e & 1 ? x.z : x.x) * up, f1 = __uint_as_float(e & 1 ? x.w : x.y) * up;
          const __half2 a = __floats2half2_rn(f0, f1);
          const float2 back = __half22float2(a);
          h[e] = word_of(a);
          l[e] = word_of(__floats2half2_rn(f0 - back.x, f1 - back.y));
        }
        *at(b, i) = make_uint4(h[0], h[1], h[2], h[3]);
        *at(b + DP / 64, i) = make_uint4(l[0], l[1], l[2], l[3]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint4 x = *at(b, i);
        const auto scaled = [&](uint32_t v) {
          return word_of(__floats2half2_rn(__uint_as_float(v << 16) * up, __uint_as_float(v & 0xffff0000u) * up));
        };
        *at(b, i) = make_uint4(scaled(x.x), scaled(x.y), scaled(x.z), scaled(x.w));
      }
    }
  }
}

constexpr int kChunkTcCtas = 148;  // one per SM

// Whether the tensor-memory kernel takes this call's shapes.
bool chunk_tc_takes(const ChunkArgs& a);
// Its plan, from one with the call's sizes.
PlanArgs chunk_tc_plan(const PlanArgs& base);
// CTAs of a launch: no more than have their least share of the longest that the batch can
// be.
int chunk_tc_ctas(const ChunkArgs& a);
size_t chunk_tc_workspace_size(const ChunkArgs& a);
// The units of a plan in head and seq; with zero_rows also rows outside all sequences.
int launch_chunk_tc(const ChunkArgs& a, PlanHead* head, PlanSeq* seq, uint8_t* ws, bool zero_rows,
                    cudaStream_t stream);

}  // namespace pkv
