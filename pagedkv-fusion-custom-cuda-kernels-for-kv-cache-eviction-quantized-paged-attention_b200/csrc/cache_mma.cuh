// Pieces of the kernels in which a warp multiplies INT8 pages by mma.sync: the codes go
// from shared memory to fp16 fragments in registers, where they are exact, and rows of
// queries are fp16 with a power of two apart (two numbers, 22 bits, for fp32 queries).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "pkv_common.cuh"
#include "pkv_internal.h"

namespace pkv {

constexpr float kLog2e = 1.4426950408889634f;

// A kernel that may be launched while the one in front of it in the stream still runs
// (programmatic dependent launch): it sets up what needs nothing of that one, and waits
// for its end, and so for everything earlier, in behind_the_last().  Every thread of every
// kernel of such a row calls that before it reads or writes global memory, and the kernels
// in front let the next be launched at their start.  (A call is a row of two to six kernels of
// 2 us and more.)
__device__ __forceinline__ void behind_the_last() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void launch_the_next() { asm volatile("griddepcontrol.launch_dependents;"); }

template <typename... Params, typename... Args>
inline void launch_behind(void (*kernel)(Params...), dim3 grid, int threads, size_t shared,
                          cudaStream_t stream, Args... args) {
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3((unsigned)threads);
  config.dynamicSmemBytes = shared;
  config.stream = stream;
  config.attrs = &attr;
  config.numAttrs = 1;
  cudaLaunchKernelEx(&config, kernel, Params(args)...);  // (errors: cudaGetLastError, as after <<<>>>)
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Asynchronous copies of 16 or 4 bytes of global memory to shared memory, or zeros.
__device__ __forceinline__ void copy16_if(bool on, uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(on ? 16u : 0u)
               : "memory");
}
__device__ __forceinline__ void copy4_if(bool on, uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src),
               "r"(on ? 4u : 0u)
               : "memory");
}
__device__ __forceinline__ void copies_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Four INT8 codes (little-endian) as two words of fp16 pairs, exact: byte + 128
// in the low mantissa bits of 1024, minus 1152.
__device__ __forceinline__ uint2 codes_to_half(uint32_t w) {
  const uint32_t u = w ^ 0x80808080u;
  const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
  const __half2 bias = __float2half2_rn(1152.0f);
  const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), bias);
  const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), bias);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
}

__device__ __forceinline__ uint32_t word_of(__half2 h) {
  return *reinterpret_cast<const uint32_t*>(&h);
}

// d += a b, 16 x 8 x 16, fp16 with fp32 sums.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint4 a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }

// Four consecutive values, 8- (16-bit types) or 16-byte aligned.
template <typename T>
__device__ __forceinline__ float4 load4(const T* p) {
  if constexpr (sizeof(T) == 4) {
    return *reinterpret_cast<const float4*>(p);
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    const T* v = reinterpret_cast<const T*>(&w);
    return make_float4(widen(v[0]), widen(v[1]), widen(v[2]), widen(v[3]));
  }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, float4 v) {  // (aligned as above)
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = v;
  } else if constexpr (std::is_same<T, __half>::value) {
    const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(p) = make_uint2(word_of(a), word_of(b));
  } else {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a),
                                              *reinterpret_cast<const uint32_t*>(&b));
  }
}

// The power of two that takes a row of largest magnitude `big` to [2^10, 2^11), as
// its exponent; 0 for rows that are zero or not finite.
__device__ __forceinline__ int row_exponent(float big) {
  int e = 137 - (int)(__float_as_uint(big) >> 23);
  if (big == 0.0f || !(big <= 3.402823466e38f)) e = 0;
  return min(e, 126);
}
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }

// Codes as they stand in a word, plus 128, as fp16 pairs of 2^-24 times that: a byte in the
// low bits of fp16 is a subnormal number, which the tensor cores multiply exactly.
// (3 instructions a word instead of 5; the sum of 128 q is taken off beforehand.)
__device__ __forceinline__ uint2 codes_plus_128(uint32_t w) {
  const uint32_t u = w ^ 0x80808080u;
  return make_uint2(__byte_perm(u, 0, 0x4140), __byte_perm(u, 0, 0x4342));
}

// Two 8 x 8 matrices' worth of 16-bit values turned around: lane (g, t) has row g, columns
// 2 t and 2 t + 1 of the transposed one.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}

// `count` rows of queries (a multiple of 8) in shared memory in the order in which lanes
// read mma operands: [8 rows][half][DP / 16][lane] of 8 bytes.  Called by `warps` warps,
// each for some rows; lane = 4 channels.  A k step of 16 stands for channels
// p * 64 + t * 16 + w * 4 + 0..3 of lane t (of 4), step p * 4 + w, as the codes are read:
// 16 bytes a lane.  row(r) is the row's first channel or null; factor[r] becomes what its
// products have to be multiplied by, start[r] what their sums start from where codes come
// as codes_plus_128.
template <typename T, int DP, int HALVES, typename Row>
__device__ __forceinline__ void stage_queries(uint2* frag, float* factor, float* start, int dim,
                                              int count, int warp, int warps, Row row) {
  const int lane = threadIdx.x & 31;
  for (int r = warp; r < count; r += warps) {
    const T* from = row(r);
    constexpr int kParts = (DP + 127) / 128;
    float4 v[kParts];
    float big = 0.0f;
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const int c = i * 128 + lane * 4;
      v[i] = from != nullptr && c < dim ? load4(from + c) : make_float4(0, 0, 0, 0);
      big = fmaxf(big, fmaxf(fmaxf(fabsf(v[i].x), fabsf(v[i].y)), fmaxf(fabsf(v[i].z), fabsf(v[i].w))));
    }
    float up = 1.0f, down = 1.0f;
    if constexpr (!std::is_same<T, __half>::value) {
      big = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(big)));
      const int e = row_exponent(big);
      up = power_of_two(e);
      down = power_of_two(-e);
    }
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const int c = i * 128 + lane * 4;
      if (c >= DP) continue;
      const float f[4] = {v[i].x * up, v[i].y * up, v[i].z * up, v[i].w * up};
      const __half2 h0 = __floats2half2_rn(f[0], f[1]), h1 = __floats2half2_rn(f[2], f[3]);
      uint2* to = &frag[(r >> 3) * (HALVES * DP / 16 * 32) + (c / 64 * 4 + c % 16 / 4) * 32 +
                        (r & 7) * 4 + c % 64 / 16];
      *to = make_uint2(word_of(h0), word_of(h1));
      const float2 b0 = __half22float2(h0), b1 = __half22float2(h1);
      sum += (b0.x + b0.y) + (b1.x + b1.y);
      if constexpr (HALVES == 2) {
        const __half2 l0 = __floats2half2_rn(f[0] - b0.x, f[1] - b0.y);
        const __half2 l1 = __floats2half2_rn(f[2] - b1.x, f[3] - b1.y);
        to[DP / 16 * 32] = make_uint2(word_of(l0), word_of(l1));
        const float2 c0 = __half22float2(l0), c1 = __half22float2(l1);
        sum += (c0.x + c0.y) + (c1.x + c1.y);
      }
    }
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    if (lane == 0) {
      factor[r] = down;
      start[r] = sum * -7.62939453125e-6f;  // 128 / 2^24
    }
  }
}

// One row of queries in the four lanes t of a lane group g, as operands of 8 columns:
// channels p * 64 + t * 16 + w * 4 + 0..3 for step p * 4 + w.  First the loads: `from` is
// row g's first channel or null.
template <typename T>
using Raw4 = std::conditional_t<sizeof(T) == 4, uint4, uint2>;
template <typename T, int DP>
__device__ __forceinline__ void load_queries(const T* from, int dim, Raw4<T> (&raw)[DP / 16]) {
  const int t = threadIdx.x & 3;
#pragma unroll
  for (int p = 0; p < DP / 64; ++p) {
    const int c = p * 64 + t * 16;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      raw[p * 4 + w] = Raw4<T>{};
      if (from != nullptr && c < dim)
        raw[p * 4 + w] = *reinterpret_cast<const Raw4<T>*>(from + c + w * 4);
    }
  }
}
// Then the operands.  factor and start, as above, are those of rows 2 t and 2 t + 1.
template <typename T, int DP, int HALVES>
__device__ __forceinline__ void split_queries(const Raw4<T> (&raw)[DP / 16], uint2 (&frag)[HALVES][DP / 16],
                                              float (&factor)[2], float (&start)[2]) {
  const int t = threadIdx.x & 3;
  float4 v[DP / 16];
  float big = 0.0f;
#pragma unroll
  for (int k = 0; k < DP / 16; ++k) v[k] = load4(reinterpret_cast<const T*>(&raw[k]));
#pragma unroll
  for (int k = 0; k < DP / 16; ++k)
    big = fmaxf(big, fmaxf(fmaxf(fabsf(v[k].x), fabsf(v[k].y)), fmaxf(fabsf(v[k].z), fabsf(v[k].w))));
  float up = 1.0f, down = 1.0f;
  if constexpr (!std::is_same<T, __half>::value) {
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
    const int e = row_exponent(big);
    up = power_of_two(e);
    down = power_of_two(-e);
  }
  float sum = 0.0f;
#pragma unroll
  for (int k = 0; k < DP / 16; ++k) {
    const float f[4] = {v[k].x * up, v[k].y * up, v[k].z * up, v[k].w * up};
    const __half2 h0 = __floats2half2_rn(f[0], f[1]), h1 = __floats2half2_rn(f[2], f[3]);
    frag[0][k] = make_uint2(word_of(h0), word_of(h1));
    const float2 b0 = __half22float2(h0), b1 = __half22float2(h1);
    sum += (b0.x + b0.y) + (b1.x + b1.y);
    if constexpr (HALVES == 2) {
      const __half2 l0 = __floats2half2_rn(f[0] - b0.x, f[1] - b0.y);
      const __half2 l1 = __floats2half2_rn(f[2] - b1.x, f[3] - b1.y);
      frag[HALVES - 1][k] = make_uint2(word_of(l0), word_of(l1));
      const float2 c0 = __half22float2(l0), c1 = __half22float2(l1);
      sum += (c0.x + c0.y) + (c1.x + c1.y);
    }
  }
  sum += __shfl_xor_sync(0xffffffffu, sum, 1);
  sum += __shfl_xor_sync(0xffffffffu, sum, 2);
  sum *= -7.62939453125e-6f;  // 128 / 2^24
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    factor[e] = __shfl_sync(0xffffffffu, down, 8 * t + 4 * e);
    start[e] = __shfl_sync(0xffffffffu, sum, 8 * t + 4 * e);
  }
}

// 16-byte piece of a key's row of DP codes in shared memory, so that the lanes that
// read 8 keys' pieces at once (K: pieces t, keys g; V: pieces g, keys 2 t) meet no bank
// twice.
template <int DP>
__device__ __forceinline__ int piece_at(int key, int piece) {
  if constexpr (DP >= 128)
    return (piece & ~7) | ((piece & 7) ^ ((key & 6) ^ ((key & 1) << 2)));
  else
    return piece ^ ((key >> 1) & 3);
}

// ---------------------------------------------------------------------------
// The plan of a call over packed new tokens and their sequences' pages
// ---------------------------------------------------------------------------

constexpr float kCodeUnit = 16777216.0f;  // 2^24: what codes_plus_128 divides by

// A sequence's work: its query rows of a KV head in blocks of `rows`, a unit each, times
// its keys in steps of `step`, one at least, behind `over` places that stand for what a
// unit costs however short.  Units follow each other sequence by sequence, and in a
// sequence block by block, the KV heads of a block next to one another.  A plan has all
// sequences, or those of few rows of a KV head (at most few_rows, or so short that blocks
// of 8 rows have no more than few_steps steps of 16 keys), or the others.
//
// With `workers`, each of which takes a share of the places, the plan says how large it is:
// equal shares of all places (at least `least`), in which units follow each other and are
// cut anywhere; or, where the call is so small that kPartSteps or twice as many steps a worker
// do, parts of a unit of so many, a worker each (`over` is 0 then).
enum PlanWhich { kPlanAll = 0, kPlanFew = 1, kPlanMany = 2 };
constexpr int kPartSteps = 4;
struct PlanSeq {
  int64_t first;  // places in front of the sequence's
  int q0, lq;     // its rows in the packed queries
  int len;        // its cached tokens, the new ones among them
  int steps;      // of a unit
  int pitch;      // places of a unit
  int unused;
};

struct PlanHead {
  int64_t places;      // in all
  int q_begin, q_end;  // rows of all sequences
  int64_t share;       // places of a worker
  int over;            // places in front of a unit's steps
  int unused;
};

struct PlanArgs {
  const int32_t* cu;
  const int32_t* lens;
  int seqs, total_q;
  int group, kv_heads, block_size, width;
  int rows, step, over;
  int workers, least;
  int which, few_rows, few_steps;
  PlanHead* head;
  PlanSeq* seq;   // [seqs]
  int* counters;  // [counts], zeroed
  int counts;
};

// One or two plans of a call, the second for another kernel.
int launch_plan(const PlanArgs& a, const PlanArgs* second, const ZeroArgs& zero, int* err,
                cudaStream_t stream);

// The sequence of a place; one warp, a search of 32 at a time.
__device__ __forceinline__ int plan_find(const PlanSeq* seq, int seqs, int64_t place) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = seqs;  // the last sequence of [lo, lo + n) whose first place is <= this
  while (n > 1) {
    const int stride = (n + 31) / 32;
    const bool below = lane * stride < n && seq[lo + lane * stride].first <= place;
    const int last = 31 - __clz(__ballot_sync(0xffffffffu, below));
    lo += last * stride;
    n = min(stride, n - last * stride);
  }
  return lo;
}

}  // namespace pkv
