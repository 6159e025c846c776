// Decode attention for a batch that shares a prefix, over the INT8 paged
// cache: the prefix's pages are read once for the whole batch instead of once
// per sequence.
//
//   prefix_kernel   (KV head, 256 query rows, part of the prefix): partial
//                   (acc, m, l) of every row over that part;
//   the decode split kernels (decode.cu) on the sequences' own pages, asked
//                   for partials;
//   join_kernel     one warp per (sequence, query head): all partials of the
//                   row, joined by their maxima.
//
// A query row is a (sequence, query head of the group) pair: with S sequences
// and G heads per KV head, S G rows meet every K and V tile, so the products
// are matrix products and run on tcgen05 kind::f16.  fp32 accuracy comes from
// splitting the fp32 operands: INT8 codes are exact in fp16; a query row,
// scaled by a power of two, is hi + lo in fp16 (22 bits), and so is p * v_scale.
// Both halves accumulate into the same fp32 accumulator, so S and O are one
// 128-column tile each.  (Three signed byte digits on kind::i8, as the decode
// kernel for single sequences has them, would cost 3/4 of the tensor time but
// three accumulators per product -- more tensor memory than there is -- and
// about twice the instructions per score, which are what bounds this kernel.)
//
// Roles: two softmax warpgroups (one 128-row tile each, one thread per row),
// four converting warps (global INT8 pages -> fp16 tiles in shared memory, and
// the pages' scales; the codes come by cp.async into the half of their stage that
// is converted last), one MMA warp per row tile; two warps idle, so that the
// registers split evenly.  The row tiles take turns on the tensor cores as in
// prefill.cu.  Where a KV head has at most 128 rows (SHARED), both warpgroups work
// on the one row tile, and the free tensor memory holds the next tile's scores.
//
// What bounds it: 32,768 tokens for 64 sequences of 32 query heads (8 KV heads,
// head_dim 128) are 69 GFLOP with both halves (41 us at the cuBLAS rate) and 67 MB
// (10 us); the kernel takes 83 us, its tensor pipe 43% and its issue slots 46% busy.
// A row tile's step is about 2,400 clocks of products (S reads both operands from
// shared memory) and 4,900 of softmax, of which the other row tile hides half; 144
// CTAs of 14 or 15 tiles also pay for the query split, the first loads and the
// partials' stores.  With one row tile a step was a chain that nothing overlapped:
// 16,384 tokens, 20 rows of each of 40 KV heads took 159 us with one warpgroup,
// 144 us with two, and take 122 us with two buffers of scores.
// (Loads into registers cost the converting warps 2,000 clocks for 8 loads a
// thread: with 200 KB of shared memory in use the L1 cache holds few misses.)
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "pkv_common.cuh"
#include "pkv_internal.h"

namespace pkv {
namespace {

constexpr int kRows = 128;
constexpr int kKeys = 128;
constexpr int kPrefixThreads = 16 * 32;
constexpr int kConvWarp = 8, kMmaWarp = 12, kIdleWarp = 14;
constexpr int kEarly = 4;         // MMAs left of a step when the turn is passed on
constexpr float kLog2e = 1.4426950408889634f;
// A row's maximum moves when a tile exceeds it by more than 2^kLazy, and p is
// kept times 2^kPShift: at most 2^15 in fp16.  The low half has fp16's smallest
// step, 2^-24, so p * v_scale is kept to 2^-25 - kPShift of the row's largest p
// times the largest V scale.
constexpr float kLazy = 2.0f;
constexpr float kPShift = 13.0f;

template <int DP, bool SHARED>
struct PrefixCfg {
  static constexpr int kChunks = DP / 64;
  static constexpr int kTileBytes = kKeys * DP * 2;
  static constexpr int kStages = DP == 128 ? (SHARED ? 4 : 3) : 6;
  // Scales of a tile are reused by tile j + kSlots.  They are written after the
  // copies of tile j were started, which waits for stages that P V (j - 2) frees (3
  // or 4 stages), or a product behind P V (j - 4) (6 stages).
  static constexpr int kSlots = DP == 128 ? 2 : 4;
  static constexpr int kOffQ = 0;  // [row tile][hi, lo]
  static constexpr int kOffXch = 2 * kTileBytes;  // SHARED: values exchanged within a row
  static constexpr int kOffKV = SHARED ? kOffXch + 4096 : 4 * kTileBytes;
  static constexpr int kOffScale = kOffKV + kStages * kTileBytes;  // [slot][k, v][128]
  static constexpr int kOffMask = kOffScale + kSlots * 2 * kKeys * 4;
  static constexpr int kOffBar = kOffMask + kSlots * 16;
  static constexpr int kBars = 2 * kStages + kSlots + 10 + 3;
  static constexpr int kOffMisc = kOffBar + kBars * 8;
  static constexpr int kSmemBytes = kOffMisc + 32;
  static constexpr int kOCol = 256;
  static_assert(kSmemBytes <= 227 * 1024, "shared memory");
};

// The tensor cores cut off the bits that an fp32 sum cannot hold, so a sum of one
// sign shrinks by 8e-7 in a tile (16 products; 6.4e-6 in 8 tiles), one of mixed
// signs by about a third of that.  Every few tiles O is therefore added to a sum of
// its own, rounded to nearest, and started anew.  Where tensor memory has columns
// left (head_dim up to 64, or one row tile) the sum is there and takes O every 2
// tiles: V of one sign is then off by 1.6e-6 of the result in the mean.  Else it is in
// global memory and takes O every 5: V of one sign is off by 4.1e-6, of mixed
// signs by 1.9e-6, and 32,768 tokens for 64 sequences, 32 / 8 heads take 115 us a call.
// Every 8 were 6.3e-6, 2.6e-6 and 112 us, every 4 3.2e-6, 1.6e-6 and 118 us.
constexpr int kFlushNear = 2, kFlushFar = 5;

struct PrefixParams {
  const float* q;
  const int8_t* k_cache;
  const float* k_scale;
  const int8_t* v_cache;
  const float* v_scale;
  const int32_t* table;       // [width]
  const int32_t* prefix_len;  // [1]
  float* acc;                 // [splits][num_seqs * heads][dim]
  float2* ml;                 // [splits][num_seqs * heads]
  float4* sums;               // per CTA and row tile: [DP / 4][128 rows], O of earlier tiles
  int64_t num_blocks;
  int num_seqs, heads, kv_heads, group, dim, bs, width, splits;
  float qk_scale;  // sm_scale log2e
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16 bytes of global memory to shared memory, or zeros.
__device__ __forceinline__ void copy16_if(bool on, uint32_t dst, const int8_t* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(on ? 16u : 0u)
               : "memory");
}
// A float of read-only memory, or zero.  (In assembly: of a load behind a branch the
// compiler takes the products in the branch too, and so waits for it there.)
__device__ __forceinline__ float load_if(bool on, const float* p) {
  float v;
  asm volatile(
      "{\n\t.reg .pred on;\n\tsetp.ne.u32 on, %2, 0;\n\tmov.f32 %0, 0f00000000;\n\t"
      "@on ld.global.nc.f32 %0, [%1];\n\t}"
      : "=&f"(v)
      : "l"(p), "r"((uint32_t)on));
  return v;
}

// Tokens of the prefix: the given length, at most what the table covers.
__device__ __forceinline__ int prefix_tokens(const int32_t* len, int width, int bs) {
  return min(max(*len, 0), width * bs);
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

// GROUPS: the pages hold a multiple of 16 tokens, so 16 columns of a tile share
// their scales and one load serves them; else every token has its own.
// SHARED: one row tile (at most 128 rows a KV head).  Both softmax groups then work
// on it, each on 64 of a tile's tokens and half of O's columns: a thread and the one
// 128 further have a row, and exchange its maximum by shared memory.
template <int DP, bool GROUPS, bool SHARED>
__global__ void __launch_bounds__(kPrefixThreads, 1)
    prefix_kernel(const PrefixParams p, int* err) {
  using C = PrefixCfg<DP, SHARED>;
  extern __shared__ __align__(1024) uint8_t smem[];  // no static shared memory: 1024-aligned
  float* s_scale = reinterpret_cast<float*>(smem + C::kOffScale);
  uint32_t* s_mask = reinterpret_cast<uint32_t*>(smem + C::kOffMask);
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* kv_empty = kv_full + C::kStages;
  uint64_t* sc_full = kv_empty + C::kStages;
  uint64_t* q_full = sc_full + C::kSlots;  // per row tile, as the next three
  uint64_t* s_full = q_full + 2;
  uint64_t* p_full = s_full + 2;  // [row tile][half of the tokens]
  uint64_t* o_full = p_full + 4;
  uint64_t* pv_done = o_full + 1;  // SHARED: every tile's P V
  uint64_t* mma_done = o_full + 2;
  uint64_t* turn = mma_done + 1;  // per row tile
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + C::kOffMisc);
  float* s_vmax = reinterpret_cast<float*>(smem + C::kOffMisc + 16);  // of each converting warp

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kvh = blockIdx.x % p.kv_heads, pair = blockIdx.x / p.kv_heads;
  const int split = blockIdx.y;
  const int rows = p.num_seqs * p.group;
  const int len = prefix_tokens(p.prefix_len, p.width, p.bs);
  if (blockIdx.x == 0 && split == 0 && tid == 0 && *p.prefix_len > len)
    record_error(err, kDevSeqTooLong);
  // this part's tokens: equal numbers of tiles
  const int tiles = (len + kKeys - 1) / kKeys;
  const int per_split = (tiles + p.splits - 1) / p.splits;
  const int tile0 = min(split * per_split, tiles);
  const int n = min(per_split, tiles - tile0);
  const bool two = !SHARED && pair * 256 + kRows < rows;  // the second row tile has rows
  const bool near = DP == 64 || !two;          // see kFlushNear
  const int flush = near ? kFlushNear : kFlushFar;

  if (tid == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&kv_full[i], 128);
      mbar_init(&kv_empty[i], two ? 2 : 1);  // the MMA warps at work
    }
    for (int i = 0; i < C::kSlots; ++i) mbar_init(&sc_full[i], 128);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], SHARED ? 256 : 128);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[2 * i], 128);
      mbar_init(&p_full[2 * i + 1], 128);
      mbar_init(&o_full[i], 1);
    }
    mbar_init(mma_done, 2);
    mbar_init(&turn[0], 1);
    mbar_init(&turn[1], 1);
    mbar_fence_init();
  }
  if (warp == kMmaWarp) tmem_alloc(s_tmem, 512);
  tmem_fence_before_sync();
  __syncthreads();
  tmem_fence_after_sync();
  const uint32_t tmem = *s_tmem;
  if (warp >= kConvWarp) {
  // 256 x 136 + 256 x 120 = 65,536 = 512 x 128, the registers at launch
  registers_down<120>();
  if (warp < kMmaWarp) {
    // ---- pages to fp16 tiles -----------------------------------------------------
    constexpr int kLanes = DP / 16;            // 16-byte pieces of a token row
    constexpr int kStep = 128 / kLanes;        // token rows per pass
    constexpr int kPass = kKeys / kStep;
    const int ct = tid - kConvWarp * 32;
    const int piece = ct % kLanes, row0 = ct / kLanes;
    const uint32_t row_bytes = (uint32_t)(p.kv_heads * p.dim);
    const bool in_dim = piece * 16 < p.dim;
    constexpr int kFar = C::kStages / 3;  // tiles that are on their way
    // With three stages the next K waits for V (j - 1)'s, and V (j) is not to wait
    // for that: both copies are started after both conversions.  With four, each
    // after its own.
    constexpr bool kBetween = C::kStages == 4;
    bool ok = true;
    // Cache rows of a tile's tokens, found a tile ahead by the warp's lanes (with
    // GROUPS lane l & 7 finds those of 16 tokens, else a lane finds 4) and handed
    // to the threads that read them by shuffle.
    constexpr int kFinds = GROUPS ? 1 : 4;
    constexpr uint32_t kNoRow = 0xffffffffu;  // no token, or a page outside the cache
    uint32_t at[kFinds];
    int entry[kFinds], rem[kFinds];  // of the next tile
    const int last_page = n > 0 ? (len - 1) / p.bs : 0;
    auto token = [&](int j, int u) {
      return (tile0 + j) * kKeys + (GROUPS ? (lane & 7) * 16 : u * 32 + lane);
    };
    auto look_up = [&](int j) {
#pragma unroll
      for (int u = 0; u < kFinds; ++u) {
        const int page = token(j, u) / p.bs;
        rem[u] = token(j, u) - page * p.bs;
        entry[u] = p.table[min(page, last_page)];  // past the end the last page again
      }
    };
    // scales of the thread's token, of the tile at hand and those on their way
    float ks[kFar] = {}, vs[kFar] = {};
    bool good[kFar] = {};
    auto resolve = [&](int j) {
      int phys;  // of the thread's own token
      if constexpr (GROUPS) {
        phys = __shfl_sync(0xffffffffu, entry[0], ct / 16);
      } else {
        phys = entry[0];
#pragma unroll
        for (int u = 1; u < kFinds; ++u)
          if (ct / 32 == u) phys = entry[u];
      }
      const bool counts = (tile0 + j) * kKeys + ct < len;
      const bool ok_page = counts && phys >= 0 && (int64_t)phys < p.num_blocks;
      if (counts && !ok_page) record_error(err, kDevBadBlockId);
      good[kFar - 1] = ok_page;
      ks[kFar - 1] = load_if(ok_page, p.k_scale + (int64_t)phys * p.kv_heads + kvh);
      vs[kFar - 1] = load_if(ok_page, p.v_scale + (int64_t)phys * p.kv_heads + kvh);
#pragma unroll
      for (int u = 0; u < kFinds; ++u) {
        const bool in = token(j, u) < len && entry[u] >= 0 && (int64_t)entry[u] < p.num_blocks;
        at[u] = in ? (uint32_t)entry[u] * p.bs + rem[u] : kNoRow;
      }
    };
    // Item i is tile i / 2, K or V.  Its codes are copied into the second half of its
    // stage, kFar tiles ahead; each thread converts what it copied.
    auto stage_of = [&](int i) { return smem + C::kOffKV + (i % C::kStages) * C::kTileBytes; };
    auto issue = [&](int j, int kind) {
      if (kFar == 2 && kind == 0)
        ks[0] = ks[kFar - 1], vs[0] = vs[kFar - 1], good[0] = good[kFar - 1];
      if (j < n) {
        if (kind == 0) {
          resolve(j);
          if (j + 1 < n) look_up(j + 1);
        }
        const int i = 2 * j + kind, st = i % C::kStages;
        if (ok && !mbar_wait_bounded(&kv_empty[st], ((uint32_t)(i / C::kStages) & 1u) ^ 1u, err)) {
          record_error(err, kDevWaitTimeout);
          ok = false;
        }
        const int8_t* base = (kind ? p.v_cache : p.k_cache) + (int64_t)kvh * p.dim + piece * 16;
        const uint32_t dst = smem_u32(stage_of(i)) + C::kTileBytes / 2 + ct * 16;
#pragma unroll
        for (int r = 0; r < kPass; ++r) {
          const int o = r * kStep;
          const uint32_t row =
              GROUPS ? __shfl_sync(0xffffffffu, at[0], o / 16 + row0 / 16)
                     : __shfl_sync(0xffffffffu, at[GROUPS ? 0 : o / 32], o % 32 + row0);
          const bool on = row != kNoRow && in_dim;
          // (rows past the length on its last page are read: any codes will do)
          const uint64_t from = (uint64_t)(on ? row + (GROUPS ? row0 % 16 : 0) : 0) * row_bytes;
          copy16_if(on, dst + r * 2048, base + from);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    float inv_vmax = 0.0f;
    if (n > 0) {
      look_up(0);
#pragma unroll
      for (int j = 0; j < kFar; ++j) {
        issue(j, 0);
        issue(j, 1);
      }
      // the largest V scale of this part: p * v_scale is kept relative to it
      const int first = tile0 * kKeys / p.bs;
      const int last = (min((tile0 + n) * kKeys, len) - 1) / p.bs;
      float v = 0.0f;
      for (int i = first + ct; i <= last; i += 128) {
        const int phys = p.table[i];
        if (phys >= 0 && (int64_t)phys < p.num_blocks)
          v = fmaxf(v, fabsf(p.v_scale[(int64_t)phys * p.kv_heads + kvh]));
      }
      v = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
      if (lane == 0) s_vmax[warp - kConvWarp] = v;
      named_barrier(1, 128);  // also seen by the softmax warps, through sc_full
      const float vmax = fmaxf(fmaxf(s_vmax[0], s_vmax[1]), fmaxf(s_vmax[2], s_vmax[3]));
      inv_vmax = vmax > 0.0f ? 1.0f / vmax : 0.0f;
    }
    for (int j = 0; j < n; ++j) {
#pragma unroll
      for (int kind = 0; kind < 2; ++kind) {
        const int i = 2 * j + kind;
        if (kind == 0) {  // the tile's scales and which of its tokens count
          const int slot = j % C::kSlots;
          s_scale[(slot * 2) * kKeys + ct] = ks[0] * p.qk_scale;
          s_scale[(slot * 2 + 1) * kKeys + ct] = vs[0] * inv_vmax;
          const unsigned m = __ballot_sync(0xffffffffu, good[0]);
          if (lane == 0) s_mask[slot * 4 + (ct >> 5)] = m;
          mbar_arrive(&sc_full[slot]);
        }
        if (kind == 0 || kBetween)
          asm volatile("cp.async.wait_group %0;" ::"n"(2 * kFar - 1) : "memory");
        else
          asm volatile("cp.async.wait_group %0;" ::"n"(2 * kFar - 2) : "memory");
        uint4 raw[kPass];
#pragma unroll
        for (int r = 0; r < kPass; ++r)
          raw[r] = *reinterpret_cast<const uint4*>(stage_of(i) + C::kTileBytes / 2 + (r * 128 + ct) * 16);
        named_barrier(1, 128);  // every code is read
        uint8_t* tile = stage_of(i) + (piece / 4) * (kKeys * 128);
        const uint32_t off = sw128_offset(row0, (piece % 4) * 32);
        const uint32_t off16 = sw128_offset(row0, (piece % 4) * 32 + 16);
#pragma unroll
        for (int r = 0; r < kPass; ++r) {  // (kStep % 8 = 0: one swizzle for all)
          const uint4 w = raw[r];
          const uint2 a = codes_to_half(w.x), b = codes_to_half(w.y), c = codes_to_half(w.z),
                      d = codes_to_half(w.w);
          *reinterpret_cast<uint4*>(tile + off + r * kStep * 128) = make_uint4(a.x, a.y, b.x, b.y);
          *reinterpret_cast<uint4*>(tile + off16 + r * kStep * 128) =
              make_uint4(c.x, c.y, d.x, d.y);
        }
        fence_proxy_async_smem();  // an MMA operand
        mbar_arrive(&kv_full[i % C::kStages]);
        if (kBetween) issue(j + 1, kind);
      }
      if (!kBetween) {
        issue(j + kFar, 0);
        issue(j + kFar, 1);
      }
    }
  } else if (warp < kIdleWarp) {
    // ---- MMA issue: a warp for each row tile, in strict turns (see prefill.cu) ---------
    if (n > 0) {
      constexpr uint32_t kIdQK = umma_f16_idesc(0, 0, kRows, kKeys);
      constexpr uint32_t kIdPV = umma_f16_idesc(0, 1, kRows, DP);
      const int x = warp - kMmaWarp;
      const bool mine = x == 0 || two;
      const uint32_t kv = smem_u32(smem + C::kOffKV);
      const uint64_t q_desc =
          umma_sw128_desc(smem_u32(smem + C::kOffQ + 2 * x * C::kTileBytes), 16, 1024);
      const uint64_t k_desc = umma_sw128_desc(kv, 16, 1024);
      const uint64_t v_desc = umma_sw128_desc(kv, kKeys * 128, 1024);
      const uint32_t s_col = tmem + x * 128, o_col = tmem + C::kOCol + x * 128;
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (ok && !mbar_wait_short(bar, parity, err)) {
          record_error(err, kDevWaitTimeout);
          ok = false;
        }
      };
      auto wait_tile = [&](int i) {
        wait(&kv_full[i % C::kStages], (uint32_t)(i / C::kStages) & 1u);
      };
      auto stage_of = [&](int i) { return (uint32_t)(i % C::kStages) * C::kTileBytes; };
      // The warps at work release a stage, each after it saw the tile, and only if
      // a later tile reuses the stage.
      auto release = [&](int i) {
        if (i + C::kStages < 2 * n) umma_commit_warp(&kv_empty[i % C::kStages]);
      };
      auto pass_turn = [&]() {
        if (lane == 0) mbar_arrive(&turn[x ^ 1]);
        __syncwarp();
      };
      auto s_of = [&](int j) { return s_col + (SHARED ? (uint32_t)(j & 1) * 128 : 0u); };
      auto qk = [&](int j, bool pass) {
        const uint64_t b = umma_desc_at(k_desc, stage_of(2 * j));
#pragma unroll
        for (int half = 1; half >= 0; --half) {  // lo first: roundings of a small sum
          const uint64_t a = umma_desc_at(q_desc, (uint32_t)half * C::kTileBytes);
#pragma unroll
          for (int kk = 0; kk < DP / 16; ++kk) {
            const uint32_t off = (uint32_t)(kk / 4) * (kKeys * 128) + (uint32_t)(kk % 4) * 32;
            umma_f16_warp(s_of(j), umma_desc_at(a, off), umma_desc_at(b, off), kIdQK,
                          (half < 1 || kk > 0) ? 1u : 0u);
            if (half == 0 && kk == DP / 16 - kEarly && pass) pass_turn();
          }
        }
        umma_commit_warp(&s_full[SHARED ? j & 1 : x]);
      };
      if (mine) {
        wait_tile(0);
        wait(&q_full[x], 0);
        tmem_fence_after_sync();
        if (ok) qk(0, false);
        release(0);
        for (int j = 0; j < n && ok; ++j) {
          if (SHARED && j + 1 < n) {  // into the other S, whose P (j - 1) is used up
            wait_tile(2 * j + 2);
            if (!ok) break;
            tmem_fence_after_sync();
            qk(j + 1, false);
            release(2 * j + 2);
          }
          wait_tile(2 * j + 1);
          if (two && (x == 1 || j > 0)) wait(&turn[x], (uint32_t)(x == 1 ? j : j - 1) & 1u);
          wait(&p_full[2 * x], (uint32_t)j & 1u);
          tmem_fence_after_sync();
          if (!ok) break;
          // P of tokens 32 i .. 32 i + 31 is in columns 32 i: hi in 16, lo in 16
          const uint64_t b = umma_desc_at(v_desc, stage_of(2 * j + 1));
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk) {
            if (kk == kKeys / 32) {
              wait(&p_full[2 * x + 1], (uint32_t)j & 1u);
              tmem_fence_after_sync();
            }
#pragma unroll
            for (int half = 0; half < 2; ++half)
              umma_f16_ta_warp(o_col, s_of(j) + (kk / 2) * 32 + half * 16 + (kk % 2) * 8,
                               umma_desc_at(b, kk * 2048), kIdPV,
                               (j % flush > 0 || kk > 0 || half > 0) ? 1u : 0u);
          }
          if (j == n - 1) umma_commit_warp(&o_full[x]);
          release(2 * j + 1);
          if constexpr (SHARED) {
            umma_commit_warp(pv_done);
            continue;
          }
          // the next K tile is converted while these run
          if (j + 1 < n) wait_tile(2 * j + 2);
          if (!ok) break;
          if (j + 1 < n) qk(j + 1, true);  // over P (j): a warp's MMAs run in order
          else pass_turn();
          if (j + 1 < n) release(2 * j + 2);
        }
      }
      umma_commit_warp(mma_done);
      mbar_drain(mma_done, 0);  // every MMA is done before tensor memory is freed
    }
  }
  } else {
  registers_up<136>();
  if (SHARED || warp < 4 || two) {
    // ---- query split, softmax, partials: thread = row --------------------------------------
    const int x = SHARED ? 0 : warp >> 2, row = tid & 127;
    const int half = SHARED ? warp >> 2 : 0;
    // exchanged between the two threads of a row: [tile parity][half][row], then [row]
    float* xch = reinterpret_cast<float*>(smem + C::kOffXch);
    auto meet = [&]() { named_barrier(2 + (warp & 3), 64); };
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t s_addr0 = tmem + lanes + x * 128, o_addr = tmem + lanes + C::kOCol + x * 128;
    const int r = pair * 256 + x * kRows + row;
    const bool valid = r < rows;
    const int seq = r / p.group;
    const int64_t head_row = (int64_t)seq * p.heads + kvh * p.group + (r - seq * p.group);
    float rf = 1.0f;  // power of two that the row was divided by
    if (n > 0) {
      // The warp takes its 32 rows one after the other, a lane per 4 channels.
      // A row's largest magnitude is scaled to [2^10, 2^11): exact, and lo's steps
      // stay far below hi's.
      uint8_t* hi_t = smem + C::kOffQ + (2 * x) * C::kTileBytes;
      uint8_t* lo_t = hi_t + C::kTileBytes;
      const int base = pair * 256 + (SHARED ? warp & 3 : warp) * 32;
      const int i_end = SHARED ? 16 + half * 16 : 32;
      const int from = base + half * 16;
      int gi = from % p.group;
      const float* row_ptr =
          p.q + ((int64_t)(from / p.group) * p.heads + kvh * p.group + gi) * p.dim + lane * 4;
      const int64_t wrap = (int64_t)(p.heads - p.group) * p.dim;  // to the next sequence's group
#pragma unroll 1
      for (int i0 = half * 16; i0 < i_end; i0 += 8) {
      float4 rowv[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {  // all loads first
        rowv[u] = make_float4(0, 0, 0, 0);
        if (base + i0 + u < rows && lane * 4 < p.dim)
          rowv[u] = *reinterpret_cast<const float4*>(row_ptr);
        row_ptr += p.dim;
        if (++gi == p.group) {
          gi = 0;
          row_ptr += wrap;
        }
      }
#pragma unroll
      for (int u8 = 0; u8 < 8; ++u8) {
        const int i = i0 + u8;
        const float4 v = rowv[u8];
        float big = fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)));
        big = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(big)));
        // 2^e from the exponent bits: e = 10 - floor(log2 big), at most 126
        int e = 137 - (int)(__float_as_uint(big) >> 23);
        if (big == 0.0f || !(big <= 3.402823466e38f)) e = 0;
        e = min(e, 126);
        const float up = __int_as_float((e + 127) << 23);
        if (lane == i) rf = __int_as_float((127 - e) << 23);
        const float f[4] = {v.x * up, v.y * up, v.z * up, v.w * up};
        uint32_t hi[2], lo[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const __half2 h = __floats2half2_rn(f[2 * u], f[2 * u + 1]);
          const float2 b = __half22float2(h);
          const __half2 r2 = __floats2half2_rn(f[2 * u] - b.x, f[2 * u + 1] - b.y);
          hi[u] = *reinterpret_cast<const uint32_t*>(&h);
          lo[u] = *reinterpret_cast<const uint32_t*>(&r2);
        }
        if (lane * 4 < DP) {
          const uint32_t off = (lane / 16) * (kRows * 128) +
                               sw128_offset((warp & 3) * 32 + i, (lane % 16) * 8);
          *reinterpret_cast<uint2*>(hi_t + off) = make_uint2(hi[0], hi[1]);
          *reinterpret_cast<uint2*>(lo_t + off) = make_uint2(lo[0], lo[1]);
        }
      }
      }
      fence_proxy_async_smem();  // an MMA operand
      mbar_arrive(&q_full[x]);
      if constexpr (SHARED) {
        if (lane / 16 == half) xch[2 * 2 * kRows + row] = rf;
        meet();
        rf = xch[2 * 2 * kRows + row];
      }
    }
    // Warps without rows only keep the hand-offs going.
    const bool busy = r - lane < rows;
    const bool flushes = n > flush;
    const uint32_t o2_addr = DP == 64 ? o_addr + 64 : tmem + lanes + C::kOCol + 128;
    float4* sums = p.sums + (((int64_t)split * gridDim.x + blockIdx.x) * 2 + x) * (DP / 4) * kRows + row;
    const int col0 = half * (DP / 2), col1 = SHARED ? col0 + DP / 2 : DP;  // of O
    const int part0 = half * 2, part1 = SHARED ? part0 + 2 : 4;  // chunks of a tile
    float since = 1.0f;  // by what O's unit has changed since `sums` was written
    float m = -INFINITY, l = 0.0f;  // m in units of S * k_scale * qk_scale
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      const int slot = j % C::kSlots;
      if (ok && (!mbar_wait_bounded(&sc_full[slot], (uint32_t)(j / C::kSlots) & 1u, err) ||
                 !mbar_wait_short(&s_full[SHARED ? j & 1 : x],
                                  (uint32_t)(SHARED ? j >> 1 : j) & 1u, err))) {
        record_error(err, kDevWaitTimeout);
        ok = false;
      }
      __syncwarp();
      tmem_fence_after_sync();
      // S (j) does not tell that P (j - 1) was taken, nor that O has P V (j - 1).
      auto wait_pv = [&]() {
        if (j > 0 && ok && !mbar_wait_short(pv_done, (uint32_t)(j - 1) & 1u, err)) {
          record_error(err, kDevWaitTimeout);
          ok = false;
        }
        __syncwarp();
        tmem_fence_after_sync();
      };
      if (!busy) {
        if constexpr (SHARED) wait_pv();  // else an arrival could count for tile j - 1
        if (!SHARED || half == 0) mbar_arrive(&p_full[2 * x]);
        if (!SHARED || half == 1) mbar_arrive(&p_full[2 * x + 1]);
        continue;
      }
      const uint32_t s_addr = s_addr0 + (SHARED ? (uint32_t)(j & 1) * 128 : 0u);
      auto flush_o = [&]() {
#pragma unroll 1
        for (int c = col0; c < col1; c += 16) {
          alignas(16) uint32_t o[16], was[16];
          tmem_load<16>(o_addr + c, o);
          if (j == flush) {
#pragma unroll
            for (int e = 0; e < 16; ++e) was[e] = 0u;
          } else if (near) {
            tmem_load<16>(o2_addr + c, was);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              *reinterpret_cast<float4*>(&was[4 * e]) = sums[(c / 4 + e) * kRows];
          }
          tmem_wait_load();
#pragma unroll
          for (int e = 0; e < 16; ++e)
            o[e] = __float_as_uint(
                fmaf(__uint_as_float(was[e]), since, __uint_as_float(o[e])));
          if (near) {
            tmem_store<16>(o2_addr + c, o);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              sums[(c / 4 + e) * kRows] = *reinterpret_cast<const float4*>(&o[4 * e]);
          }
        }
        tmem_wait_store();
        since = 1.0f;
      };
      if (!SHARED && j > 0 && j % flush == 0) flush_o();
      const float* ks = s_scale + slot * 2 * kKeys;
      const float* vs = ks + kKeys;
      const uint32_t* mask = s_mask + slot * 4;
      const bool all = (mask[0] & mask[1] & mask[2] & mask[3]) == 0xffffffffu;
      // Scores of chunk c (32 tokens) times their pages' K scales; tokens that do
      // not count become -inf.  The next chunk's loads are issued before this one's
      // arithmetic: each takes about 150 clocks.
      uint32_t s[32];
      tmem_load<32>(s_addr + part0 * 32, s);
      float k0 = ks[part0 * 32], k1 = ks[part0 * 32 + 16];  // GROUPS: of the chunk's two groups
      auto scores = [&](int c, uint64_t (&y)[16]) {
        const int next = (c + 1 < part1 ? c + 1 : part0) * 32;
        tmem_wait_load();
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float g = e < 8 ? k0 : k1;
          const uint64_t k =
              GROUPS ? f32x2(g, g) : *reinterpret_cast<const uint64_t*>(ks + c * 32 + 2 * e);
          y[e] = mul_f32x2(f32x2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), k);
        }
        tmem_load<32>(s_addr + next, s);  // after the last one the first again
        if constexpr (GROUPS) {
          k0 = ks[next];
          k1 = ks[next + 16];
        }
        if (!all) {
          const uint32_t bits = mask[c];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 a = unpack_f32x2(y[e]);
            y[e] = f32x2(bits >> (2 * e) & 1u ? a.x : -INFINITY,
                         bits >> (2 * e + 1) & 1u ? a.y : -INFINITY);
          }
        }
      };
      float tm[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      // (rolled: unrolled, the two passes were 40 KB of code, and fetching it cost
      // the first tile 16,000 clocks)
#pragma unroll 1
      for (int c = part0; c < part1; ++c) {
        uint64_t y[16];
        scores(c, y);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float2 a = unpack_f32x2(y[e]);
          tm[e & 3] = max3_nan(tm[e & 3], a.x, a.y);
        }
      }
      float t = max3_nan(max3_nan(tm[0], tm[1], tm[2]), tm[3], tm[3]);
      if constexpr (SHARED) {
        float* of = xch + (j & 1) * 2 * kRows + row;
        of[half * kRows] = t;
        meet();
        const float u = of[(half ^ 1) * kRows];
        t = max3_nan(t, u, u);
        wait_pv();
        if (j > 0 && j % flush == 0) {
          flush_o();
          tmem_fence_before_sync();
          meet();  // P of the first half lets the product start
          tmem_fence_after_sync();
        }
      }
      const bool move = valid && t > m && (m == -INFINITY || (t - m) * rf > kLazy);
      if (__any_sync(0xffffffffu, move)) {
        const float alpha = move ? ex2((m - t) * rf) : 1.0f;
        if (move) m = t;
        l *= alpha;
        since *= alpha;
        // (all columns by the first group: its P lets the product start)
        if (j % flush != 0 && half == 0) {
#pragma unroll 1
          for (int c = 0; c < DP; c += 16) {
            uint32_t o[16];
            tmem_load<16>(o_addr + c, o);
            tmem_wait_load();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_store<16>(o_addr + c, o);
          }
        }
      }
      // a NaN score makes the whole row NaN
      const float ms = t != t ? t : (m == -INFINITY ? 0.0f : m * rf) - kPShift;
      const uint64_t rf2 = f32x2(rf, rf), ms2 = f32x2(-ms, -ms);
      uint64_t sum[2] = {0, 0};
      float v0 = vs[part0 * 32], v1 = vs[part0 * 32 + 16];
#pragma unroll 1
      for (int c = part0; c < part1; ++c) {
        uint64_t y[16];
        const float u0 = v0, u1 = v1;
        if constexpr (GROUPS) {
          v0 = vs[((c + 1) & 3) * 32];
          v1 = vs[((c + 1) & 3) * 32 + 16];
        }
        scores(c, y);
        uint32_t w[32];  // 16 columns of hi, 16 of lo
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float g = e < 8 ? u0 : u1;
          const uint64_t v =
              GROUPS ? f32x2(g, g) : *reinterpret_cast<const uint64_t*>(vs + c * 32 + 2 * e);
          float2 z = unpack_f32x2(fma_f32x2(y[e], rf2, ms2));
          z.x = ex2(z.x);
          z.y = ex2(z.y);
          const uint64_t pr = f32x2(z.x, z.y);
          sum[e & 1] = add_f32x2(sum[e & 1], pr);
          const uint64_t pv = mul_f32x2(pr, v);
          const float2 f = unpack_f32x2(pv);
          const __half2 hi = __floats2half2_rn(f.x, f.y);
          const float2 b = __half22float2(hi);
          const float2 r = unpack_f32x2(sub_f32x2(pv, f32x2(b.x, b.y)));
          const __half2 lo = __floats2half2_rn(r.x, r.y);
          w[e] = *reinterpret_cast<const uint32_t*>(&hi);
          w[16 + e] = *reinterpret_cast<const uint32_t*>(&lo);
        }
        tmem_store<32>(s_addr + c * 32, w);
        if (!SHARED && c == 1) {  // half of P is there: its product can start
          tmem_wait_store();
          tmem_fence_before_sync();
          mbar_arrive(&p_full[2 * x]);
        }
      }
      const float2 l2 = unpack_f32x2(add_f32x2(sum[0], sum[1]));
      l += l2.x + l2.y;
      tmem_wait_load();  // the load that ran ahead
      tmem_wait_store();
      tmem_fence_before_sync();
      mbar_arrive(&p_full[2 * x + (SHARED ? half : 1)]);
    }
    if (n > 0) {
      if (ok && !mbar_wait_bounded(&o_full[x], 0, err)) record_error(err, kDevWaitTimeout);
      __syncwarp();
      tmem_fence_after_sync();
    }
    const float vmax = fmaxf(fmaxf(s_vmax[0], s_vmax[1]), fmaxf(s_vmax[2], s_vmax[3]));
    const int64_t slot_row = (int64_t)split * p.num_seqs * p.heads + head_row;
    if constexpr (SHARED) {  // the row's sum: the first tokens' half, then the others'
      if (n > 0 && busy) {
        float* of = xch + (n & 1) * 2 * kRows + row;
        of[half * kRows] = l;
        meet();
        l = of[0] + of[kRows];
      }
    }
    if (valid && half == 0) {
      // nothing attended: (-inf, 0); every score NaN: a NaN that the join keeps
      float2 ml = make_float2(m * rf - kPShift, l);
      if (m == -INFINITY) ml = l == 0.0f ? make_float2(-INFINITY, 0.0f) : make_float2(-1e30f, l);
      p.ml[slot_row] = ml;
    }
    if (n > 0) {
      // The rows leave through the tile's query buffers (every product with them is
      // done) in whole lines; 16-byte pieces are swizzled against bank conflicts.
      uint8_t* stage = smem + C::kOffQ + 2 * x * C::kTileBytes;
      if (busy) {
#pragma unroll 1
        for (int c = col0; c < col1; c += 16) {
          uint32_t o[16];
          alignas(16) uint32_t was[16];
          tmem_load<16>(o_addr + c, o);
          if (!flushes) {
#pragma unroll
            for (int e = 0; e < 16; ++e) was[e] = 0u;
          } else if (near) {
            tmem_load<16>(o2_addr + c, was);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              *reinterpret_cast<float4*>(&was[4 * e]) = sums[(c / 4 + e) * kRows];
          }
          tmem_wait_load();
          auto total = [&](int e) {
            return fmaf(__uint_as_float(was[e]), since, __uint_as_float(o[e])) * vmax;
          };
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *reinterpret_cast<float4*>(stage + row * DP * 4 + (((c / 4 + e) ^ (row & 7)) * 16)) =
                make_float4(total(4 * e), total(4 * e + 1), total(4 * e + 2), total(4 * e + 3));
        }
      }
      if constexpr (SHARED) meet();
      __syncwarp();  // a warp writes out its own rows, or half of them
      constexpr int kPieces = DP / 4;
      const int piece = lane % kPieces;
      if (piece * 4 < p.dim)
        for (int i = half * 16 + lane / kPieces; i < (SHARED ? 16 + half * 16 : 32);
             i += 32 / kPieces) {
          const int ri = r - lane + i, si = ri / p.group, rr = (warp & 3) * 32 + i;
          if (ri >= rows) break;
          const int64_t to = (int64_t)split * p.num_seqs * p.heads + (int64_t)si * p.heads +
                             kvh * p.group + (ri - si * p.group);
          *reinterpret_cast<float4*>(p.acc + to * p.dim + piece * 4) =
              *reinterpret_cast<const float4*>(stage + rr * DP * 4 + ((piece ^ (rr & 7)) * 16));
        }
    }
  }
  }
  tmem_fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

// ---------------------------------------------------------------------------
// Own tokens of the shapes that the decode split kernels do not take (head_dim 32,
// 64 and 96, groups of other than 1, 2, 4 or 8 heads, other page sizes).
// ---------------------------------------------------------------------------
//
// A CTA of 128 threads has up to 8 query heads of one KV head and a part of one
// sequence's pages, 64 tokens at a time: LP lanes a token, 16 codes of K and of V a
// lane, all loaded at once; products in fp32 on the CUDA cores (a few heads do not
// fill a tensor-core tile).  Partials as the decode split kernels leave them, for
// the join.  A call with 32 sequences of 20 to 520 tokens behind 4,000, 32 / 8 heads,
// head_dim 96, takes 44 us so, 294 us with the decode kernel for any shape (a CTA per
// query head, a warp per token, a thread per channel).
constexpr int kOwnTokens = 64, kOwnHeads = 8;

struct OwnParams {
  const float* q;
  const int8_t* k_cache;
  const float* k_scale;
  const int8_t* v_cache;
  const float* v_scale;
  const int32_t* tables;
  const int32_t* lens;
  float* acc;
  float2* ml;
  int64_t num_blocks;
  int heads, kv_heads, group, dim, bs, width, pages_per_split, splits;
  float qk_scale;
};

// Four INT8 codes as floats, exact: byte + 128 in the mantissa of 2^23.
__device__ __forceinline__ void codes_to_float(uint32_t w, float* f) {
  const uint32_t u = w ^ 0x80808080u;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    f[e] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 + e)) - 8388736.0f;
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int b = 16; b > 0; b /= 2) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, b));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int b = 16; b > 0; b /= 2) v += __shfl_xor_sync(0xffffffffu, v, b);
  return v;
}

template <int LP>
__global__ void __launch_bounds__(128) own_kernel(const OwnParams p, int* err) {
  constexpr int kAtOnce = 128 / LP, kPer = kOwnTokens / kAtOnce, D = LP * 16;
  constexpr int kRed = 16 * LP / 32;  // channels a lane has after the reduction
  constexpr uint32_t kNoRow = 0xffffffffu;
  __shared__ __align__(16) float s_q[kOwnHeads][D];
  __shared__ __align__(16) float s_red[4][kOwnHeads][D];
  __shared__ float s_p[kOwnHeads][kOwnTokens];
  __shared__ float s_ks[kOwnTokens], s_vs[kOwnTokens];
  __shared__ uint32_t s_row[kOwnTokens];
  __shared__ float s_m[kOwnHeads], s_l[kOwnHeads], s_alpha[kOwnHeads];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int seq = blockIdx.x / p.splits, split = blockIdx.x % p.splits;
  const int chunks = (p.group + kOwnHeads - 1) / kOwnHeads;
  const int kvh = blockIdx.y / chunks, g0 = (blockIdx.y % chunks) * kOwnHeads;
  const int ng = min(kOwnHeads, p.group - g0);
  const int want = max(p.lens[seq], 0);
  const int len = (int)min((int64_t)want, (int64_t)p.width * p.bs);
  if (len != want && split == 0 && blockIdx.y == 0 && tid == 0) record_error(err, kDevSeqTooLong);
  const int64_t t0 = (int64_t)split * p.pages_per_split * p.bs;
  const int64_t t1 = min((int64_t)len, t0 + p.pages_per_split * p.bs);
  if (t0 >= t1) return;
  const int head0 = kvh * p.group + g0;
  for (int i = tid; i < ng * D; i += 128) {
    const int g = i / D, d = i % D;
    s_q[g][d] = d < p.dim ? p.q[((int64_t)seq * p.heads + head0 + g) * p.dim + d] : 0.0f;
  }
  if (tid < kOwnHeads) s_m[tid] = -INFINITY, s_l[tid] = 0.0f;
  const int piece = tid % LP, tok0 = tid / LP;
  const uint32_t row_bytes = (uint32_t)(p.kv_heads * p.dim);
  const int64_t base = (int64_t)kvh * p.dim + piece * 16;
  float acc[kOwnHeads];
#pragma unroll
  for (int g = 0; g < kOwnHeads; ++g) acc[g] = 0.0f;

  for (int64_t t = t0; t < t1; t += kOwnTokens) {
    __syncthreads();  // the last tokens' values are used up
    if (tid < kOwnTokens) {
      const int64_t at = t + tid;
      int phys = -1, page = 0;
      if (at < t1) {
        page = (int)at / p.bs;  // (lengths are 32-bit)
        phys = p.tables[(int64_t)seq * p.width + page];
        if (phys < 0 || (int64_t)phys >= p.num_blocks) {
          phys = -1;
          record_error(err, kDevBadBlockId);
        }
      }
      s_row[tid] = phys < 0 ? kNoRow : (uint32_t)phys * p.bs + ((uint32_t)at - (uint32_t)page * p.bs);
      s_ks[tid] = phys < 0 ? 0.0f : p.k_scale[(int64_t)phys * p.kv_heads + kvh] * p.qk_scale;
      s_vs[tid] = phys < 0 ? 0.0f : p.v_scale[(int64_t)phys * p.kv_heads + kvh];
    }
    __syncthreads();
    uint4 k[kPer], v[kPer];
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const uint32_t row = s_row[tok0 + u * kAtOnce];
      k[u] = v[u] = make_uint4(0, 0, 0, 0);
      if (row != kNoRow && piece * 16 < p.dim) {
        const int64_t at = base + (int64_t)((uint64_t)row * row_bytes);
        k[u] = __ldg(reinterpret_cast<const uint4*>(p.k_cache + at));
        v[u] = __ldg(reinterpret_cast<const uint4*>(p.v_cache + at));
      }
    }
    {
      float f[kPer][16];
#pragma unroll
      for (int u = 0; u < kPer; ++u) {
        codes_to_float(k[u].x, &f[u][0]);
        codes_to_float(k[u].y, &f[u][4]);
        codes_to_float(k[u].z, &f[u][8]);
        codes_to_float(k[u].w, &f[u][12]);
      }
#pragma unroll 1
      for (int g = 0; g < ng; ++g) {
        float dot[kPer];
#pragma unroll
        for (int u = 0; u < kPer; ++u) dot[u] = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const float4 q = *reinterpret_cast<const float4*>(&s_q[g][piece * 16 + e]);
#pragma unroll
          for (int u = 0; u < kPer; ++u)
            dot[u] = fmaf(q.w, f[u][e + 3],
                          fmaf(q.z, f[u][e + 2], fmaf(q.y, f[u][e + 1], fmaf(q.x, f[u][e], dot[u]))));
        }
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
#pragma unroll
          for (int b = 1; b < LP; b *= 2) dot[u] += __shfl_xor_sync(0xffffffffu, dot[u], b);
          const int i = tok0 + u * kAtOnce;
          if (piece == 0) s_p[g][i] = s_row[i] != kNoRow ? dot[u] * s_ks[i] : -INFINITY;
        }
      }
    }
    __syncthreads();
    for (int g = warp; g < ng; g += 4) {
      const float a = s_p[g][lane], b = s_p[g][lane + 32];
      const float m_old = s_m[g], m = fmaxf(m_old, warp_max(fmaxf(a, b)));
      // (a token that does not count weighs 0; a NaN score makes the sum NaN)
      const float pa = a == -INFINITY ? 0.0f : exp2f(a - m), pb = b == -INFINITY ? 0.0f : exp2f(b - m);
      const float l = warp_sum(pa + pb);
      s_p[g][lane] = pa * s_vs[lane];
      s_p[g][lane + 32] = pb * s_vs[lane + 32];
      if (lane == 0) {
        const float alpha = m_old == -INFINITY ? 0.0f : exp2f(m_old - m);
        s_alpha[g] = alpha;
        s_l[g] = s_l[g] * alpha + l;
        s_m[g] = m;
      }
    }
    __syncthreads();
    {
      float f[kPer][16];
#pragma unroll
      for (int u = 0; u < kPer; ++u) {
        codes_to_float(v[u].x, &f[u][0]);
        codes_to_float(v[u].y, &f[u][4]);
        codes_to_float(v[u].z, &f[u][8]);
        codes_to_float(v[u].w, &f[u][12]);
      }
#pragma unroll 1
      for (int g = 0; g < ng; ++g) {
        float part[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) part[e] = 0.0f;
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
          const float w = s_p[g][tok0 + u * kAtOnce];
#pragma unroll
          for (int e = 0; e < 16; ++e) part[e] = fmaf(w, f[u][e], part[e]);
        }
        // the sum over the warp's tokens, a part of the channels to each lane
        int n = 16, first = 0;
#pragma unroll
        for (int b = 16; b >= LP; b /= 2) {
          n /= 2;
          const bool up = lane & b;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e < n) {
              const float give = up ? part[e] : part[n + e], keep = up ? part[n + e] : part[e];
              part[e] = keep + __shfl_xor_sync(0xffffffffu, give, b);
            }
          if (up) first += n;
        }
#pragma unroll
        for (int e = 0; e < kRed; ++e) s_red[warp][g][piece * 16 + first + e] = part[e];
      }
    }
    __syncthreads();
    if (tid < D)
#pragma unroll
      for (int g = 0; g < kOwnHeads; ++g)
        if (g < ng)
          acc[g] = acc[g] * s_alpha[g] +
                   ((s_red[0][g][tid] + s_red[1][g][tid]) + (s_red[2][g][tid] + s_red[3][g][tid]));
  }
  const int64_t slot = ((int64_t)seq * p.splits + split) * p.heads + head0;
#pragma unroll
  for (int g = 0; g < kOwnHeads; ++g)
    if (g < ng && tid < p.dim) p.acc[(slot + g) * p.dim + tid] = acc[g];
  // nothing attended: (-inf, 0); every score NaN: a NaN that the join keeps
  if (tid < ng) {
    const float m = s_m[tid], l = s_l[tid];
    p.ml[slot + tid] = make_float2(m == -INFINITY && l != 0.0f ? -1e30f : m, l);
  }
}

// One warp per (sequence, query head): the prefix's partials, then those of
// the sequence's own pages, in that order (deterministic).  V = dim / 32.
// Tables without any page have no kernel that reports lengths beyond them, so
// this one does.
template <int V>
__global__ void __launch_bounds__(128)
    join_kernel(const int32_t* __restrict__ seq_lens, const float* __restrict__ pre_acc,
                const float2* __restrict__ pre_ml, int pre_splits, const float* __restrict__ own_acc,
                const float2* __restrict__ own_ml, float* __restrict__ out, int num_seqs, int heads,
                int bs, int width, int pages_per_split, int own_splits,
                const int32_t* __restrict__ prefix_len, int* err) {
  constexpr int D = 32 * V;
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int64_t rows = (int64_t)num_seqs * heads;
  if (row >= rows) return;  // whole warps
  const int seq = (int)(row / heads), head = (int)(row - (int64_t)seq * heads);
  if (lane == 0 && head == 0 &&
      ((own_splits == 0 && seq_lens[seq] > 0) ||
       (seq == 0 && pre_splits == 0 && prefix_len != nullptr && *prefix_len > 0)))
    record_error(err, kDevSeqTooLong);
  const int pages = covered_pages(seq_lens[seq], bs, width);
  const int n_own = own_splits > 0 ? (pages + pages_per_split - 1) / pages_per_split : 0;
  const int n = pre_splits + n_own;
  const int64_t own0 = (int64_t)seq * own_splits * heads + head;
  auto slot = [&](int i, const float*& acc) {
    if (i < pre_splits) {
      acc = pre_acc;
      return (int64_t)i * rows + row;
    }
    acc = own_acc;
    return own0 + (int64_t)(i - pre_splits) * heads;
  };
  auto load_ml = [&](int i) {
    if (i >= n) return make_float2(-INFINITY, 0.0f);
    const float* acc;
    const int64_t s = slot(i, acc);
    return __ldcg((i < pre_splits ? pre_ml : own_ml) + s);
  };
  float M = -INFINITY;
  for (int b = 0; b < n; b += 32) M = fmaxf(M, load_ml(b + lane).x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  float den = 0.0f, sum[V];
#pragma unroll
  for (int c = 0; c < V; ++c) sum[c] = 0.0f;
  for (int b = 0; b < n; b += 32) {
    const float2 ml = load_ml(b + lane);
    const float w = ml.x != -INFINITY ? exp2f(ml.x - M) : 0.0f;
    if (ml.x != -INFINITY) den += w * ml.y;
    const int nb = min(32, n - b);
    for (int j0 = 0; j0 < nb; j0 += 8) {
      float x[8][V];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float* acc;
        const int64_t s = slot(b + min(j0 + j, nb - 1), acc);
#pragma unroll
        for (int c = 0; c < V; ++c) x[j][c] = __ldcg(acc + s * D + lane + 32 * c);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float wj = __shfl_sync(0xffffffffu, w, (j0 + j) & 31);
        if (j0 + j < nb && wj != 0.0f) {  // empty parts were not written
#pragma unroll
          for (int c = 0; c < V; ++c) sum[c] += wj * x[j][c];
        }
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) den += __shfl_xor_sync(0xffffffffu, den, o);
  const float inv = den > 0.0f || den != den ? 1.0f / den : 0.0f;
#pragma unroll
  for (int c = 0; c < V; ++c)
    out[row * D + lane + 32 * c] = den == 0.0f ? 0.0f : sum[c] * inv;
}

// Parts of the prefix: the CTAs run in waves of one per SM, a part of t tiles
// costs about t + 2 tile times (query split, pipeline start, partial).
int prefix_splits(const SharedPrefixArgs& a) {
  const int64_t tiles =
      std::max<int64_t>(1, ((int64_t)a.prefix_width * a.own.block_size + kKeys - 1) / kKeys);
  const int64_t rows = (int64_t)a.own.num_seqs * (a.own.num_heads / a.own.num_kv_heads);
  const int64_t ctas = (rows + 255) / 256 * a.own.num_kv_heads;
  int best = 1;
  int64_t best_cost = INT64_MAX;
  for (int s = 1; s <= 148 && s <= tiles; ++s) {
    const int64_t cost = (ctas * s + 147) / 148 * ((tiles + s - 1) / s + 2);
    if (cost < best_cost) {
      best_cost = cost;
      best = s;
    }
  }
  return best;
}

size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

struct PrefixWs {
  size_t pre_acc, pre_ml, own_acc, own_ml, sums, bytes;
  int splits, own_splits, own_pages;
  bool own_decode;  // own tokens by the decode split kernels
};

PrefixWs prefix_ws(const SharedPrefixArgs& a) {
  PrefixWs w;
  w.splits = a.prefix_width > 0 ? prefix_splits(a) : 0;
  w.own_decode = decode_partials_plan(a.own, &w.own_splits, &w.own_pages);
  if (!w.own_decode) {
    // Parts of 64 tokens, or longer where the tables are wide (their width says
    // little about the lengths): at most 8 to 64 parts a sequence.
    const int64_t units = (int64_t)a.own.num_seqs * a.own.num_kv_heads;
    const int most = (int)std::min<int64_t>(64, std::max<int64_t>(8, 4736 / std::max<int64_t>(units, 1)));
    w.own_pages = std::max({1, kOwnTokens / a.own.block_size,
                            (a.own.max_blocks_per_seq + most - 1) / most});
    w.own_splits = (a.own.max_blocks_per_seq + w.own_pages - 1) / w.own_pages;
  }
  if (a.own.max_blocks_per_seq == 0) w.own_splits = 0;
  const size_t rows = (size_t)a.own.num_seqs * a.own.num_heads;
  const size_t pre = rows * w.splits, own = rows * w.own_splits;
  w.pre_acc = 0;
  w.pre_ml = up256(pre * a.own.head_dim * sizeof(float));
  w.own_acc = w.pre_ml + up256(pre * sizeof(float2));
  w.own_ml = w.own_acc + up256(own * a.own.head_dim * sizeof(float));
  w.sums = w.own_ml + up256(own * sizeof(float2));
  const size_t per_head = (size_t)a.own.num_seqs * (a.own.num_heads / a.own.num_kv_heads);
  const size_t ctas = (per_head + 255) / 256 * a.own.num_kv_heads * w.splits;
  const size_t tiles = (size_t)a.prefix_width * a.own.block_size / kKeys + 1;
  const bool far = a.own.head_dim > 64 && per_head > (size_t)kRows && w.splits > 0 &&
                   (tiles + w.splits - 1) / w.splits > (size_t)kFlushFar;
  w.bytes = w.sums + (far ? ctas * 2 * kRows * 128 * sizeof(float) : 0) + 256;
  return w;
}

template <int DP, bool GROUPS, bool SHARED>
void launch_prefix_t(const PrefixParams& p, cudaStream_t stream) {
  using C = PrefixCfg<DP, SHARED>;
  auto kern = prefix_kernel<DP, GROUPS, SHARED>;
  static std::atomic<uint64_t> done{0};
  allow_shared_memory(reinterpret_cast<const void*>(kern), C::kSmemBytes, done);
  const int64_t pairs = ((int64_t)p.num_seqs * p.group + 255) / 256;
  const dim3 grid((unsigned)(pairs * p.kv_heads), (unsigned)p.splits);
  kern<<<grid, kPrefixThreads, C::kSmemBytes, stream>>>(p, device_error_word());
}

int launch_own(const DecodeArgs& o, const PrefixWs& w, float* acc, float2* ml,
               cudaStream_t stream) {
  OwnParams p;
  p.q = o.q;
  p.k_cache = o.k_cache;
  p.k_scale = o.k_scale;
  p.v_cache = o.v_cache;
  p.v_scale = o.v_scale;
  p.tables = o.block_tables;
  p.lens = o.seq_lens;
  p.acc = acc;
  p.ml = ml;
  p.num_blocks = o.num_blocks;
  p.heads = o.num_heads;
  p.kv_heads = o.num_kv_heads;
  p.group = o.num_heads / o.num_kv_heads;
  p.dim = o.head_dim;
  p.bs = o.block_size;
  p.width = o.max_blocks_per_seq;
  p.pages_per_split = w.own_pages;
  p.splits = w.own_splits;
  p.qk_scale = o.sm_scale * kLog2e;
  const int64_t x = (int64_t)o.num_seqs * w.own_splits;
  const int64_t y = (int64_t)o.num_kv_heads * ((p.group + kOwnHeads - 1) / kOwnHeads);
  if (x > 0x7fffffffLL || y > 65535) {
    set_error("more than 2^31 parts or 65,535 groups of heads");
    return kUnsupported;
  }
  const dim3 grid((unsigned)x, (unsigned)y);
  int* err = device_error_word();
  if (o.head_dim == 32)
    own_kernel<2><<<grid, 128, 0, stream>>>(p, err);
  else if (o.head_dim == 64)
    own_kernel<4><<<grid, 128, 0, stream>>>(p, err);
  else
    own_kernel<8><<<grid, 128, 0, stream>>>(p, err);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_error(std::string("own tokens launch failed: ") + cudaGetErrorString(e));
    return kCudaError;
  }
  return kOk;
}

}  // namespace

size_t shared_prefix_workspace_size(const SharedPrefixArgs& a) { return prefix_ws(a).bytes; }

int launch_shared_prefix(const SharedPrefixArgs& a, void* workspace, size_t workspace_bytes,
                         cudaStream_t stream) {
  const DecodeArgs& o = a.own;
  if (o.num_seqs == 0) return kOk;
  const PrefixWs w = prefix_ws(a);
  if (workspace == nullptr || workspace_bytes < w.bytes) {
    set_error("workspace too small for shared_prefix_attention: need " + std::to_string(w.bytes) +
              " bytes");
    return kWorkspace;
  }
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(workspace) + 255) &
                                             ~(uintptr_t)255);
  float* pre_acc = reinterpret_cast<float*>(base + w.pre_acc);
  float2* pre_ml = reinterpret_cast<float2*>(base + w.pre_ml);
  float* own_acc = reinterpret_cast<float*>(base + w.own_acc);
  float2* own_ml = reinterpret_cast<float2*>(base + w.own_ml);
  if (w.splits > 0) {
    PrefixParams p;
    p.q = o.q;
    p.k_cache = o.k_cache;
    p.k_scale = o.k_scale;
    p.v_cache = o.v_cache;
    p.v_scale = o.v_scale;
    p.table = a.prefix_table;
    p.prefix_len = a.prefix_len;
    p.acc = pre_acc;
    p.ml = pre_ml;
    p.sums = reinterpret_cast<float4*>(base + w.sums);
    p.num_blocks = o.num_blocks;
    p.num_seqs = o.num_seqs;
    p.heads = o.num_heads;
    p.kv_heads = o.num_kv_heads;
    p.group = o.num_heads / o.num_kv_heads;
    p.dim = o.head_dim;
    p.bs = o.block_size;
    p.width = a.prefix_width;
    p.splits = w.splits;
    p.qk_scale = o.sm_scale * kLog2e;
    const bool groups = o.block_size % 16 == 0;
    const bool shared = o.num_seqs * (o.num_heads / o.num_kv_heads) <= kRows;
    auto with = [&](auto dp, auto g, auto s) {
      launch_prefix_t<decltype(dp)::value, decltype(g)::value, decltype(s)::value>(p, stream);
    };
    auto with_dim = [&](auto g, auto s) {
      o.head_dim <= 64 ? with(std::integral_constant<int, 64>{}, g, s)
                       : with(std::integral_constant<int, 128>{}, g, s);
    };
    auto with_groups = [&](auto s) {
      groups ? with_dim(std::true_type{}, s) : with_dim(std::false_type{}, s);
    };
    shared ? with_groups(std::true_type{}) : with_groups(std::false_type{});
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) {
      set_error(std::string("prefix launch failed: ") + cudaGetErrorString(e));
      return kCudaError;
    }
  }
  if (w.own_splits > 0) {
    const int rc = w.own_decode ? launch_decode_partials(o, own_acc, own_ml, stream)
                                : launch_own(o, w, own_acc, own_ml, stream);
    if (rc != kOk) return rc;
  }
  const int64_t rows = (int64_t)o.num_seqs * o.num_heads;
  const unsigned grid = (unsigned)((rows + 3) / 4);
#define PKV_JOIN(V)                                                                              \
  case V:                                                                                        \
    join_kernel<V><<<grid, 128, 0, stream>>>(o.seq_lens, pre_acc, pre_ml, w.splits, own_acc,     \
                                             own_ml, o.out, o.num_seqs, o.num_heads,             \
                                             o.block_size, o.max_blocks_per_seq, w.own_pages,    \
                                             w.own_splits, a.prefix_len, device_error_word());   \
    break;
  switch (o.head_dim / 32) {
    PKV_JOIN(1) PKV_JOIN(2) PKV_JOIN(3) PKV_JOIN(4)
  }
#undef PKV_JOIN
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_error(std::string("join launch failed: ") + cudaGetErrorString(e));
    return kCudaError;
  }
  return kOk;
}

}  // namespace pkv
