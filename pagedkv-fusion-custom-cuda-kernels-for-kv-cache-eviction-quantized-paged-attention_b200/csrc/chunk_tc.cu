// Attention of new tokens over the INT8 paged cache (see chunk.cu) where a KV head has
// more rows than one mma.sync tile: chunks of prompts, drafted tokens of wide groups.
//
// A unit is 256 query rows (token, head of the group) of one KV head over the keys that
// its last row sees, in tiles of 128 keys; one CTA per SM takes an equal share of all
// units' tiles.  A unit that is cut leaves partial results, joined by a kernel behind.
// Per row tile of 128 rows
//   S = Q K^T    tcgen05 kind::f16, K's codes as exact fp16, Q as fp16 times a power of
//                two per row (two numbers, hi and lo, for fp32 queries);
//   P = exp2(...) times the key's V scale, fp16 (again two for fp32), written over S;
//   O += P V     V's codes as fp16 read MN-major.
// With 16-bit queries P is one fp16 number, whose 2^-11 adds 0.8% to the error of bf16 results
// and 43% to that of fp16 ones (3.0e-4 instead of 2.1e-4 of their root mean square): with two,
// 2,048 tokens behind 14,336 take 892 us instead of 647, 512 beside 7 decoding 100 instead of
// 80.  The row tiles take turns on the tensor cores as in prefill.cu; a unit of at most 128
// rows has its even key tiles taken by the one and its odd ones by the other, joined at its
// end.
//
// What bounds it: the softmax warps, 3,900 clocks a pair of row tiles and 128 keys (2,048 of
// them exponentials) and 1,300 in which they wait for the products between them, against
// 2,050 of products; the tensor pipe is 37% busy.  2,048 tokens behind 14,336, 32 / 8 heads:
// 636 us, 810 TFLOP/s.  A unit costs about 10 us to start and end (512 tokens behind 2,800:
// 61 us, 430 TFLOP/s).  Steps of 64 keys with two buffers of S took 720 us.
//
// Roles: two softmax warpgroups (thread = row), a loading warp (16 tokens of a page a
// box, by TMA into the half of a stage that is converted last, and the scales), four
// converting warps, an issuing warp per row tile; one warp idles.  Every role finds the
// CTA's segments by itself; rings and barriers run on over them.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "cache_mma.cuh"
#include "chunk.h"
#include "pkv_internal.h"

namespace pkv {
namespace {

constexpr int kTileRows = 128;
constexpr int kUnitRows = kTileUnitRows;
constexpr int kKeys = kTileKeys;
constexpr int kThreads = 512;
constexpr int kConvWarp = 8, kMmaWarp = 12, kLoadWarp = 14;
constexpr int kEarly = 4;      // MMAs left of a step when the turn is passed on
constexpr int kOver = kTileOver;
constexpr int kLeast = kTileLeast;
// p is kept times 2^kPShift.  A row's maximum moves in front of the next tile when a tile
// exceeded it by more than 2^kLazy, at once when it would exceed it by more than 2^kRoom:
// p is at most 2^15 in fp16, whose smallest step, 2^-24, is 2^-30 of the row's largest.
constexpr float kLazy = 4.0f, kRoom = 9.0f;
constexpr float kPShift = 6.0f;

template <int DP, int HALVES>
struct TcCfg {
  static constexpr int kTileBytes = kKeys * DP * 2;
  static constexpr int kStages = DP == 128 ? (HALVES == 1 ? 5 : 3) : 6;
  static constexpr int kSlots = 4;  // scales of so many tiles: at most three are in flight
  // The tensor cores cut off the bits that an fp32 sum cannot hold (8e-7 of a tile's sum
  // of one sign): every so many tiles O is added to a sum of its own, rounded to nearest,
  // and started anew.  16-bit results take it every 16,384 keys as prefill.cu's.
  static constexpr int kFlush = HALVES == 2 ? 5 : 128;
  static constexpr int kOffQ = 0;  // [row tile][hi, lo]; results leave through them
  static constexpr int kOffKV = 2 * HALVES * kTileBytes;
  static constexpr int kOffScale = kOffKV + kStages * kTileBytes;  // [slot][k, v][8 groups]
  static constexpr int kOffMask = kOffScale + kSlots * 64;  // [slot]: bits of the groups that count, K scales
                                                            // times sm_scale negative or not finite
  static constexpr int kOffMax = kOffMask + kSlots * 4;     // [slot]: the largest V scale
  // (base, l) of the rows of a row tile: behind the results in its query tile, or apart
  static constexpr int kOffMl = DP == 128 ? kOffQ + 16384 : kOffMax + kSlots * 4;
  static constexpr int kMlPitch = DP == 128 ? HALVES * kTileBytes : kTileRows * 8;
  static constexpr int kOffBar = kOffMax + kSlots * 4 + (DP == 128 ? 0 : 2 * kTileRows * 8);
  static constexpr int kBars = 3 * kStages + kSlots + 2 + 2 + 4 + 2 + 2 + 1;
  static constexpr int kOffMisc = kOffBar + kBars * 8;
  static constexpr int kSmemBytes = kOffMisc + 16;
  static constexpr int kOCol = 256;
  // 512 registers x 128: softmax and the others
  static constexpr int kSoftRegs = 192, kOtherRegs = 64;
  static_assert(kSmemBytes <= 227 * 1024, "shared memory");
  static_assert(256 * (kSoftRegs + kOtherRegs) <= 65536, "registers");
};

struct TcParams : TileWork {
  const void* q;
  const int8_t* k_cache;
  const float* k_scale;
  const int8_t* v_cache;
  const float* v_scale;
  const int32_t* tables;
  void* out;
  float* lse;  // nullable
  CutUnit* cuts;   // per CTA
  uint8_t* slots;  // per CTA two: of the unit that it begins with, and that it ends with
  float4* sums;    // per CTA and row tile: [DP / 4][128 rows], O of earlier tiles
  int64_t q_tok, q_head;
  int64_t num_blocks;
  int total_q, heads, dim, bs, width;
  int zero_rows;   // this kernel is the one that zeroes rows outside all sequences
  float qk_scale;  // sm_scale log2e
};

template <int DP>
struct TcSlot {
  static constexpr int kMl = kUnitRows * DP * 4;
  static constexpr int kBytes = kMl + kUnitRows * 8;
};

template <int BYTES>
__device__ __forceinline__ uint8_t* slot_of(const TcParams& p, const TileUnit& u, int part) {
  return p.slots + (int64_t)(2 * (u.cta0 + part) + (part == 0 ? 1 : 0)) * BYTES;
}

template <typename T, int DP, int HALVES>
__global__ void __launch_bounds__(kThreads, 1)
    chunk_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                    const TcParams p, int* err) {
  using C = TcCfg<DP, HALVES>;
  using S = TcSlot<DP>;
  constexpr int kStages = C::kStages, kSlots = C::kSlots;
  extern __shared__ __align__(1024) uint8_t smem[];
  float* s_scale = reinterpret_cast<float*>(smem + C::kOffScale);
  uint32_t* s_mask = reinterpret_cast<uint32_t*>(smem + C::kOffMask);
  float* s_max = reinterpret_cast<float*>(smem + C::kOffMax);
  const auto s_ml = [&](int x) { return reinterpret_cast<float2*>(smem + C::kOffMl + x * C::kMlPitch); };
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* kv_empty = kv_full + kStages;
  uint64_t* raw_full = kv_empty + kStages;  // codes that are not converted yet
  uint64_t* sc_full = raw_full + kStages;
  uint64_t* q_full = sc_full + kSlots;  // per row tile, as the next three
  uint64_t* s_full = q_full + 2;
  uint64_t* p_full = s_full + 2;  // [row tile][half of the tokens]
  uint64_t* o_full = p_full + 4;
  uint64_t* turn = o_full + 2;
  uint64_t* mma_done = turn + 2;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + C::kOffMisc);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&kv_full[i], 128);
      mbar_init(&kv_empty[i], 2);
      mbar_init(&raw_full[i], 1);
    }
    for (int i = 0; i < kSlots; ++i) mbar_init(&sc_full[i], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 128);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[2 * i], 128);
      mbar_init(&p_full[2 * i + 1], 128);
      mbar_init(&o_full[i], 1);
      mbar_init(&turn[i], 1);
    }
    mbar_init(mma_done, 2);
    mbar_fence_init();
  }
  launch_the_next();
  behind_the_last();
  if (tid == 0) p.cuts[blockIdx.x].parts = 0;
  const PlanHead head = *p.head;
  const int64_t share = tile_share(p);
  const int64_t begin = blockIdx.x * share, stop = min(begin + share, head.places);
  // rows in front of the first and behind the last sequence become zero
  if (p.zero_rows) {
    const int64_t front = (int64_t)head.q_begin * p.heads;
    const int64_t behind = (int64_t)head.q_end * p.heads;
    const int64_t outside = front + (int64_t)p.total_q * p.heads - behind;
    for (int64_t i = blockIdx.x * (kThreads / 32) + warp; i < outside; i += gridDim.x * (kThreads / 32)) {
      const int64_t r = i < front ? i : behind + i - front;
      for (int c = lane * 4; c < p.dim; c += 128)
        store4(static_cast<T*>(p.out) + r * p.dim + c, make_float4(0, 0, 0, 0));
      if (lane == 0 && p.lse != nullptr) p.lse[r] = -INFINITY;
    }
  }
  if (begin >= stop) return;

  if (warp == kMmaWarp) tmem_alloc(s_tmem, 512);
  tmem_fence_before_sync();
  __syncthreads();
  tmem_fence_after_sync();
  const uint32_t tmem = *s_tmem;
  // ok: false in a thread whose wait gave up (bounded; then every wait of the grid gives
  // up at once).  It goes on without waiting and without storing results.
  bool ok = true;
  const auto wait = [&](uint64_t* bar, int phase) {
    if (ok && !mbar_wait_short(bar, (uint32_t)phase & 1u, err)) {
      record_error(err, kDevWaitTimeout);
      ok = false;
    }
  };
  int tiles_before = 0;  // of the CTA's earlier segments
  int loaded = 0;        // tiles, by the loading warp

  if (warp >= kConvWarp) {
    registers_down<C::kOtherRegs>();
    if (warp < kMmaWarp) {
      // ---- codes to fp16 tiles ---------------------------------------------------------
      // 8 codes a lane and pass: 8 lanes' stores are then 8 pieces of one row (16 codes a
      // lane met every bank twice)
      constexpr int kLanes = DP / 8;
      constexpr int kStep = 128 / kLanes;  // token rows per pass
      constexpr int kPass = kKeys / kStep;
      const int ct = tid - kConvWarp * 32;
      const int piece = ct % kLanes, row0 = ct / kLanes;
      TileUnit u;
      u.s = plan_find(p.seq, p.seqs, begin);
      int st = 0, use = 0;
      for (int64_t now = begin; now < stop; now = u.at + u.seq.steps + kOver) {
        u.find(p, now, share);
        if (u.empty(stop)) continue;
        u.cut(p, now, stop);
#pragma unroll 1
        for (int i = 0; i < 2 * u.n; ++i) {  // K and V in turns
          uint8_t* tile = smem + C::kOffKV + st * C::kTileBytes;
          wait(&raw_full[st], use);
          uint2 raw[kPass];
#pragma unroll
          for (int r = 0; r < kPass; ++r)
            raw[r] = *reinterpret_cast<const uint2*>(tile + C::kTileBytes / 2 + (r * 128 + ct) * 8);
          named_barrier(1, 128);  // every code is read
#pragma unroll
          for (int r = 0; r < kPass; ++r) {
            const uint2 a = codes_to_half(raw[r].x), b = codes_to_half(raw[r].y);
            // (8 rows further the swizzle is the same)
            const uint32_t off = sw128_offset(row0 + r * kStep % 8, (piece % 8) * 16) + r * kStep / 8 * 1024;
            *reinterpret_cast<uint4*>(tile + (piece / 8) * (kKeys * 128) + off) =
                make_uint4(a.x, a.y, b.x, b.y);
          }
          fence_proxy_async_smem();  // an MMA operand
          mbar_arrive(&kv_full[st]);
          if (++st == kStages) st = 0, ++use;
        }
      }
    } else if (warp == kLoadWarp) {
      // ---- pages and scales ---------------------------------------------------------------
      // Lane l has the tile's group l & 7 of 16 tokens, which is on one page: its entry is
      // loaded two tiles ahead, its scales (K: lanes 0-7, V: 8-15) one.
      const uint64_t hold = l2_policy_evict_last();
      const float* scales = lane < 8 ? p.k_scale : p.v_scale;
      if (lane == 0 && p.num_blocks > 0) {  // (an empty cache has no maps)
        prefetch_tensormap(&map_k);
        prefetch_tensormap(&map_v);
      }
      TileUnit u;
      u.s = plan_find(p.seq, p.seqs, begin);
      for (int64_t now = begin; now < stop && ok; now = u.at + u.seq.steps + kOver) {
        u.find(p, now, share);
        if (u.empty(stop)) continue;
        u.cut(p, now, stop);
        const int n = u.n, len = u.seq.len;
        const int32_t* table = p.tables + (int64_t)u.s * p.width;
        const auto token_of = [&](int j) { return (u.tile0 + j) * kKeys + (lane & 7) * 16; };
        const auto entry_of = [&](int j) {
          return j < n && token_of(j) < len ? table[token_of(j) / p.bs] : -1;
        };
        const auto good = [&](int entry) { return entry >= 0 && (int64_t)entry < p.num_blocks; };
        const auto scale_of = [&](int entry) {
          return load_if(lane < 16 && good(entry), scales + (int64_t)entry * p.kv_heads + u.kvh);
        };
        int entry = entry_of(0), entry1 = entry_of(1);
        float scale = scale_of(entry);
        for (int j = 0; j < n; ++j) {
          const int entry2 = entry_of(j + 2);
          const float scale1 = scale_of(entry1);
          const int token = token_of(j), jj = tiles_before + j, slot = jj % kSlots;
          const bool there = lane < 8 && good(entry);
          const unsigned boxes = __ballot_sync(0xffffffffu, there);
          if (token < len && !good(entry)) record_error(err, kDevBadBlockId);
          const int at = entry * p.bs + token % p.bs;
#pragma unroll
          for (int kind = 0; kind < 2; ++kind) {
            const int i = 2 * jj + kind, st = i % kStages;
            wait(&kv_empty[st], i / kStages + 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            if (kind == 0) {
              // (what the slot held is used: three tiles at most are in flight)
              const float factor = lane < 8 ? scale * p.qk_scale : scale;
              if (lane < 16) s_scale[slot * 16 + lane] = factor;
              // groups behind the length are hidden by the rows' limits
              const unsigned count = boxes | __ballot_sync(0xffffffffu, token >= len);
              // (a negative sm_scale turns the order around as a negative K scale does)
              const bool odd = __any_sync(0xffffffffu, lane < 8 && !(factor >= 0.0f && factor <= 3.0e38f));
              // the largest V scale; infinity where one is not finite
              const float a = fabsf(scale);
              const uint32_t big = __reduce_max_sync(
                  0xffffffffu, lane < 8 || lane >= 16 ? 0u : a <= 3.0e38f ? __float_as_uint(a) : 0x7f800000u);
              if (lane == 0) {
                s_mask[slot] = (count & 0xffu) | (odd ? 0x100u : 0u);
                s_max[slot] = __uint_as_float(big);
              }
              __syncwarp();
              if (lane == 0) mbar_arrive(&sc_full[slot]);
            }
            if (lane == 0) mbar_arrive_expect_tx(&raw_full[st], __popc(boxes) * 16 * DP);
            __syncwarp();
            if (there)
              tma_load_3d(smem + C::kOffKV + st * C::kTileBytes + C::kTileBytes / 2 + (lane & 7) * 16 * DP,
                          kind ? &map_v : &map_k, &raw_full[st], 0, u.kvh, at, hold);
          }
          if (!ok) break;
          entry = entry1;
          entry1 = entry2;
          scale = scale1;
          loaded = jj + 1;
        }
        tiles_before += n;
      }
      // no copy and no release outlives the CTA
      if (lane == 0) {
        drain_ring(raw_full, kStages, 2 * loaded);
        drain_ring(kv_empty, kStages, 2 * loaded);
      }
    } else if (warp < kLoadWarp) {
      // ---- MMA issue: a warp for each row tile, in strict turns (see prefill.cu) ---------
      constexpr uint32_t kIdQK = umma_f16_idesc(0, 0, kTileRows, kKeys);
      constexpr uint32_t kIdPV = umma_f16_idesc(0, 1, kTileRows, DP);
      const int x = warp - kMmaWarp;
      const uint32_t kv = smem_u32(smem + C::kOffKV);
      const uint64_t q_desc =
          umma_sw128_desc(smem_u32(smem + C::kOffQ + x * HALVES * C::kTileBytes), 16, 1024);
      const uint64_t k_desc = umma_sw128_desc(kv, 16, 1024);
      const uint64_t v_desc = umma_sw128_desc(kv, kKeys * 128, 1024);
      const uint32_t s_col = tmem + x * 128, o_col = tmem + C::kOCol + x * 128;
      // a warp's lanes give up together
      const auto wait_warp = [&](uint64_t* bar, int phase) {
        wait(bar, phase);
        ok = __all_sync(0xffffffffu, ok);
      };
      const auto item = [&](int i) { return 2 * tiles_before + i; };
      const auto wait_load = [&](int i) { wait_warp(&kv_full[item(i) % kStages], item(i) / kStages); };
      const auto stage_at = [&](int i) { return (uint32_t)(item(i) % kStages) * C::kTileBytes; };
      // both warps release a stage, each after it saw the load
      const auto release = [&](int i) { umma_commit_warp(&kv_empty[item(i) % kStages]); };
      const auto pass_over = [&](int i) {
        if (lane == 0) mbar_arrive(&kv_empty[item(i) % kStages]);
        __syncwarp();
      };
      const auto pass_turn = [&]() {
        if (lane == 0) mbar_arrive(&turn[x ^ 1]);
        __syncwarp();
      };
      const auto qk = [&](int j, bool pass) {
        const uint64_t b = umma_desc_at(k_desc, stage_at(2 * j));
#pragma unroll
        for (int half = HALVES - 1; half >= 0; --half) {  // lo first: roundings of a small sum
          const uint64_t a = umma_desc_at(q_desc, (uint32_t)half * C::kTileBytes);
#pragma unroll
          for (int kk = 0; kk < DP / 16; ++kk) {
            const uint32_t off = (uint32_t)(kk / 4) * (kKeys * 128) + (uint32_t)(kk % 4) * 32;
            umma_f16_warp(s_col, umma_desc_at(a, off), umma_desc_at(b, off), kIdQK,
                          (half < HALVES - 1 || kk > 0) ? 1u : 0u);
            if (half == 0 && kk == DP / 16 - kEarly && pass) pass_turn();
          }
        }
        umma_commit_warp(&s_full[x]);
      };
      int q_uses = 0, p_uses = 0, steps = 0;
      // c: how many tiles this row tile has had
      const auto pv = [&](int j, int c) {
        const uint64_t b = umma_desc_at(v_desc, stage_at(2 * j + 1));
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk) {
          if (kk == kKeys / 32) {
            wait_warp(&p_full[2 * x + 1], p_uses);
            tmem_fence_after_sync();
            if (!ok) return;
          }
          // P of tokens 32 i .. 32 i + 31 is in columns 32 i: hi in 16, lo in 16; or
          // (16 bits) of token t in columns t / 2
#pragma unroll
          for (int half = 0; half < HALVES; ++half) {
            const uint32_t a =
                HALVES == 2 ? s_col + (kk / 2) * 32 + half * 16 + (kk % 2) * 8 : s_col + kk * 8;
            umma_f16_ta_warp(o_col, a, umma_desc_at(b, kk * 2048), kIdPV,
                             (c % C::kFlush > 0 || kk > 0 || half > 0) ? 1u : 0u);
          }
        }
        ++p_uses;
      };
      TileUnit u;
      u.s = plan_find(p.seq, p.seqs, begin);
      for (int64_t now = begin; now < stop && ok; now = u.at + u.seq.steps + kOver) {
        u.find(p, now, share);
        if (u.empty(stop)) continue;
        u.cut(p, now, stop);
        const int n = u.n, nt = x ? u.tiles[1] : u.tiles[0];
        if (n == 0) continue;
        if (u.dual) {
          // this warp's tiles are x, x + 2, ...
          if (x < n) wait_warp(&q_full[x], q_uses++);
          for (int j = 0; j < n && ok; ++j) {
            wait_load(2 * j);
            if (!ok) break;
            if ((j & 1) != x) {
              pass_over(2 * j);
              wait_load(2 * j + 1);
              pass_over(2 * j + 1);
              continue;
            }
            tmem_fence_after_sync();
            qk(j, false);
            release(2 * j);
            wait_load(2 * j + 1);
            wait_warp(&p_full[2 * x], p_uses);
            tmem_fence_after_sync();
            if (!ok) break;
            pv(j, j / 2);
            if (!ok) break;
            if (j + 2 >= n) umma_commit_warp(&o_full[x]);
            release(2 * j + 1);
          }
        } else {
          wait_load(0);
          if (nt > 0) {
            wait_warp(&q_full[x], q_uses++);
            tmem_fence_after_sync();
            if (ok) qk(0, false);
          }
          release(0);
          for (int j = 0; j < n && ok; ++j, ++steps) {
            wait_load(2 * j + 1);
            if (j + 1 < n) wait_load(2 * j + 2);
            if (x == 1 || steps > 0) wait_warp(&turn[x], x == 1 ? steps : steps - 1);
            if (j < nt) wait_warp(&p_full[2 * x], p_uses);
            tmem_fence_after_sync();
            if (!ok) break;
            if (j < nt) {
              pv(j, j);
              if (!ok) break;
              if (j == nt - 1) umma_commit_warp(&o_full[x]);
              if (j + 1 < nt) qk(j + 1, true);  // over P (j): a warp's MMAs run in order
              else pass_turn();
            } else {
              pass_turn();
            }
            release(2 * j + 1);
            if (j + 1 < n) release(2 * j + 2);
          }
        }
        tiles_before += n;
      }
      umma_commit_warp(mma_done);
      mbar_drain(mma_done, 0);  // every MMA is done before tensor memory is freed
    }
  } else {
    registers_up<C::kSoftRegs>();
    // ---- query split, softmax, results: thread = row --------------------------------------
    const int x = warp >> 2, row = tid & 127;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t s_addr = tmem + lanes + x * 128, o_addr = tmem + lanes + C::kOCol + x * 128;
    const uint32_t o2_addr = o_addr + 64;  // DP = 64: O of earlier tiles
    float4* sums = p.sums + ((int64_t)blockIdx.x * 2 + x) * (DP / 4) * kTileRows + row;
    uint8_t* q_tile = smem + C::kOffQ + x * HALVES * C::kTileBytes;
    const auto meet = [&]() { named_barrier(2 + x, 128); };
    int s_uses = 0, o_uses = 0;
    TileUnit u;
    u.s = plan_find(p.seq, p.seqs, begin);
    for (int64_t now = begin; now < stop; now = u.at + u.seq.steps + kOver) {
      u.find(p, now, share);
      if (u.empty(stop)) continue;
      u.cut(p, now, stop);
      if (tid == 0 && u.parts > 1 && u.cta0 == (int)blockIdx.x)
        p.cuts[blockIdx.x] = CutUnit{u.parts, u.rows, u.kvh, u.block, u.seq.q0, u.cta0};
      const bool dual = u.dual;
      const int first = dual ? x : 0, by = dual ? 2 : 1;
      const int nt = dual ? u.n : (x ? u.tiles[1] : u.tiles[0]);  // its tiles: first, first + by, ... < nt
      const int r0 = dual ? 0 : x * kTileRows;
      const int r = r0 + row;
      const bool valid = r < u.rows;
      const int limit = u.limit(p, r);
      const bool busy = r - lane < u.rows;  // warps without rows only keep the hand-offs going
      // tiles from here on hold keys that some row of the warp does not see
      const int first_masked = max(u.limit(p, r - lane), 0) / kKeys - u.tile0;
      float rf = 1.0f;  // power of two that the row was divided by
      if (first < nt) {
        // A row's largest magnitude is scaled to [2^10, 2^11): exact, and lo's steps stay far
        // below hi's.  (fp16 queries are as they are.)
        const T* any = static_cast<const T*>(p.q);
        const T* mine = any;
        if (valid) {
          int h;
          const int64_t tok = u.token(p, r, &h);
          mine += tok * p.q_tok + h * p.q_head;
        }
        constexpr int kBox = kTileRows * 128;
        copy_query_rows<T, DP, kBox>(smem_u32(q_tile), row - lane, any, mine, u.rows - (r - lane), p.dim);
        if constexpr (!std::is_same<T, __half>::value) {
          const int e = row_exponent(query_row_most<T, DP, kBox>(q_tile, row));
          rf = power_of_two(-e);
          split_query_row<T, DP, kBox>(q_tile, row, power_of_two(e));
        }
        fence_proxy_async_smem();  // an MMA operand
        mbar_arrive(&q_full[x]);
      }
      float since = 1.0f;  // by what O's unit has changed since the sum was written
      float m = -INFINITY, l = 0.0f;  // m in units of S * k_scale * qk_scale
      float next = -INFINITY;         // what m becomes in front of the next tile
      float unit_v = 0.0f, inv_v = 0.0f;  // a power of two above the V scales so far: O's unit
      bool spoilt = false;  // the row sees a V scale that is not finite
      int c_tile = 0;  // tiles so far
      for (int j = first; j < nt; j += by, ++c_tile) {
        const int jj = tiles_before + j, slot = jj % kSlots;
        wait(&sc_full[slot], jj / kSlots);
        const float* ks = s_scale + slot * 16;
        const float* vs = ks + 8;
        const uint32_t groups = s_mask[slot];
        float big = s_max[slot];
        const bool scaled = groups != 0xffu || j >= first_masked;
        wait(&s_full[x], s_uses++);
        __syncwarp();
        tmem_fence_after_sync();
        if (!busy) {
          mbar_arrive(&p_full[2 * x]);
          mbar_arrive(&p_full[2 * x + 1]);
          continue;
        }
        if (c_tile > 0 && c_tile % C::kFlush == 0) {  // O has the products of all earlier tiles
#pragma unroll 1
          for (int c = 0; c < DP; c += 16) {
            alignas(16) uint32_t o[16], was[16];
            tmem_load<16>(o_addr + c, o);
            if (c_tile == C::kFlush) {
#pragma unroll
              for (int e = 0; e < 16; ++e) was[e] = 0u;
            } else if (DP == 64) {
              tmem_load<16>(o2_addr + c, was);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                *reinterpret_cast<float4*>(&was[4 * e]) = sums[(c / 4 + e) * kTileRows];
            }
            tmem_wait_load();
#pragma unroll
            for (int e = 0; e < 16; ++e)
              o[e] = __float_as_uint(fmaf(__uint_as_float(was[e]), since, __uint_as_float(o[e])));
            if (DP == 64) {
              tmem_store<16>(o2_addr + c, o);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                sums[(c / 4 + e) * kTileRows] = *reinterpret_cast<const float4*>(&o[4 * e]);
            }
          }
          tmem_wait_store();
          since = 1.0f;
        }
        if (scaled) {
          // scores times their K scales, the masked ones -inf by selection, in place
          // (seldom: a rolled loop)
          const int seen = limit - (u.tile0 + j) * kKeys;  // columns below this are seen
#pragma unroll 1
          for (int c = 0; c < kKeys; c += 16) {
            uint32_t w[16];
            tmem_load<16>(s_addr + c, w);
            tmem_wait_load();
            const int here = groups >> (c / 16) & 1u ? seen - c : 0;
#pragma unroll
            for (int e = 0; e < 16; ++e)
              w[e] = e < here ? __float_as_uint(__uint_as_float(w[e]) * ks[c / 16]) : 0xff800000u;
            tmem_store<16>(s_addr + c, w);
          }
          tmem_wait_store();
        }
        float s[kKeys];
        {
          uint32_t(&w)[kKeys] = reinterpret_cast<uint32_t(&)[kKeys]>(s);
#pragma unroll
          for (int c = 0; c < kKeys; c += 32)
            tmem_load<32>(s_addr + c, reinterpret_cast<uint32_t(&)[32]>(w[c]));
          tmem_wait_load();
        }
        if (big > 3.0e38f) {
          // A V scale that is not finite makes the rows that see it NaN, and only those: it
          // counts as 0 in the products.
          big = 0.0f;
          for (int c = 0; c < kKeys / 16; ++c) {
            const float v = fabsf(vs[c]);
            if (v <= 3.0e38f) big = fmaxf(big, v);
            else if ((u.tile0 + j) * kKeys + c * 16 < limit) spoilt = true;
          }
        }
        // P is taken with the maximum as it was: the tile's own is looked for beside the
        // first half's exponentials, and moves it in front of the next tile, or, where P
        // would leave fp16 (the first tile, seldom another), at once.
        bool move = valid && next > m;
        float t = next;
        uint64_t sum[2];
        float ms;
        const auto part = [&](int c) {  // P of tokens c .. c + 31
          uint32_t hi[16], lo[HALVES == 2 ? 16 : 1];
          float g0 = vs[c / 16] * inv_v, g1 = vs[c / 16 + 1] * inv_v;
          const float k0 = scaled ? rf : ks[c / 16] * rf, k1 = scaled ? rf : ks[c / 16 + 1] * rf;
          const uint64_t ms2 = f32x2(-ms, -ms);
          if (!(fabsf(g0) <= 1.0f)) g0 = 0.0f;
          if (!(fabsf(g1) <= 1.0f)) g1 = 0.0f;
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float g = (e & 16) ? g1 : g0;
            const float k = (e & 16) ? k1 : k0;
            float2 z = unpack_f32x2(fma_f32x2(f32x2(s[c + e], s[c + e + 1]), f32x2(k, k), ms2));
            z.x = ex2(z.x);
            z.y = ex2(z.y);
            const uint64_t pr = f32x2(z.x, z.y);
            sum[(e / 2) & 1] = add_f32x2(sum[(e / 2) & 1], pr);
            const uint64_t pv = mul_f32x2(pr, f32x2(g, g));
            const float2 f = unpack_f32x2(pv);
            const __half2 h = __floats2half2_rn(f.x, f.y);
            hi[e / 2] = word_of(h);
            if constexpr (HALVES == 2) {
              const float2 b = __half22float2(h);
              lo[e / 2] = word_of(__floats2half2_rn(f.x - b.x, f.y - b.y));
            }
          }
          if constexpr (HALVES == 2) {
            tmem_store<16>(s_addr + c, hi);
            tmem_store<16>(s_addr + c + 16, lo);
          } else {
            tmem_store<16>(s_addr + c / 2, hi);
          }
        };
        for (;;) {
          if (__any_sync(0xffffffffu, move || big > unit_v)) {
            float alpha = move ? (m == -INFINITY ? 0.0f : ex2((m - t) * rf)) : 1.0f;
            if (move) m = t;
            l *= alpha;
            if (big > unit_v) {  // (the same in all threads)
              const int e = min(max((int)(__float_as_uint(big) >> 23) - 126, -126), 126);
              inv_v = power_of_two(-e);
              alpha *= unit_v * inv_v;
              unit_v = power_of_two(e);
            }
            since *= alpha;
            if (c_tile % C::kFlush != 0) {
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
          ms = (m == -INFINITY ? 0.0f : m * rf) - kPShift;
          sum[0] = sum[1] = 0;
          part(0);
          part(32);
          // The largest of each 16 tokens, which share their scale, then times it.  (K scales
          // that would change the order are among the scores already.)
          t = -INFINITY;
#pragma unroll
          for (int c = 0; c < kKeys; c += 16) {
            float tm[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) tm[e] = max3_nan(s[c + e], s[c + e + 4], s[c + e + 8]);
#pragma unroll
            for (int e = 0; e < 2; ++e) tm[e] = max3_nan(tm[e], tm[e + 2], s[c + 12 + e]);
            tm[0] = max3_nan(tm[0], tm[1], s[c + 14]);
            const float k = scaled ? 1.0f : ks[c / 16];
            t = max3_nan(t, max3_nan(tm[0], s[c + 15], s[c + 15]) * k, t);
          }
          // (NaN moves nothing, and makes the row NaN)
          move = valid && t > m && (m == -INFINITY || (t - m) * rf > kRoom);
          if (!__any_sync(0xffffffffu, move)) break;
          tmem_wait_store();  // O and P of this pass are there before the next one's accesses
          big = 0.0f;
        }
        next = (t - m) * rf > kLazy ? t : m;
        tmem_wait_store();
        tmem_fence_before_sync();
        mbar_arrive(&p_full[2 * x]);  // half of P is there: its product can start
        part(64);
        part(96);
        tmem_wait_store();
        tmem_fence_before_sync();
        mbar_arrive(&p_full[2 * x + 1]);
        const float2 l2 = unpack_f32x2(add_f32x2(sum[0], sum[1]));
        l += l2.x + l2.y;
      }
      tiles_before += u.n;
      const bool had = first < nt;
      if (had) {
        wait(&o_full[x], o_uses++);
        __syncwarp();
        tmem_fence_after_sync();
      }
      // ---- results ------------------------------------------------------------------
      const bool flushed = c_tile > C::kFlush;
      // 32 channels of the row's O, times by
      const auto take = [&](int c, float by, float (&f)[32]) {
        if (!had) {
#pragma unroll
          for (int e = 0; e < 32; ++e) f[e] = 0.0f;
          return;
        }
        uint32_t o[32];
        tmem_load<32>(o_addr + c, o);
        tmem_wait_load();
        if (flushed) {
          alignas(16) uint32_t was[32];
          if (DP == 64) {
            tmem_load<32>(o2_addr + c, was);
            tmem_wait_load();
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              *reinterpret_cast<float4*>(&was[4 * e]) = sums[(c / 4 + e) * kTileRows];
          }
#pragma unroll
          for (int e = 0; e < 32; ++e)
            o[e] = __float_as_uint(fmaf(__uint_as_float(was[e]), since, __uint_as_float(o[e])));
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) f[e] = __uint_as_float(o[e]) * by;
      };
      // base such that O and l are sums of 2^(score - base)
      float base = m == -INFINITY && l == l ? -INFINITY : (m == -INFINITY ? 0.0f : m * rf) - kPShift;
      float mine = spoilt ? __int_as_float(0x7fffffff) : unit_v;  // what this thread's O is multiplied by
      uint8_t* stage = smem + C::kOffQ + x * HALVES * C::kTileBytes;  // rows of 128 bytes, swizzled
      uint8_t* other = smem + C::kOffQ + HALVES * C::kTileBytes;
      if (dual) {  // the row's two halves meet in the first warpgroup
        s_ml(x)[row] = make_float2(base, l);
        named_barrier(4, 256);
        const float2 a = s_ml(0)[row], b = s_ml(1)[row];
        const float top = fmaxf(a.x, b.x);
        const float fa = a.x == -INFINITY ? 0.0f : ex2(a.x - top);
        const float fb = b.x == -INFINITY ? 0.0f : ex2(b.x - top);
        mine *= x ? fb : fa;
        if ((x ? b.x : a.x) == -INFINITY && !spoilt) mine = 0.0f;
        base = top;
        l = (a.x == -INFINITY ? 0.0f : a.y * fa) + (b.x == -INFINITY ? 0.0f : b.y * fb);
      }
      const bool whole = u.parts == 1;
      const bool stores = !dual || x == 0;
      const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
      uint8_t* slot = slot_of<S::kBytes>(p, u, (int)blockIdx.x - u.cta0);
      const int rows = min(kTileRows, u.rows - r0);
      // 32 channels at a time; whole units' through shared memory, so that they leave in
      // whole lines, parts as [4 channels][row]
      int to[8];  // the (token, head) of rows that this thread stores
      if (whole && stores) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          int h;
          const int64_t tok = u.token(p, r0 + min((row >> 3) + 16 * i, rows - 1), &h);
          to[i] = (int)(tok * p.heads + h);
        }
      }
#pragma unroll 1
      for (int c = 0; c < DP; c += 32) {
        float f[32];
        take(c, mine, f);
        if (dual) {
          if (x == 1) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              *reinterpret_cast<float4*>(other + row * 128 + ((e ^ (row & 7)) * 16)) =
                  make_float4(f[4 * e], f[4 * e + 1], f[4 * e + 2], f[4 * e + 3]);
          }
          named_barrier(4, 256);
          if (x == 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float4 v = *reinterpret_cast<const float4*>(other + row * 128 + ((e ^ (row & 7)) * 16));
              f[4 * e] += v.x, f[4 * e + 1] += v.y, f[4 * e + 2] += v.z, f[4 * e + 3] += v.w;
            }
          }
          named_barrier(4, 256);
        }
        if (!stores) continue;
        if (!whole) {
          if (ok && valid)
#pragma unroll
            for (int e = 0; e < 8; ++e)
              reinterpret_cast<float4*>(slot)[(c / 4 + e) * kUnitRows + r] =
                  make_float4(f[4 * e], f[4 * e + 1], f[4 * e + 2], f[4 * e + 3]);
          continue;
        }
        const bool none = l == 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          *reinterpret_cast<float4*>(stage + row * 128 + ((e ^ (row & 7)) * 16)) =
              none ? make_float4(0, 0, 0, 0)
                   : make_float4(f[4 * e] * inv, f[4 * e + 1] * inv, f[4 * e + 2] * inv, f[4 * e + 3] * inv);
        meet();
        const int piece = row & 7, at = c + piece * 4;
        if (ok && at < p.dim)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int from = (row >> 3) + 16 * i;
            if (from < rows)
              store4(static_cast<T*>(p.out) + (int64_t)to[i] * p.dim + at,
                     *reinterpret_cast<const float4*>(stage + from * 128 + ((piece ^ (from & 7)) * 16)));
          }
        meet();  // the buffer is free
      }
      if (ok && valid && stores) {
        if (whole) {
          if (p.lse != nullptr) {
            int h;
            const int64_t tok = u.token(p, r, &h);
            p.lse[tok * p.heads + h] =
                l == 0.0f ? -INFINITY : (base + log2f(l)) * (1.0f / kLog2e);
          }
        } else {
          reinterpret_cast<float2*>(slot + S::kMl)[r] = make_float2(base, l);
        }
      }
    }
  }
  tmem_fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

// Units that were cut: a CTA has 32 rows, lane = row, a warp every eighth 4 channels of
// all parts in order; the rows leave through shared memory.  Most of the CTAs have none:
// what counts is how soon they see that, and how many there are at a time (the search of
// the plan and 110 registers a thread took 12.6 us for 64 units in 148 CTAs).
constexpr int kJoinRows = 32, kJoinWarps = 8;
template <typename T, int DP>
__global__ void __launch_bounds__(kJoinWarps * 32, 4) join_tc_kernel(const TcParams p) {
  using S = TcSlot<DP>;
  constexpr int kBatch = 2, kEach = DP / 4 / kJoinWarps;
  __shared__ float4 s_out[kJoinRows][DP / 4 + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  launch_the_next();
  behind_the_last();
  const CutUnit cut = p.cuts[blockIdx.x];
  const int row0 = blockIdx.y * kJoinRows, r = row0 + lane;
  if (cut.parts == 0 || row0 >= cut.rows) return;
  TileUnit u;
  u.cta0 = blockIdx.x, u.parts = cut.parts, u.rows = cut.rows;
  u.kvh = cut.kvh, u.block = cut.block, u.seq.q0 = cut.q0;
  const bool valid = r < u.rows;
  float m = -INFINITY, l = 0.0f;
  float4 acc[kEach];
#pragma unroll
  for (int c = 0; c < kEach; ++c) acc[c] = make_float4(0, 0, 0, 0);
#pragma unroll 1
  for (int i = 0; i < u.parts; i += kBatch) {
    float2 ml[kBatch];
    float4 v[kBatch][kEach];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const bool there = valid && i + b < u.parts;
      const uint8_t* from = slot_of<S::kBytes>(p, u, i + b < u.parts ? i + b : i);
      ml[b] = there ? __ldcg(reinterpret_cast<const float2*>(from + S::kMl) + r)
                    : make_float2(-INFINITY, 0.0f);
#pragma unroll
      for (int c = 0; c < kEach; ++c)
        v[b][c] = there ? __ldcg(reinterpret_cast<const float4*>(from) + (warp + c * kJoinWarps) * kUnitRows + r)
                        : make_float4(0, 0, 0, 0);
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (ml[b].x == -INFINITY) continue;
      const float big = fmaxf(m, ml[b].x);
      const float f = m == -INFINITY ? 0.0f : ex2(m - big), k = ex2(ml[b].x - big);
      m = big;
      l = l * f + ml[b].y * k;
#pragma unroll
      for (int c = 0; c < kEach; ++c) {
        acc[c].x = acc[c].x * f + v[b][c].x * k, acc[c].y = acc[c].y * f + v[b][c].y * k;
        acc[c].z = acc[c].z * f + v[b][c].z * k, acc[c].w = acc[c].w * f + v[b][c].w * k;
      }
    }
  }
  const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
#pragma unroll
  for (int c = 0; c < kEach; ++c)
    s_out[lane][warp + c * kJoinWarps] =
        l == 0.0f ? make_float4(0, 0, 0, 0)
                  : make_float4(acc[c].x * inv, acc[c].y * inv, acc[c].z * inv, acc[c].w * inv);
  if (warp == 0 && valid && p.lse != nullptr) {
    int h;
    const int64_t tok = u.token(p, r, &h);
    p.lse[tok * p.heads + h] = l == 0.0f ? -INFINITY : (m + log2f(l)) * (1.0f / kLog2e);
  }
  __syncthreads();
#pragma unroll
  for (int i = warp; i < kJoinRows; i += kJoinWarps) {
    if (row0 + i >= u.rows || lane * 4 >= p.dim) continue;
    int h;
    const int64_t tok = u.token(p, row0 + i, &h);
    store4(static_cast<T*>(p.out) + (tok * p.heads + h) * p.dim + lane * 4, s_out[i][lane]);
  }
}

struct TcLayout {
  size_t cuts, slots, sums, total;
};

TcLayout tc_layout(const ChunkArgs& a) {
  const int dp = a.dim <= 64 ? 64 : 128;
  const int64_t tiles = ((int64_t)a.width * a.block_size + kKeys - 1) / kKeys;
  const int flush = a.dtype == 0 ? TcCfg<128, 2>::kFlush : TcCfg<128, 1>::kFlush;
  TcLayout l;
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  l.cuts = take(sizeof(CutUnit) * kChunkTcCtas);
  l.slots = take((size_t)2 * kChunkTcCtas * (dp == 64 ? TcSlot<64>::kBytes : TcSlot<128>::kBytes));
  l.sums = take(dp == 128 && tiles > flush ? (size_t)kChunkTcCtas * 2 * kTileRows * dp * 4 : 0);
  l.total = at;
  return l;
}

template <typename T, int DP>
int launch_tc(const ChunkArgs& a, PlanHead* head, PlanSeq* seq, uint8_t* ws, bool zero_rows,
              cudaStream_t stream) {
  constexpr int HALVES = sizeof(T) == 4 ? 2 : 1;
  using C = TcCfg<DP, HALVES>;
  const TcLayout lay = tc_layout(a);
  TcParams p;
  p.q = a.q;
  p.k_cache = a.k_cache;
  p.k_scale = a.k_scale;
  p.v_cache = a.v_cache;
  p.v_scale = a.v_scale;
  p.tables = a.tables;
  p.out = a.out;
  p.lse = a.lse;
  p.head = head;
  p.seq = seq;
  p.cuts = reinterpret_cast<CutUnit*>(ws + lay.cuts);
  p.slots = ws + lay.slots;
  p.sums = reinterpret_cast<float4*>(ws + lay.sums);
  p.q_tok = a.q_token_stride;
  p.q_head = a.q_head_stride;
  p.num_blocks = a.num_blocks;
  p.seqs = a.seqs;
  p.total_q = (int)a.total_q;
  p.heads = a.heads;
  p.kv_heads = a.kv_heads;
  p.group = a.heads / a.kv_heads;
  p.dim = a.dim;
  p.bs = a.block_size;
  p.width = a.width;
  p.qk_scale = a.sm_scale * kLog2e;
  p.zero_rows = zero_rows ? 1 : 0;
  const int ctas = chunk_tc_ctas(a);
  p.ctas = ctas;
  auto kern = chunk_tc_kernel<T, DP, HALVES>;
  static std::atomic<uint64_t> done{0};
  allow_shared_memory(reinterpret_cast<const void*>(kern), C::kSmemBytes, done);
  CUtensorMap map_k = {}, map_v = {};
  if (!cache_map(&map_k, a.k_cache, a, DP, 16, false) || !cache_map(&map_v, a.v_cache, a, DP, 16, false)) {
    set_error("cuTensorMapEncodeTiled failed for the caches");
    return kCudaError;
  }
  launch_behind(kern, dim3((unsigned)ctas), kThreads, C::kSmemBytes, stream, map_k, map_v, p,
                device_error_word());
  if (ctas > 1)
    launch_behind(join_tc_kernel<T, DP>, dim3((unsigned)ctas, kUnitRows / kJoinRows), kJoinWarps * 32, 0,
                  stream, p);
  return kOk;
}

}  // namespace

bool chunk_tc_takes(const ChunkArgs& a) { return a.dim <= 128 && a.block_size % 16 == 0; }

int chunk_tc_ctas(const ChunkArgs& a) {
  const int64_t units = (a.total_q * (a.heads / a.kv_heads) / kUnitRows +
                         std::min<int64_t>(a.seqs, a.total_q) + 1) * a.kv_heads;
  const int64_t steps = ((int64_t)a.width * a.block_size + kKeys - 1) / kKeys + 1 + kOver;
  return (int)std::min<int64_t>(
      kChunkTcCtas, units >= (int64_t)kChunkTcCtas * kLeast ? kChunkTcCtas : (units * steps + kLeast - 1) / kLeast);
}

PlanArgs chunk_tc_plan(const PlanArgs& base) {
  PlanArgs p = base;
  p.rows = kUnitRows;
  p.step = kKeys;
  p.over = kOver;
  p.workers = p.least = 0;
  p.counters = nullptr;
  p.counts = 0;
  return p;
}

size_t chunk_tc_workspace_size(const ChunkArgs& a) { return tc_layout(a).total; }

int launch_chunk_tc(const ChunkArgs& a, PlanHead* head, PlanSeq* seq, uint8_t* ws, bool zero_rows,
                    cudaStream_t stream) {
  const auto with_dim = [&](auto t) {
    using T = decltype(t);
    return a.dim <= 64 ? launch_tc<T, 64>(a, head, seq, ws, zero_rows, stream)
                       : launch_tc<T, 128>(a, head, seq, ws, zero_rows, stream);
  };
  return a.dtype == 0   ? with_dim(0.0f)
         : a.dtype == 1 ? with_dim(__half())
                        : with_dim(__nv_bfloat16());
}

}  // namespace pkv
