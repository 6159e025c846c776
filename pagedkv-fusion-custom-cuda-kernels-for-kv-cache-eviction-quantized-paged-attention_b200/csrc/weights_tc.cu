// Attention weights gathered per cached token (see weights.cu), by tcgen05: pages of a
// multiple of 16 tokens, head_dim up to 128.
//
// A unit is 256 query rows of one KV head over the keys that its last row sees, in tiles
// of 128 keys; one CTA per SM takes an equal share of all units' tiles.  The keys are the
// products' M and the rows their N:
//   S^T = K Q^T   tcgen05 kind::f16, 128 x (rows), K's codes as exact fp16 and Q as fp16
//                 times a power of two (two numbers for fp32 queries): of the unit, or, for
//                 rows much smaller than its largest, of the row
// so that a thread has a key and its sum over the rows crosses no lanes.  Q stays in
// shared memory for the segment, the K tiles pass, and their products have two buffers
// in tensor memory, each read by a warpgroup of its own.
//
// What bounds it: an exponential for each (row, key), 2,048 clocks a tile of 256 rows at
// 16 a clock and SM, against 1,024 of products; with what a warpgroup does between its tiles
// it is 3,000, behind 9,000 clocks until the first.  64 tokens over 32,768 cached ones,
// 32 / 8 heads: 33 us, 520 TFLOP/s.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "chunk.h"
#include "weights.h"

namespace pkv {
namespace {

constexpr int kRows = kTileUnitRows;
constexpr int kKeys = kTileKeys;
constexpr int kThreads = 512;
constexpr int kConvWarp = 8, kMmaWarp = 12, kLoadWarp = 14;
constexpr int kSlots = 8;  // scales of so many tiles
// Rows whose largest query is within 2^kNear of the unit's share its power of two: their
// operands keep 2^-26 of the row's largest.  Units with other rows take the masked tiles' loop,
// where each row has its own.
constexpr int kNear = 8;

template <int DP, int HALVES>
struct GatherCfg {
  static constexpr int kTileBytes = kKeys * DP * 2;
  static constexpr int kQBytes = kRows * DP * 2;
  static constexpr int kStages = HALVES == 2 && DP == 128 ? 3 : 4;
  static constexpr int kOffQ = 0;  // [hi, lo][64 channels][row]
  static constexpr int kOffK = HALVES * kQBytes;
  static constexpr int kOffLse = kOffK + kStages * kTileBytes;  // [row], in powers of two
  static constexpr int kOffLimit = kOffLse + kRows * 4;
  static constexpr int kOffScale = kOffLimit + kRows * 4;       // [slot][8 groups]
  static constexpr int kOffRow = kOffScale + kSlots * 32;       // [slot][8 groups]: cache rows
  static constexpr int kOffPower = kOffRow + kSlots * 32;       // [row]: exponents, 8 bits
  static constexpr int kOffBar = kOffPower + kRows;
  static constexpr int kBars = 3 * kStages + kSlots + 1 + 2 + 2 + 1;
  static constexpr int kOffMisc = kOffBar + kBars * 8;
  static constexpr int kSmemBytes = kOffMisc + 16 + 32;
  static_assert(kSmemBytes <= 227 * 1024, "shared memory");
};

struct GatherTcParams : TileWork {
  const void* q;
  const int8_t* k_cache;
  const float* k_scale;
  const int32_t* tables;
  const float* lse;
  unsigned long long* sums;
  int64_t q_tok, q_head;
  int64_t num_blocks;
  int heads, dim, bs, width;
  float qk_scale;  // sm_scale log2e
};

template <typename T, int DP, int HALVES>
__global__ void __launch_bounds__(kThreads, 1)
    gather_tc_kernel(const __grid_constant__ CUtensorMap map_k, const GatherTcParams p, int* err) {
  using C = GatherCfg<DP, HALVES>;
  constexpr int kStages = C::kStages;
  constexpr uint32_t kNoRow = 0xffffffffu;
  extern __shared__ __align__(1024) uint8_t smem[];
  float* s_lse = reinterpret_cast<float*>(smem + C::kOffLse);
  int* s_limit = reinterpret_cast<int*>(smem + C::kOffLimit);
  float* s_scale = reinterpret_cast<float*>(smem + C::kOffScale);
  uint32_t* s_row = reinterpret_cast<uint32_t*>(smem + C::kOffRow);
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* kv_empty = kv_full + kStages;
  uint64_t* raw_full = kv_empty + kStages;  // codes that are not converted yet
  uint64_t* sc_full = raw_full + kStages;
  uint64_t* q_full = sc_full + kSlots;
  uint64_t* s_full = q_full + 1;   // per buffer, as the next
  uint64_t* s_empty = s_full + 2;
  uint64_t* mma_done = s_empty + 2;
  int8_t* s_power = reinterpret_cast<int8_t*>(smem + C::kOffPower);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + C::kOffMisc);
  uint8_t* s_rows = smem + C::kOffMisc + 8;  // of each staging warp: 1: far rows, 2: idle ones
  float* s_big = reinterpret_cast<float*>(smem + C::kOffMisc + 16);  // of each staging warp

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&kv_full[i], 128);
      mbar_init(&kv_empty[i], 1);
      mbar_init(&raw_full[i], 1);
    }
    for (int i = 0; i < kSlots; ++i) mbar_init(&sc_full[i], 1);
    mbar_init(q_full, 256);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], 128);
    }
    mbar_init(mma_done, 1);
    mbar_fence_init();
  }
  launch_the_next();
  behind_the_last();
  const int64_t share = tile_share(p);
  const int64_t begin = blockIdx.x * share, stop = min(begin + share, p.head->places);
  if (begin >= stop) return;
  if (warp == kMmaWarp) tmem_alloc(s_tmem, 512);
  tmem_fence_before_sync();
  __syncthreads();
  tmem_fence_after_sync();
  const uint32_t tmem = *s_tmem;
  // ok: false in a thread whose wait gave up (bounded; then every wait of the grid gives
  // up at once).  It goes on without waiting and without adding results.
  bool ok = true;
  const auto wait = [&](uint64_t* bar, int phase) {
    if (ok && !mbar_wait_short(bar, (uint32_t)phase & 1u, err)) {
      record_error(err, kDevWaitTimeout);
      ok = false;
    }
  };
  int before = 0;  // tiles of the CTA's earlier segments
  TileUnit u;
  u.s = plan_find(p.seq, p.seqs, begin);

  if (warp >= kConvWarp && warp < kMmaWarp) {
    // ---- codes to fp16 tiles ---------------------------------------------------------
    // 8 codes a lane and pass: 8 lanes' stores are then 8 pieces of one row
    constexpr int kLanes = DP / 8;
    constexpr int kStep = 128 / kLanes;  // token rows per pass
    constexpr int kPass = kKeys / kStep;
    const int ct = tid - kConvWarp * 32;
    const int piece = ct % kLanes, row0 = ct / kLanes;
    int st = 0, use = 0;
    for (int64_t now = begin; now < stop; now = u.at + u.seq.steps + kTileOver) {
      u.find(p, now, share);
      if (u.empty(stop)) continue;
      u.cut(p, now, stop);
#pragma unroll 1
      for (int i = 0; i < u.n; ++i) {
        uint8_t* tile = smem + C::kOffK + st * C::kTileBytes;
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
    // ---- pages, scales and cache rows ------------------------------------------------------
    // Lane l has the tile's group l & 7 of 16 tokens, which is on one page: its entry is
    // loaded two tiles ahead, its scale one.
    const uint64_t hold = l2_policy_evict_first();
    if (lane == 0 && p.num_blocks > 0) prefetch_tensormap(&map_k);  // (an empty cache has no map)
    int loaded = 0;
    for (int64_t now = begin; now < stop && ok; now = u.at + u.seq.steps + kTileOver) {
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
        return load_if(lane < 8 && good(entry), p.k_scale + (int64_t)entry * p.kv_heads + u.kvh);
      };
      int entry = entry_of(0), entry1 = entry_of(1);
      float scale = scale_of(entry);
      for (int j = 0; j < n; ++j) {
        const int entry2 = entry_of(j + 2);
        const float scale1 = scale_of(entry1);
        const int token = token_of(j), jj = before + j, slot = jj % kSlots, st = jj % kStages;
        const bool there = lane < 8 && good(entry);
        const unsigned boxes = __ballot_sync(0xffffffffu, there);
        if (token < len && !good(entry)) record_error(err, kDevBadBlockId);
        const int at = entry * p.bs + token % p.bs;
        wait(&kv_empty[st], jj / kStages + 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        // (what the slot held is used: its tile's product, and with it that of the tile two
        // further, were taken up before the stages that are in flight were free)
        if (lane < 8) {
          s_scale[slot * 8 + lane] = scale * p.qk_scale;
          s_row[slot * 8 + lane] = there ? (uint32_t)at : kNoRow;
        }
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&sc_full[slot]);
          mbar_arrive_expect_tx(&raw_full[st], __popc(boxes) * 16 * DP);
        }
        __syncwarp();
        if (there)
          tma_load_3d(smem + C::kOffK + st * C::kTileBytes + C::kTileBytes / 2 + lane * 16 * DP, &map_k,
                      &raw_full[st], 0, u.kvh, at, hold);
        entry = entry1;
        entry1 = entry2;
        scale = scale1;
        loaded = jj + 1;
      }
      before += n;
    }
    // no copy and no release outlives the CTA
    if (lane == 0) {
      drain_ring(raw_full, kStages, loaded);
      drain_ring(kv_empty, kStages, loaded);
    }
  } else if (warp == kMmaWarp) {
    // ---- products -----------------------------------------------------------------------
    const uint64_t q_desc = umma_sw128_desc(smem_u32(smem + C::kOffQ), 16, 1024);
    const uint64_t k_desc = umma_sw128_desc(smem_u32(smem + C::kOffK), 16, 1024);
    // a warp's lanes give up together
    const auto wait_warp = [&](uint64_t* bar, int phase) {
      wait(bar, phase);
      ok = __all_sync(0xffffffffu, ok);
    };
    int segments = 0;
    for (int64_t now = begin; now < stop && ok; now = u.at + u.seq.steps + kTileOver) {
      u.find(p, now, share);
      if (u.empty(stop)) continue;
      u.cut(p, now, stop);
      if (u.n == 0) continue;
      // as many columns as are read
      const uint32_t id = umma_f16_idesc(0, 0, kKeys, (u.rows + 31) / 32 * 32);
      wait_warp(q_full, segments++);
      for (int j = 0; j < u.n && ok; ++j) {
        const int jj = before + j, st = jj % kStages, buffer = jj & 1;
        wait_warp(&kv_full[st], jj / kStages);
        wait_warp(&s_empty[buffer], jj / 2 + 1);
        tmem_fence_after_sync();
        if (!ok) break;
        const uint64_t a = umma_desc_at(k_desc, (uint32_t)st * C::kTileBytes);
#pragma unroll
        for (int half = HALVES - 1; half >= 0; --half) {  // lo first: roundings of a small sum
          const uint64_t b = umma_desc_at(q_desc, (uint32_t)half * C::kQBytes);
#pragma unroll
          for (int kk = 0; kk < DP / 16; ++kk)
            umma_f16_warp(tmem + buffer * 256,
                          umma_desc_at(a, (uint32_t)(kk / 4) * (kKeys * 128) + (uint32_t)(kk % 4) * 32),
                          umma_desc_at(b, (uint32_t)(kk / 4) * (kRows * 128) + (uint32_t)(kk % 4) * 32), id,
                          (half < HALVES - 1 || kk > 0) ? 1u : 0u);
        }
        umma_commit_warp(&s_full[buffer]);
        umma_commit_warp(&kv_empty[st]);
      }
      before += u.n;
    }
    umma_commit_warp(mma_done);
    mbar_drain(mma_done, 0);  // every MMA is done before tensor memory is freed
  } else if (warp < kConvWarp) {
    // ---- queries, then a thread per key ---------------------------------------------------
    const int x = warp >> 2, row = tid & 127;
    const uint32_t s_at = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + x * 256;
    for (int64_t now = begin; now < stop; now = u.at + u.seq.steps + kTileOver) {
      u.find(p, now, share);
      if (u.empty(stop)) continue;
      u.cut(p, now, stop);
      if (u.n == 0) continue;
      named_barrier(2, 256);  // both warpgroups have seen every product of the last segment
      float down = 1.0f;      // what the products are multiplied by, for the power of two
      {
        // thread = row: its denominator, how far it sees, and its queries
        const int r = tid;
        const T* any = static_cast<const T*>(p.q);
        const T* mine = any;
        float lse2 = INFINITY;  // rows that are not there, or have no denominator, add nothing
        bool idle = false, far = false;
        if (r < u.rows) {
          int h;
          const int64_t tok = u.token(p, r, &h);
          mine += tok * p.q_tok + h * p.q_head;
          const float v = p.lse[tok * p.heads + h];
          idle = v == -INFINITY;
          if (!idle) lse2 = v * kLog2e;
        }
        s_lse[r] = lse2;
        s_limit[r] = idle ? 0 : u.limit(p, r);  // (their queries may be NaN)
        constexpr int kBox = kRows * 128;
        uint8_t* tile = smem + C::kOffQ;
        copy_query_rows<T, DP, kBox>(smem_u32(tile), r - lane, any, mine, u.rows - (r - lane), p.dim);
        if constexpr (!std::is_same<T, __half>::value) {
          // the largest magnitude is scaled to [2^10, 2^11); infinity and NaN are no matter,
          // since they take their row's weights with them
          const float row_big = query_row_most<T, DP, kBox>(tile, r);
          const bool finite = row_big <= 3.402823466e38f;
          float big = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(finite ? row_big : 0.0f)));
          if (lane == 0) s_big[warp] = big;
          named_barrier(2, 256);
          for (int w = 0; w < 8; ++w) big = fmaxf(big, s_big[w]);
          const int unit_e = row_exponent(big), own_e = row_exponent(row_big);
          far = finite && row_big != 0.0f && own_e - unit_e > kNear;
          const int e = far ? own_e : unit_e;
          down = power_of_two(-unit_e);
          s_power[r] = (int8_t)-e;
          split_query_row<T, DP, kBox>(tile, r, power_of_two(e));
        }
        // (rows that see no key anyway are not the point)
        const int odd = (__any_sync(0xffffffffu, far) ? 1 : 0) |
                        (__any_sync(0xffffffffu, idle && u.limit(p, r) > 0) ? 2 : 0);
        if (lane == 0) s_rows[warp] = (uint8_t)odd;
        fence_proxy_async_smem();  // an MMA operand
        mbar_arrive(q_full);
        named_barrier(2, 256);  // all denominators are there
      }
      int odd_rows = 0;
      for (int w = 0; w < 8; ++w) odd_rows |= s_rows[w];
      const bool apart = odd_rows & 1;                   // rows have their own power, s_power's
      const int clear = odd_rows != 0 ? 0 : s_limit[0];  // every row sees, and counts for, the keys below
      const int columns = (u.rows + 31) / 32 * 32;
      for (int j = (before & 1) == x ? 0 : 1; j < u.n; j += 2) {
        const int jj = before + j, slot = jj % kSlots;
        wait(&sc_full[slot], jj / kSlots);
        const float k_scale = s_scale[slot * 8 + row / 16], k = k_scale * down;
        const uint32_t group = s_row[slot * 8 + row / 16];
        const int key = (u.tile0 + j) * kKeys + row;
        wait(&s_full[x], jj / 2);
        __syncwarp();
        tmem_fence_after_sync();
        uint64_t sum[2] = {0, 0};
        const uint64_t k2 = f32x2(k, k);
        uint32_t w[32];
        if ((u.tile0 + j + 1) * kKeys <= clear) {
          tmem_load<32>(s_at, w);
#pragma unroll 1
          for (int c = 0; c < columns; c += 32) {
            tmem_wait_load();
            float2 z[16];
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              const float4 b = *reinterpret_cast<const float4*>(s_lse + c + 2 * e);
              z[e] = unpack_f32x2(fma_f32x2(
                  f32x2(__uint_as_float(w[2 * e]), __uint_as_float(w[2 * e + 1])), k2, f32x2(-b.x, -b.y)));
              z[e + 1] = unpack_f32x2(fma_f32x2(
                  f32x2(__uint_as_float(w[2 * e + 2]), __uint_as_float(w[2 * e + 3])), k2, f32x2(-b.z, -b.w)));
            }
            if (c + 32 < columns) {
              tmem_load<32>(s_at + c + 32, w);  // on its way meanwhile
            } else {  // the next products can come
              tmem_fence_before_sync();
              mbar_arrive(&s_empty[x]);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e)
              sum[e & 1] = add_f32x2(sum[e & 1], f32x2(ex2(z[e].x), ex2(z[e].y)));
          }
        } else {
          // tiles with keys that some row does not see, or with odd rows
          float total = 0.0f;
          const auto masked = [&](auto own) {
#pragma unroll 1
            for (int c = 0; c < columns; c += 32) {
              tmem_load<32>(s_at + c, w);
              tmem_wait_load();
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                const float by = decltype(own)::value ? k_scale * power_of_two(s_power[c + e]) : k;
                const float z = ex2(fmaf(__uint_as_float(w[e]), by, -s_lse[c + e]));
                total += key < s_limit[c + e] ? z : 0.0f;
              }
            }
          };
          if (std::is_same<T, __half>::value || !apart) masked(std::false_type{});
          else masked(std::true_type{});
          sum[0] = f32x2(total, 0.0f);
          tmem_fence_before_sync();
          mbar_arrive(&s_empty[x]);
        }
        const float2 a = unpack_f32x2(add_f32x2(sum[0], sum[1]));
        if (ok && group != kNoRow && key < u.seq.len) add_weight(p.sums + group + row % 16, a.x + a.y);
      }
      before += u.n;
    }
  }
  tmem_fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

template <typename T, int DP>
int launch_gather_tc_t(const ChunkArgs& a, const float* lse, PlanHead* head, PlanSeq* seq,
                       unsigned long long* sums, cudaStream_t stream) {
  constexpr int HALVES = sizeof(T) == 4 ? 2 : 1;
  using C = GatherCfg<DP, HALVES>;
  GatherTcParams p;
  p.head = head;
  p.seq = seq;
  p.seqs = a.seqs;
  p.group = a.heads / a.kv_heads;
  p.kv_heads = a.kv_heads;
  p.q = a.q;
  p.k_cache = a.k_cache;
  p.k_scale = a.k_scale;
  p.tables = a.tables;
  p.lse = lse;
  p.sums = sums;
  p.q_tok = a.q_token_stride;
  p.q_head = a.q_head_stride;
  p.num_blocks = a.num_blocks;
  p.heads = a.heads;
  p.dim = a.dim;
  p.bs = a.block_size;
  p.width = a.width;
  p.qk_scale = a.sm_scale * kLog2e;
  p.ctas = chunk_tc_ctas(a);
  CUtensorMap map_k = {};
  if (!cache_map(&map_k, a.k_cache, a, DP, 16, false)) {
    set_error("cuTensorMapEncodeTiled failed for the cache");
    return kCudaError;
  }
  auto kern = gather_tc_kernel<T, DP, HALVES>;
  static std::atomic<uint64_t> done{0};
  allow_shared_memory(reinterpret_cast<const void*>(kern), C::kSmemBytes, done);
  launch_behind(kern, dim3((unsigned)p.ctas), kThreads, C::kSmemBytes, stream, map_k, p, device_error_word());
  return kOk;
}

}  // namespace

int launch_gather_tc(const ChunkArgs& a, const float* lse, PlanHead* head, PlanSeq* seq,
                     unsigned long long* sums, cudaStream_t stream) {
  const auto with_dim = [&](auto t) {
    using T = decltype(t);
    return a.dim <= 64 ? launch_gather_tc_t<T, 64>(a, lse, head, seq, sums, stream)
                       : launch_gather_tc_t<T, 128>(a, lse, head, seq, sums, stream);
  };
  return a.dtype == 0   ? with_dim(0.0f)
         : a.dtype == 1 ? with_dim(__half())
                        : with_dim(__nv_bfloat16());
}

}  // namespace pkv
