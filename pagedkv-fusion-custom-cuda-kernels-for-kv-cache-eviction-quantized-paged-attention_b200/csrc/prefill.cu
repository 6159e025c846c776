// Attention over packed prompts: out[i] = sum_j softmax_j(scale q_i . k_j) v_j
// over the keys j of token i's sequence, causal from the sequences' ends
// (j <= i + Lk - Lq), grouped heads, fp16 or bf16 with fp32 accumulators.
//
// One CTA owns two row tiles of 128 rows of one KV head.  A row is a (token,
// query head of the group) pair, so the G heads of a group share every K / V
// tile that is loaded.  Keys come in tiles of 128 tokens; per row tile
//   S = Q K^T    tcgen05 kind::f16, 128 x 128, K-major A and B from shared
//                memory, S in 128 columns of tensor memory;
//   P = exp2(scale log2e (S - m)), one thread per row, written back over S as
//                16-bit values;
//   O += P V     A = P from tensor memory, B = the V tile read MN-major.
// The two row tiles alternate: while the softmax warps of one turn S into P,
// the tensor cores work for the other.
//
// The running maximum m is moved only when a tile's maximum exceeds it by
// more than 2^8 (the exponentials then stay below 2^8, exact enough in fp32
// sums and 16-bit P); O is rescaled in tensor memory by its softmax warps
// then, which is safe because S(j) is complete only after P V (j - 1).
//
// Masked places hold no influence: masked scores become -inf by selection,
// and in tiles that contain masked keys the V rows are cleaned first (by
// five warps, off the critical path): rows past the sequence become zero, and
// where causal masking hides a key from some rows, its non-finite values are
// taken out of the product and added, in the epilogue, to the rows that see
// it.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>
#include <string>
#include <type_traits>

#include "pkv_common.cuh"
#include "pkv_internal.h"

namespace pkv {
namespace {

constexpr int kRows = 128;      // rows of a row tile (MMA M)
constexpr int kKeys = 128;      // keys of a tile (MMA N of Q K^T, K of P V)
constexpr int kPreThreads = 512;  // softmax A and B (4 warps each), load, MMA A and B, cleaning (5)
constexpr int kLoadWarp = 8, kMmaWarp = 9, kCleanWarp = 11;
constexpr int kCleaners = kPreThreads - kCleanWarp * 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLazy = 8.0f;   // log2 growth of a row maximum that moves it
constexpr int kPart = 64;        // keys of P that are handed over first
constexpr int kEarly = 4;        // MMAs left of a step when the turn is passed on
constexpr int kMaskedTiles = 4; // tiles with masked keys per CTA: 256 tokens span at most 3

template <int DP>
struct PreCfg {
  static constexpr int kChunks = DP / 64;               // 128-byte column chunks
  static constexpr int kTileBytes = kKeys * DP * 2;     // a K, V or Q tile
  static constexpr int kStages = DP == 128 ? 5 : 8;     // K / V ring
  static constexpr int kOffQ = 0;                       // two Q tiles
  static constexpr int kOffKV = 2 * kTileBytes;
  static constexpr int kOffBar = kOffKV + kStages * kTileBytes;
  static constexpr int kBars = 2 * kStages + 10 + kMaskedTiles + 3;
  static constexpr int kOffMisc = kOffBar + kBars * 8;
  static constexpr int kSmemBytes = kOffMisc + 64 + kMaskedTiles * 16 + 1024;
  static constexpr int kSCol = 0;                       // S / P of the two tiles
  static constexpr int kOCol = 256;
};

struct PreParams {
  const int32_t* cu_q;
  const int32_t* cu_k;
  void* out;
  float* lse;   // nullable
  const void* v;
  int64_t v_tok, v_head;
  int num_seqs, total_q, total_k;
  int heads, kv_heads, group, dim, tile_tokens;
  float scale_log2, scale;
  int causal;
};

struct PreWork {
  int q0, lq, k0, lk;  // the sequence's rows in the packed tensors
  int t0;              // first token (in the sequence) of row tile 0
};

// Sequence and token range of pair `pair` (of 2 * tile_tokens tokens).  Pairs
// are numbered sequence by sequence, the last pair of a sequence first: under
// a causal mask it is the longest, and long work should start early.  The rows
// behind the last sequence form one more sequence without keys (zeros).
// One warp; false when `pair` is past the end.
__device__ bool find_work(const PreParams& p, int pair, PreWork& w, int* err) {
  const int lane = threadIdx.x & 31;
  const int span = 2 * p.tile_tokens;
  int base = 0;
  for (int s0 = 0; s0 <= p.num_seqs; s0 += 32) {
    const int s = s0 + lane;
    int q0 = 0, q1 = 0;
    if (s < p.num_seqs) {
      const int a = p.cu_q[s], b = p.cu_q[s + 1];
      q0 = min(max(a, 0), p.total_q);
      q1 = min(max(b, q0), p.total_q);
      const int ka = p.cu_k[s], kb = p.cu_k[s + 1];
      if (pair == 0 && (a != q0 || b != q1 || ka < 0 || kb < ka || kb > p.total_k))
        record_error(err, kDevBadSeqlens);
    } else if (s == p.num_seqs) {
      q0 = min(max(p.cu_q[s], 0), p.total_q);
      q1 = p.total_q;
    }
    const int n = (q1 - q0 + span - 1) / span;
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    const int total = __shfl_sync(0xffffffffu, incl, 31);
    if (pair < base + total) {
      const unsigned m = __ballot_sync(0xffffffffu, pair < base + incl);
      const int src = __ffs(m) - 1;
      const int local = pair - base - (__shfl_sync(0xffffffffu, incl, src) -
                                       __shfl_sync(0xffffffffu, n, src));
      w.q0 = __shfl_sync(0xffffffffu, q0, src);
      w.lq = __shfl_sync(0xffffffffu, q1, src) - w.q0;
      w.t0 = (__shfl_sync(0xffffffffu, n, src) - 1 - local) * span;
      const int seq = s0 + src;
      w.k0 = 0;
      w.lk = 0;
      if (seq < p.num_seqs) {
        w.k0 = min(max(p.cu_k[seq], 0), p.total_k);
        w.lk = min(max(p.cu_k[seq + 1], w.k0), p.total_k) - w.k0;
      }
      return true;
    }
    base += total;
  }
  return false;
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }

// Both 16-bit floats of a word times zero: +-0 if they are finite, else NaN.
__device__ __forceinline__ uint32_t times_zero(uint32_t w, __nv_bfloat16) {
  const __nv_bfloat162 v = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w),
                                   __float2bfloat162_rn(0.0f));
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t times_zero(uint32_t w, __half) {
  const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&w), __float2half2_rn(0.0f));
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Whether either 16-bit float of a word is infinite or NaN (all exponent bits set).
__device__ __forceinline__ uint32_t nonfinite_mask(uint32_t w, __nv_bfloat16) {
  return ((w & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) |
         ((w & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
}
__device__ __forceinline__ uint32_t nonfinite_mask(uint32_t w, __half) {
  return ((w & 0x7c00u) == 0x7c00u ? 0xffffu : 0u) |
         ((w & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u);
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T, int DP>
__global__ void __launch_bounds__(kPreThreads, 1)
    prefill_kernel(const __grid_constant__ CUtensorMap map_q,
                   const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v, const PreParams p, int* err) {
  using C = PreCfg<DP>;
  constexpr int kBf16 = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* kv_empty = kv_full + C::kStages;
  uint64_t* q_full = kv_empty + C::kStages;  // per row tile, as the next three
  uint64_t* s_full = q_full + 2;
  uint64_t* p_full = s_full + 2;  // [row tile][part of P]
  uint64_t* o_full = p_full + 4;
  uint64_t* raw_full = o_full + 2;  // V tiles with masked keys, before they are cleaned
  uint64_t* mma_done = raw_full + kMaskedTiles;
  uint64_t* turn = mma_done + 1;  // per row tile
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + C::kOffMisc);
  int* s_work = reinterpret_cast<int*>(smem + C::kOffMisc + 16);
  uint32_t* s_flags = reinterpret_cast<uint32_t*>(smem + C::kOffMisc + 64);  // [tile][4]

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kvh = blockIdx.x % p.kv_heads;
  if (warp == 0) {
    PreWork w = {0, 0, 0, 0, 0};
    const bool any = find_work(p, blockIdx.x / p.kv_heads, w, err);
    if (lane == 0) {
      s_work[0] = any;
      s_work[1] = w.q0;
      s_work[2] = w.lq;
      s_work[3] = w.k0;
      s_work[4] = w.lk;
      s_work[5] = w.t0;
    }
  }
  if (tid == 32) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 2);  // both MMA warps
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[2 * i], 128);
      mbar_init(&p_full[2 * i + 1], 128);
      mbar_init(&o_full[i], 1);
    }
    for (int i = 0; i < kMaskedTiles; ++i) mbar_init(&raw_full[i], 1);
    mbar_init(mma_done, 2);
    mbar_init(&turn[0], 1);
    mbar_init(&turn[1], 1);
    mbar_fence_init();
  }
  if (warp == kMmaWarp) tmem_alloc(s_tmem, 512);
  if (warp == kCleanWarp && lane < kMaskedTiles * 4) s_flags[lane] = 0u;
  tmem_fence_before_sync();
  __syncthreads();
  tmem_fence_after_sync();
  const uint32_t tmem = *s_tmem;
  if (s_work[0]) {
    const int q0 = s_work[1], lq = s_work[2], k0 = s_work[3], lk = s_work[4], t0 = s_work[5];
    const int shift = lk - lq;  // key of token i under the causal mask: i + shift
    // key tiles of each row tile: up to the last key that its last token sees
    int n_tiles[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int first = t0 + x * p.tile_tokens;
      const int last = min(first + p.tile_tokens, lq) - 1;
      int keys = first < lq ? (p.causal ? min(max(last + shift + 1, 0), lk) : lk) : 0;
      n_tiles[x] = (keys + kKeys - 1) / kKeys;
    }
    const int n = max(n_tiles[0], n_tiles[1]);
    // tiles from here on hold keys that some row does not see
    const int first_masked =
        p.causal ? min(max(t0 + shift + 1, 0), lk) / kKeys : lk / kKeys;

    if (warp >= 8) {
    // 256 x 200 + 256 x 56 = 65,536 = 512 x 128, the registers at launch
    registers_down<56>();
    if (warp == kLoadWarp) {
      // ---- loads: the Q tiles, then K and V tiles in turn ----------------------
      if (lane == 0 && n > 0) {
        const uint64_t keep = l2_policy_evict_first();
        for (int x = 0; x < 2; ++x) {
          if (n_tiles[x] == 0) continue;
          mbar_arrive_expect_tx(&q_full[x],
                                (uint32_t)(C::kChunks * p.tile_tokens * p.group * 128));
          for (int c = 0; c < C::kChunks; ++c)
            tma_load_3d(smem + C::kOffQ + x * C::kTileBytes + c * kRows * 128, &map_q, &q_full[x],
                        c * 64, kvh * p.group, q0 + t0 + x * p.tile_tokens, keep);
        }
        uint64_t hold;
        asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(hold));
        int i = 0;
        bool ok = true;
        for (int j = 0; j < n && ok; ++j) {
          for (int kind = 0; kind < 2; ++kind, ++i) {
            const int st = i % C::kStages;
            if (!mbar_wait_bounded(&kv_empty[st], ((uint32_t)(i / C::kStages) & 1u) ^ 1u, err)) {
              record_error(err, kDevWaitTimeout);
              ok = false;
              break;
            }
            // a V tile with masked keys goes through the cleaning warps, which
            // complete kv_full in the load's place
            uint64_t* bar =
                kind == 1 && j >= first_masked ? &raw_full[j - first_masked] : &kv_full[st];
            mbar_arrive_expect_tx(bar, C::kTileBytes);
            for (int c = 0; c < C::kChunks; ++c)
              tma_load_3d(smem + C::kOffKV + st * C::kTileBytes + c * kKeys * 128,
                          kind ? &map_v : &map_k, bar, c * 64, kvh, k0 + j * kKeys, hold);
          }
        }
        drain_ring(kv_full, C::kStages, i);  // no copy outlives the CTA
        for (int f = 0; 2 * (first_masked + f) + 1 < i; ++f) mbar_drain(&raw_full[f], 0);
        for (int x = 0; x < 2; ++x)
          if (n_tiles[x] > 0) mbar_drain(&q_full[x], 0);
      }
    } else if (warp < kCleanWarp) {
      // ---- MMA issue: a warp for each row tile, in strict turns -----------------------
      // A wait that follows MMAs in a warp's queue returns only when they have
      // been taken up, so with one warp for both tiles the tensor cores ran dry at
      // every wait.  With two, one waits while the other's MMAs run; the turn is
      // passed on before a step's last MMAs, to cover its own latency.  Without
      // turns the tiles fall into step, and first their exponentials compete, then
      // their products.
      if (n > 0) {
        constexpr uint32_t kIdQK = umma_f16_idesc(kBf16, 0, kRows, kKeys);
        constexpr uint32_t kIdPV = umma_f16_idesc(kBf16, 1, kRows, DP);
        const int x = warp - kMmaWarp;
        const int nt = n_tiles[x];
        const uint32_t kv = smem_u32(smem + C::kOffKV);
        const uint64_t q_desc =
            umma_sw128_desc(smem_u32(smem + C::kOffQ + x * C::kTileBytes), 16, 1024);
        const uint64_t k_desc = umma_sw128_desc(kv, 16, 1024);
        const uint64_t v_desc = umma_sw128_desc(kv, kKeys * 128, 1024);
        const uint32_t s_col = tmem + C::kSCol + x * 128, o_col = tmem + C::kOCol + x * 128;
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity) {
          if (ok && !mbar_wait_short(bar, parity, err)) {
            record_error(err, kDevWaitTimeout);
            ok = false;
          }
        };
        auto wait_load = [&](int i) {
          wait(&kv_full[i % C::kStages], (uint32_t)(i / C::kStages) & 1u);
        };
        auto stage_of = [&](int i) { return (uint32_t)(i % C::kStages) * C::kTileBytes; };
        // Both warps release a stage, each after it saw the load, and only if a
        // later load reuses the stage.
        auto release = [&](int i) {
          if (i + C::kStages < 2 * n) umma_commit_warp(&kv_empty[i % C::kStages]);
        };
        auto pass_turn = [&]() {
          if (lane == 0) mbar_arrive(&turn[x ^ 1]);
          __syncwarp();
        };
        auto qk = [&](int j, bool pass) {
          const uint64_t b = umma_desc_at(k_desc, stage_of(2 * j));
#pragma unroll
          for (int kk = 0; kk < DP / 16; ++kk) {
            const uint32_t off = (uint32_t)(kk / 4) * (kKeys * 128) + (uint32_t)(kk % 4) * 32;
            umma_f16_warp(s_col, umma_desc_at(q_desc, off), umma_desc_at(b, off), kIdQK, kk > 0);
            if (kk == DP / 16 - kEarly && pass) pass_turn();
          }
          umma_commit_warp(&s_full[x]);
        };
        wait_load(0);
        if (nt > 0) {
          wait(&q_full[x], 0);
          tmem_fence_after_sync();
          if (ok) qk(0, false);
        }
        release(0);
        for (int j = 0; j < n && ok; ++j) {
          wait_load(2 * j + 1);
          if (j + 1 < n) wait_load(2 * j + 2);
          if (x == 1 || j > 0) wait(&turn[x], (uint32_t)(x == 1 ? j : j - 1) & 1u);
          if (j < nt) wait(&p_full[2 * x], (uint32_t)j & 1u);
          tmem_fence_after_sync();
          if (!ok) break;
          if (j < nt) {
            const uint64_t b = umma_desc_at(v_desc, stage_of(2 * j + 1));
#pragma unroll
            for (int kk = 0; kk < kKeys / 16; ++kk) {
              if (kk == kPart / 16) {
                wait(&p_full[2 * x + 1], (uint32_t)j & 1u);
                tmem_fence_after_sync();
              }
              umma_f16_ta_warp(o_col, s_col + kk * 8, umma_desc_at(b, kk * 2048), kIdPV,
                               (j > 0 || kk > 0) ? 1u : 0u);
            }
            if (j == nt - 1) umma_commit_warp(&o_full[x]);
            if (j + 1 < nt) qk(j + 1, true);  // over P (j): a warp's MMAs run in order
            else pass_turn();
          } else {
            pass_turn();
          }
          release(2 * j + 1);
          if (j + 1 < n) release(2 * j + 2);
        }
        umma_commit_warp(mma_done);
        mbar_drain(mma_done, 0);  // every MMA is done before tensor memory is freed
      }
    } else {
      // ---- V tiles with masked keys ----------------------------------------------
      const int ct = tid - kCleanWarp * 32;
      bool ok = true;
      for (int j = first_masked; j < n; ++j) {
        const int i = 2 * j + 1;
        if (ok && !mbar_wait_bounded(&raw_full[j - first_masked], 0, err)) {
          record_error(err, kDevWaitTimeout);
          ok = false;
        }
        if (ok) {
          uint8_t* tile = smem + C::kOffKV + (i % C::kStages) * C::kTileBytes;
          const int valid = min(lk - j * kKeys, kKeys);
          for (int r = ct; r < C::kChunks * kKeys; r += kCleaners) {  // a 128-byte row each
            const int key = r % kKeys;
            uint4* row = reinterpret_cast<uint4*>(tile + r * 128);
            if (key >= valid) {
#pragma unroll
              for (int u = 0; u < 8; ++u) row[u] = make_uint4(0, 0, 0, 0);
              continue;
            }
            uint4 w[8];
            uint32_t any = 0u;
#pragma unroll
            for (int u = 0; u < 8; ++u) w[u] = row[(u + r) & 7];  // lanes on different banks
#pragma unroll
            for (int u = 0; u < 8; ++u)
              any |= times_zero(w[u].x, T()) | times_zero(w[u].y, T()) |
                     times_zero(w[u].z, T()) | times_zero(w[u].w, T());
            if ((any & 0x7fff7fffu) == 0u) continue;  // every value finite
#pragma unroll
            for (int u = 0; u < 8; ++u)
              row[(u + r) & 7] = make_uint4(w[u].x & ~nonfinite_mask(w[u].x, T()),
                                            w[u].y & ~nonfinite_mask(w[u].y, T()),
                                            w[u].z & ~nonfinite_mask(w[u].z, T()),
                                            w[u].w & ~nonfinite_mask(w[u].w, T()));
            atomicOr(&s_flags[(j - first_masked) * 4 + key / 32], 1u << (key & 31));
          }
          fence_proxy_async_smem();  // an MMA operand
        }
        named_barrier(1, kCleaners);
        if (ct == 0) mbar_arrive(&kv_full[i % C::kStages]);
      }
    }
    } else {
      registers_up<200>();
      // ---- softmax and epilogue: thread = row ---------------------------------------
      const int x = warp >> 2;
      const int row = tid & 127;
      const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
      const uint32_t s_addr = tmem + lanes + C::kSCol + x * 128;
      const uint32_t o_addr = tmem + lanes + C::kOCol + x * 128;
      const int tok = t0 + x * p.tile_tokens + row / p.group;  // in the sequence
      const bool valid = row < p.tile_tokens * p.group && tok < lq;
      // keys below `limit` are seen
      const int limit = valid ? (p.causal ? min(tok + shift + 1, lk) : lk) : 0;
      float m = -INFINITY, l = 0.0f;
      const int nt = n_tiles[x];
      bool ok = true;
      for (int j = 0; j < nt; ++j) {
        if (ok && !mbar_wait_short(&s_full[x], (uint32_t)j & 1u, err)) {
          record_error(err, kDevWaitTimeout);
          ok = false;
        }
        __syncwarp();
        tmem_fence_after_sync();
        float s[kKeys];
        {
          uint32_t(&u)[kKeys] = reinterpret_cast<uint32_t(&)[kKeys]>(s);
#pragma unroll
          for (int c = 0; c < kKeys; c += 32)
            tmem_load<32>(s_addr + c, reinterpret_cast<uint32_t(&)[32]>(u[c]));
          tmem_wait_load();
        }
        const int seen = limit - j * kKeys;  // columns below this are seen
        if (j >= first_masked) {
#pragma unroll
          for (int c = 0; c < kKeys; ++c) s[c] = c < seen ? s[c] : -INFINITY;
        }
        float tm[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) tm[e] = s[e];
#pragma unroll
        for (int c = 8; c < kKeys - 8; c += 16)
#pragma unroll
          for (int e = 0; e < 8; ++e) tm[e] = max3_nan(tm[e], s[c + e], s[c + e + 8]);
#pragma unroll
        for (int e = 0; e < 8; e += 2) tm[e] = max3_nan(tm[e], tm[e + 1], s[kKeys - 8 + e]);
        const float t = max3_nan(
            max3_nan(tm[0], tm[2], s[kKeys - 7]), max3_nan(tm[4], tm[6], s[kKeys - 5]),
            max3_nan(s[kKeys - 3], s[kKeys - 1], tm[0]));
        // move the maximum where it grew by more than 2^kLazy (or from -inf);
        // each row by its own scores, so that its bits do not depend on others
        const bool move =
            valid && t > m && (m == -INFINITY || (t - m) * p.scale_log2 > kLazy);
        if (__any_sync(0xffffffffu, move)) {
          const float alpha = move ? exp2_approx((m - t) * p.scale_log2) : 1.0f;
          if (move) m = t;
          l *= alpha;
          if (j > 0) {
#pragma unroll
            for (int c = 0; c < DP; c += 32) {
              uint32_t o[32];
              tmem_load<32>(o_addr + c, o);
              tmem_wait_load();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_store<32>(o_addr + c, o);
            }
          }
        }
        // a NaN score makes the whole row NaN
        const float ms = t != t ? t : (m == -INFINITY ? 0.0f : m * p.scale_log2);
        const uint64_t scale2 = f32x2(p.scale_log2, p.scale_log2), ms2 = f32x2(-ms, -ms);
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int c = 0; c < kKeys; c += 32) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float2 v = unpack_f32x2(fma_f32x2(f32x2(s[c + e], s[c + e + 1]), scale2, ms2));
            v.x = exp2_approx(v.x);
            v.y = exp2_approx(v.y);
            sum[(e / 2) & 1] = add_f32x2(sum[(e / 2) & 1], f32x2(v.x, v.y));
            pk[e / 2] = pack2(v.x, v.y, T());
          }
          tmem_store<16>(s_addr + c / 2, pk);
          if (c + 32 == kPart || c + 32 == kKeys) {  // P V can start (and end)
            tmem_wait_store();
            tmem_fence_before_sync();
            mbar_arrive(&p_full[2 * x + (c + 32 == kKeys)]);
          }
        }
        const float2 l2 = unpack_f32x2(add_f32x2(sum[0], sum[1]));
        l += l2.x + l2.y;
      }
      if (nt > 0) {
        if (ok && !mbar_wait_bounded(&o_full[x], 0, err)) record_error(err, kDevWaitTimeout);
        __syncwarp();
        tmem_fence_after_sync();
      }
      const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
      uint32_t flags = 0u;
      for (int f = 0; f < kMaskedTiles * 4; ++f) flags |= s_flags[f];
      const int64_t out_row = ((int64_t)(q0 + tok) * p.heads + kvh * p.group + row % p.group);
      T* out = static_cast<T*>(p.out) + out_row * p.dim;
#pragma unroll
      for (int c = 0; c < DP; c += 32) {
        uint32_t o[32];
        if (nt > 0) {
          tmem_load<32>(o_addr + c, o);
          tmem_wait_load();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0u;
        }
        if (!valid) continue;
        float f[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) f[e] = l == 0.0f ? 0.0f : __uint_as_float(o[e]) * inv;
        if (flags != 0u) {  // non-finite values of keys that this row sees
          for (int k = 0; k < kMaskedTiles * kKeys; ++k) {
            const int key = first_masked * kKeys + k;
            if (!(s_flags[k / 32] >> (k & 31) & 1u) || key >= limit) continue;
            const T* vr = static_cast<const T*>(p.v) + (int64_t)(k0 + key) * p.v_tok +
                          (int64_t)kvh * p.v_head + c;
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const float v = c + e < p.dim ? widen(vr[e]) : 0.0f;
              if (!isfinite(v)) f[e] += v;
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 32; e += 8)
          if (c + e < p.dim)
            *reinterpret_cast<uint4*>(out + c + e) =
                make_uint4(pack2(f[e], f[e + 1], T()), pack2(f[e + 2], f[e + 3], T()),
                           pack2(f[e + 4], f[e + 5], T()), pack2(f[e + 6], f[e + 7], T()));
      }
      if (valid && p.lse != nullptr)
        p.lse[out_row] = l == 0.0f ? -INFINITY : fmaf(m, p.scale, logf(l));
    }
  }
  tmem_fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

// [tokens, heads, dim] with token and head strides (elements, multiples of
// 8) as (channel, head, token); boxes of 64 channels x box_heads x box_tokens.
// Channels past `dim` and tokens past the end load as zero.
bool make_map(CUtensorMap* map, const void* base, int bf16, int dim, int heads, int64_t tokens,
              int64_t tok_stride, int64_t head_stride, int box_heads, int box_tokens) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return false;
  cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)tokens};
  cuuint64_t strides[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)tok_stride * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tokens};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r =
      fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
         const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS;
}

template <typename T, int DP>
int launch_prefill_t(const PrefillArgs& a, cudaStream_t stream) {
  using C = PreCfg<DP>;
  const int bf16 = a.dtype == 2;
  PreParams p;
  p.cu_q = a.cu_q;
  p.cu_k = a.cu_k;
  p.out = a.out;
  p.lse = a.lse;
  p.v = a.v;
  p.v_tok = a.v_token_stride;
  p.v_head = a.v_head_stride;
  p.num_seqs = a.num_seqs;
  p.total_q = (int)a.total_q;
  p.total_k = (int)a.total_k;
  p.heads = a.heads;
  p.kv_heads = a.kv_heads;
  p.group = a.heads / a.kv_heads;
  p.dim = a.dim;
  p.tile_tokens = kRows / p.group;
  p.scale = a.sm_scale;
  p.scale_log2 = a.sm_scale * kLog2e;
  p.causal = a.causal ? 1 : 0;
  CUtensorMap mq, mk, mv;
  // without keys the key maps are never used, but a map needs memory
  const bool none = a.total_k == 0;
  if (!make_map(&mq, a.q, bf16, a.dim, a.heads, a.total_q, a.q_token_stride, a.q_head_stride,
                p.group, p.tile_tokens) ||
      !make_map(&mk, none ? a.q : a.k, bf16, a.dim, none ? a.heads : a.kv_heads,
                none ? a.total_q : a.total_k, none ? a.q_token_stride : a.k_token_stride,
                none ? a.q_head_stride : a.k_head_stride, 1, kKeys) ||
      !make_map(&mv, none ? a.q : a.v, bf16, a.dim, none ? a.heads : a.kv_heads,
                none ? a.total_q : a.total_k, none ? a.q_token_stride : a.v_token_stride,
                none ? a.q_head_stride : a.v_head_stride, 1, kKeys)) {
    set_error("cuTensorMapEncodeTiled failed for q, k or v");
    return kCudaError;
  }
  auto kern = prefill_kernel<T, DP>;
  static std::atomic<uint64_t> done{0};
  allow_shared_memory(reinterpret_cast<const void*>(kern), C::kSmemBytes, done);
  // pairs of row tiles: at most this many over all sequences (and the rest)
  const int span = 2 * p.tile_tokens;
  const int64_t pairs = a.total_q / span + std::min<int64_t>(a.num_seqs + 1, a.total_q);
  kern<<<(unsigned)(pairs * a.kv_heads), kPreThreads, C::kSmemBytes, stream>>>(
      mq, mk, mv, p, device_error_word());
  return kOk;
}

}  // namespace

int launch_prefill(const PrefillArgs& a, cudaStream_t stream) {
  if (a.total_q == 0) return kOk;
  int rc;
  if (a.dtype == 1)
    rc = a.dim <= 64 ? launch_prefill_t<__half, 64>(a, stream)
                     : launch_prefill_t<__half, 128>(a, stream);
  else
    rc = a.dim <= 64 ? launch_prefill_t<__nv_bfloat16, 64>(a, stream)
                     : launch_prefill_t<__nv_bfloat16, 128>(a, stream);
  if (rc != kOk) return rc;
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_error(std::string("prefill launch failed: ") + cudaGetErrorString(e));
    return kCudaError;
  }
  return kOk;
}

}  // namespace pkv
