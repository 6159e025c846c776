// Attention over packed prompts: out[i] = sum_j softmax_j(scale q_i . k_j) v_j
// over the keys j of token i's sequence, causal from the sequences' ends
// (j <= i + Lk - Lq), grouped heads, fp16 or bf16 with fp32 accumulators.
//
// An item of work is two row tiles of 128 rows of one KV head (one row tile in calls
// that would leave half of the SMs without); one CTA per SM takes items until none
// is left.  A row is a (token, query head of the group) pair, so the G heads of a
// group share every K / V tile that is loaded.  Keys come in tiles of 128 tokens;
// per row tile
//   S = Q K^T    tcgen05 kind::f16, 128 x 128, K-major A and B from shared
//                memory, S in 128 columns of tensor memory;
//   P = exp2(scale log2e (S - m)), one thread per row, written back over S as
//                16-bit values;
//   O += P V     A = P from tensor memory, B = the V tile read MN-major.
// The two row tiles alternate: while the softmax warps of one turn S into P,
// the tensor cores work for the other.
//
// P has 16 bits because the second product has: B is V as it was given, and A is of
// B's type.  The denominator sums the unrounded values.  Outputs of mixed signs are
// then off by 3.0e-4 (fp16) or 2.3e-3 (bf16) of their root mean square, where rounding
// the output alone leaves 2.1e-4 and 1.7e-3; P as two 16-bit numbers would be
// half as many products again and 64 more columns of stores a row.
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
//
// What bounds it: 8,192 tokens, 32 query heads of 8 KV heads, causal, head_dim
// 128 are 550 GFLOP (323 us at the cuBLAS rate) and took 466 us at best
// (1.18 PFLOP/s), 515 to 550 us in a long run, where the card's power limit
// lowers the clock to about 1.67 GHz; without the mask 984 us for 1,100 GFLOP.  The
// tensor pipe is half busy; a row tile's step is a chain -- product, softmax,
// second half of the softmax beside the first half of P V, P V -- and two row
// tiles (at head_dim 128 tensor memory holds no third) fill each other's gaps only
// in part.  16 packed prompts of 17 to 900 tokens: 92 us, of which 22 steps an SM
// are about 47 us, and the rest its seven items' own starts and ends.  64 or 128
// channels are multiplied: 8,192 tokens of head_dim 64 take 423 us (floor 162), of 32
// as much (81), of 80 and 96 458 us (202 and 242).  2,000 prompts of 1 to 8 tokens
// take 1.8 ms: 16,000 items, each found by a search among the sequences.
// Measured on the way, at 8,192 tokens: one thread issuing from its own branch
// 647 us, a converged warp with one elected lane 577 us, a warp per row tile in
// strict turns 505 us (the two unordered: slower than one; P handed over in
// halves is part of that).  A part of the exponentials as polynomials on the FMA
// units helped the first versions (with the register split, packed scaling and
// three-way maxima 798 -> 647 us) and is slower now.
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
constexpr int kConsumerWarps = 8 + 2 + kCleaners / 32;  // of an item
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 8.0f;   // log2 growth of a row maximum that moves it
constexpr int kPart = 64;        // keys of P that are handed over first
constexpr int kEarly = 4;        // MMAs left of a step when the turn is passed on
constexpr int kMaskedTiles = 4; // tiles with masked keys per CTA: 256 tokens span at most 3
// The tensor cores cut off the bits that an fp32 sum cannot hold: O loses up to
// 8.4e-7 of a sum of one sign in a tile (measured: 8.2e-7; fp16, 131,072 keys: 8.4e-4,
// twice the step of a 16-bit output).  Every so many tiles O is therefore added to a
// sum of its own, rounded to nearest, and started anew.  With head_dim up to 64 the
// sum has columns of tensor memory; above that it is in the call's workspace.  Calls
// without so many keys have a kernel without that (LONG = false), since the softmax
// loop has no register to spare: 16 packed prompts take 92 us, 94.5 with it.  600
// tokens behind 16,400 keys, 32 / 8 heads, take 265 us, 257 summed at once.
constexpr int kStretch = 128;

template <int DP>
struct PreCfg {
  static constexpr int kChunks = DP / 64;               // 128-byte column chunks
  static constexpr int kTileBytes = kKeys * DP * 2;     // a K, V or Q tile
  static constexpr int kStages = DP == 128 ? 4 : 8;     // K / V ring
  static constexpr int kStageBytes = kRows * 128;       // output staging: 64 channels a tile
  static constexpr int kOffQ = 0;                       // two Q tiles
  static constexpr int kOffKV = 2 * kTileBytes;
  static constexpr int kOffOut = kOffKV + kStages * kTileBytes;
  static constexpr int kOffBar = kOffOut + 2 * kStageBytes;
  static constexpr int kBars = 2 * kStages + 2 + 2 + 2 + 4 + 2 + kMaskedTiles + 2 + 4 + 2;
  static constexpr int kOffMisc = kOffBar + kBars * 8;  // 16-byte aligned
  static constexpr int kSmemBytes = kOffMisc + 288 + 1024;
  static constexpr int kSCol = 0;                       // S / P of the two tiles
  static constexpr int kOCol = 256;
  static_assert(kBars % 2 == 0 && kSmemBytes <= 227 * 1024, "shared memory");
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
  int item_tiles;  // row tiles of an item: 2, or 1 in calls of few items
  float scale_log2, scale;
  int causal;
  // LONG: per slot and row tile [DP / 4][128 rows], O of earlier stretches (DP = 128)
  float4* sums;
  int* ticket;  // zero: the next CTA's slot of sums
  int slots;
};

struct PreWork {
  int q0, lq, k0, lk;  // the sequence's rows in the packed tensors
  int t0;              // first token (in the sequence) of row tile 0
};

// An item of work: two row tiles of a sequence, one KV head, and the key tiles
// that they see.
struct PreItem {
  PreWork at;
  int kvh;
  int n_tiles[2];    // key tiles of each row tile: up to the last key of its last token
  int n;             // the larger; 0: nothing to load
  int first_masked;  // tiles from here on hold keys that some row does not see
  int kind;          // kNone: past the end of the work, kSome, kStop: the CTA is done
  int check;         // the grid's first item: its CTA checks the sequences' ends
};
enum ItemKind { kNone = 0, kSome = 1, kStop = 2 };

__device__ __forceinline__ void count_tiles(const PreParams& p, PreItem& w) {
  const int shift = w.at.lk - w.at.lq;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int first = w.at.t0 + x * p.tile_tokens;
    const int last = min(first + p.tile_tokens, w.at.lq) - 1;
    const int keys =
        first < w.at.lq && x < p.item_tiles ? (p.causal ? min(max(last + shift + 1, 0), w.at.lk) : w.at.lk) : 0;
    w.n_tiles[x] = (keys + kKeys - 1) / kKeys;
  }
  w.n = max(w.n_tiles[0], w.n_tiles[1]);
  w.first_masked = (p.causal ? min(max(w.at.t0 + shift + 1, 0), w.at.lk) : w.at.lk) / kKeys;
}

// Asks the hardware for a CTA of this grid that has not started yet (16 bytes
// of answer, completed on bar), and reads the answer: its block index, or -1.
__device__ __forceinline__ void request_block(void* answer, uint64_t* bar) {
  asm volatile(
      "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], "
      "[%1];" ::"r"(smem_u32(answer)),
      "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ int granted_block(const void* answer) {
  uint32_t got, x;
  asm volatile(
      "{\n\t.reg .b128 r;\n\t.reg .pred p;\n\t.reg .b32 y, z, w;\n\t"
      "ld.shared.b128 r, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, y, z, w}, r;\n\t}"
      : "=r"(got), "=r"(x)
      : "r"(smem_u32(answer))
      : "memory");
  return got ? (int)x : -1;
}

// Sequence and token range of pair `pair` (of item_tiles * tile_tokens tokens).  Pairs
// are numbered sequence by sequence, the last pair of a sequence first: under
// a causal mask it is the longest, and long work should start early.  The rows
// behind the last sequence and those in front of the first form two more
// sequences without keys (zeros).
// One warp; false when `pair` is past the end.
__device__ __forceinline__ bool find_work(const PreParams& p, int pair, PreWork& w) {
  const int lane = threadIdx.x & 31;
  const int span = p.item_tiles * p.tile_tokens;
  int base = 0;
  int q_end = 0;  // the largest end up to the last 32 that fell
  const int front = p.num_seqs + 1;
  for (int s0 = 0; s0 <= front; s0 += 32) {
    const int s = s0 + lane;
    int q0 = 0, q1 = 0;
    if (s <= front) {
      q0 = s < front ? min(max(p.cu_q[s], 0), p.total_q) : 0;
      q1 = s == p.num_seqs ? p.total_q : min(max(p.cu_q[s < front ? s + 1 : 0], 0), p.total_q);
    }
    // An entry below an earlier one counts as the largest before it: sequences then
    // share no row, and all of them together have no more items than the grid.
    const bool falls = q1 < q0 || (lane == 0 && s < front && q0 < q_end);
    if (__any_sync(0xffffffffu, falls)) {
      int most = max(max(q0, q1), q_end);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, most, o);
        if (lane >= o) most = max(most, x);
      }
      const int before = __shfl_up_sync(0xffffffffu, most, 1);
      if (s < front) {
        q0 = lane > 0 ? before : max(q0, q_end);
        q1 = most;
      }
      q_end = __shfl_sync(0xffffffffu, q1, 31);
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
      w.k0 = w.lk = 0;
      if (s0 + src < p.num_seqs) {  // (keys may be shared: they are only read)
        w.k0 = min(max(p.cu_k[s0 + src], 0), p.total_k);
        w.lk = min(max(p.cu_k[s0 + src + 1], w.k0), p.total_k) - w.k0;
      }
      return true;
    }
    base += total;
  }
  return false;
}

// Reports cu_seqlens that do not ascend within the tensors, every entry, by `n`
// threads.  (Apart from find_work, which stops at the pair that it looks for.)
__device__ __forceinline__ void check_seqlens(const PreParams& p, int thread, int n, int* err) {
  bool bad = false;
  for (int s = thread; s <= p.num_seqs; s += n) {
    const int q = p.cu_q[s], k = p.cu_k[s];
    bad |= q < (s > 0 ? p.cu_q[s - 1] : 0) || q > p.total_q;
    bad |= k < (s > 0 ? p.cu_k[s - 1] : 0) || k > p.total_k;
  }
  if (bad) record_error(err, kDevBadSeqlens);
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

template <typename T, int DP, bool LONG>
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
  uint64_t* q_full = kv_empty + C::kStages;  // per row tile, as the next four
  uint64_t* q_empty = q_full + 2;
  uint64_t* s_full = q_empty + 2;
  uint64_t* p_full = s_full + 2;  // [row tile][part of P]
  uint64_t* o_full = p_full + 4;
  uint64_t* raw_full = o_full + 2;  // V tiles with masked keys, before they are cleaned
  uint64_t* turn = raw_full + kMaskedTiles;  // per row tile
  uint64_t* item_full = turn + 2;            // two items in flight
  uint64_t* item_empty = item_full + 2;
  uint64_t* mma_done = item_empty + 2;
  uint64_t* block_full = mma_done + 1;
  uint8_t* answer = smem + C::kOffMisc;  // of request_block
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + C::kOffMisc + 16);
  PreItem* s_item = reinterpret_cast<PreItem*>(smem + C::kOffMisc + 32);            // [2]
  uint32_t* s_flags = reinterpret_cast<uint32_t*>(smem + C::kOffMisc + 32 + 96);    // [2][tile][4]
  volatile int* s_fail = reinterpret_cast<int*>(smem + C::kOffMisc + 256);  // [group][item parity]
  // O is taken before tile j > 0 where j & s_take[0] = 0; s_take[1]: the CTA's slot
  volatile int* s_take = reinterpret_cast<int*>(smem + C::kOffMisc + 280);
  static_assert(sizeof(PreItem) <= 48 && kMaskedTiles == 4, "layout");

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == kLoadWarp * 32) {
    prefetch_tensormap(&map_q);
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 2);  // both MMA warps
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[2 * i], 128);
      mbar_init(&p_full[2 * i + 1], 128);
      mbar_init(&o_full[i], 1);
      mbar_init(&turn[i], 1);
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], kConsumerWarps);
    }
    for (int i = 0; i < kMaskedTiles; ++i) mbar_init(&raw_full[i], 1);
    mbar_init(mma_done, 2);
    mbar_init(block_full, 1);
    mbar_fence_init();
    if constexpr (LONG) {
      const int slot = DP > 64 ? atomicAdd(p.ticket, 1) : 0;
      // (there are as many slots as SMs, and a CTA an SM)
      s_take[0] = slot < p.slots ? kStretch - 1 : 0x7fffffff;
      s_take[1] = slot;
    }
  }
  if (tid < 6) s_fail[tid] = 0;
  if (warp == kMmaWarp) tmem_alloc(s_tmem, 512);
  tmem_fence_before_sync();
  __syncthreads();
  tmem_fence_after_sync();
  const uint32_t tmem = *s_tmem;

  // ok: false in a thread whose wait gave up (bounded; then every wait of the grid
  // gives up at once).  Such a thread goes through the rest of its item without
  // waiting and without storing results, so that warps and named barriers stay
  // whole, and its group leaves together at the next item.
  bool ok = true;
  auto wait = [&](uint64_t* bar, int phase) {
    if (ok && !mbar_wait_short(bar, (uint32_t)phase & 1u, err)) {
      record_error(err, kDevWaitTimeout);
      ok = false;
    }
  };
  // The K / V ring runs on over the items: load i of an item is ring use base + i.
  int base = 0;
  auto stage_of = [&](int i) { return (base + i) % C::kStages; };
  // The next item, for a group of warps that share named barrier `bar`; false:
  // leave, all of them.
  auto next_item = [&](int k, int group, int bar, int threads) {
    wait(&item_full[k & 1], k >> 1);
    volatile int* fail = &s_fail[2 * group + (k & 1)];  // a fast thread may be an item ahead
    if (!ok) *fail = 1;
    named_barrier(bar, threads);
    return !*fail && s_item[k & 1].kind != kStop;
  };
  auto item_done = [&](int k) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&item_empty[k & 1]);
  };

  if (warp >= 8) {
    // 256 x 200 + 256 x 56 = 65,536 = 512 x 128, the registers at launch
    registers_down<56>();
    if (warp == kLoadWarp) {
      // ---- items and loads ------------------------------------------------------------
      // One CTA per SM takes one item after the other: its own block's, then those
      // of blocks that have not started.  The next item's loads and its first
      // product run during this one's epilogue.
      const uint64_t once = l2_policy_evict_first(), hold = l2_policy_evict_last();
      int q_loads[2] = {0, 0}, raw_loads = 0, k = 0;
      int block = blockIdx.x;
      auto publish = [&](const PreItem& w) {
        if (k >= 2) wait(&item_empty[k & 1], (k >> 1) - 1);
        if (lane < kMaskedTiles * 4) s_flags[(k & 1) * kMaskedTiles * 4 + lane] = 0u;
        if (lane == 0) s_item[k & 1] = w;
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_full[k & 1]);
      };
      auto ask = [&]() {
        mbar_arrive_expect_tx(block_full, 16);
        request_block(answer, block_full);
      };
      PreItem w = {};
      for (; block >= 0 && ok; ++k) {
        w.kvh = block % p.kv_heads;
        w.kind = find_work(p, block / p.kv_heads, w.at) ? kSome : kNone;
        w.check = block == 0;
        if (w.kind == kNone) w.n = w.n_tiles[0] = w.n_tiles[1] = w.first_masked = 0;
        else count_tiles(p, w);
        publish(w);
        if (lane == 0 && w.n > 0) {
          auto load_kv = [&](int i) {
            const int st = stage_of(i), j = i / 2, use = (base + i) / C::kStages;
            if (use > 0) wait(&kv_empty[st], use - 1);
            if (!ok) return;
            // a V tile with masked keys goes through the cleaning warps, which
            // complete kv_full in the load's place
            uint64_t* bar = (i & 1) && j >= w.first_masked
                                ? &raw_full[raw_loads++ % kMaskedTiles] : &kv_full[st];
            mbar_arrive_expect_tx(bar, C::kTileBytes);
            for (int c = 0; c < C::kChunks; ++c)
              tma_load_3d(smem + C::kOffKV + st * C::kTileBytes + c * kKeys * 128,
                          (i & 1) ? &map_v : &map_k, bar, c * 64, w.kvh, w.at.k0 + j * kKeys, hold);
          };
          int done = 0;
          load_kv(done++);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if (w.n_tiles[x] == 0) continue;
            if (q_loads[x] > 0) wait(&q_empty[x], q_loads[x] - 1);
            if (!ok) continue;
            mbar_arrive_expect_tx(&q_full[x], (uint32_t)(C::kChunks * p.tile_tokens * p.group * 128));
            for (int c = 0; c < C::kChunks; ++c)
              tma_load_3d(smem + C::kOffQ + x * C::kTileBytes + c * kRows * 128, &map_q, &q_full[x],
                          c * 64, w.kvh * p.group, w.at.q0 + w.at.t0 + x * p.tile_tokens, once);
            ++q_loads[x];
          }
          while (done < 2 * w.n && ok) {
            // early enough to be answered by the end of the loads, late enough to
            // leave the work to the CTA that is free first
            if (done == max(2 * w.n - 2 * C::kStages, 1)) ask();
            load_kv(done++);
          }
          base += done;
        }
        if (lane == 0) {
          if (w.n == 0) ask();
          wait(block_full, k);
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        block = ok ? granted_block(answer) : -1;
        fence_proxy_async_smem();  // the answer is read before the next one is written
        __syncwarp();
      }
      w.kind = kStop;
      if (ok) publish(w);
      // no copy and no release outlives the CTA
      if (lane == 0) {
        drain_ring(kv_full, C::kStages, base);
        drain_ring(kv_empty, C::kStages, base);
        for (int f = max(raw_loads - kMaskedTiles, 0); f < raw_loads; ++f)
          mbar_drain(&raw_full[f % kMaskedTiles], (uint32_t)(f / kMaskedTiles) & 1u);
#pragma unroll
        for (int x = 0; x < 2; ++x)
          if (q_loads[x] > 0) {
            mbar_drain(&q_full[x], (uint32_t)(q_loads[x] - 1) & 1u);
            mbar_drain(&q_empty[x], (uint32_t)(q_loads[x] - 1) & 1u);
          }
      }
    } else if (warp < kCleanWarp) {
      // ---- MMA issue: a warp for each row tile, in strict turns -----------------------
      // A wait that follows MMAs in a warp's queue returns only when they have
      // been taken up, so with one warp for both tiles the tensor cores ran dry at
      // every wait.  With two, one waits while the other's MMAs run; the turn is
      // passed on before a step's last MMAs, to cover its own latency.  Without
      // turns the tiles fall into step, and first their exponentials compete, then
      // their products.
      constexpr uint32_t kIdQK = umma_f16_idesc(kBf16, 0, kRows, kKeys);
      constexpr uint32_t kIdPV = umma_f16_idesc(kBf16, 1, kRows, DP);
      const int x = warp - kMmaWarp;
      const uint32_t kv = smem_u32(smem + C::kOffKV);
      const uint64_t q_desc =
          umma_sw128_desc(smem_u32(smem + C::kOffQ + x * C::kTileBytes), 16, 1024);
      const uint64_t k_desc = umma_sw128_desc(kv, 16, 1024);
      const uint64_t v_desc = umma_sw128_desc(kv, kKeys * 128, 1024);
      const uint32_t s_col = tmem + C::kSCol + x * 128, o_col = tmem + C::kOCol + x * 128;
      // both warps release a stage, each after it saw the load
      auto release = [&](int i) { umma_commit_warp(&kv_empty[stage_of(i)]); };
      auto pass_turn = [&]() {
        if (lane == 0) mbar_arrive(&turn[x ^ 1]);
        __syncwarp();
      };
      auto qk = [&](int j, bool last, bool pass) {
        const uint64_t b = umma_desc_at(k_desc, (uint32_t)stage_of(2 * j) * C::kTileBytes);
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          const uint32_t off = (uint32_t)(kk / 4) * (kKeys * 128) + (uint32_t)(kk % 4) * 32;
          umma_f16_warp(s_col, umma_desc_at(q_desc, off), umma_desc_at(b, off), kIdQK, kk > 0);
          if (kk == DP / 16 - kEarly && pass) pass_turn();
        }
        umma_commit_warp(&s_full[x]);
        if (last) umma_commit_warp(&q_empty[x]);
      };
      int q_uses = 0, p_uses = 0, steps = 0;
      const int take = LONG ? s_take[0] : 0x7fffffff;
      // a warp's lanes give up together
      auto wait_warp = [&](uint64_t* bar, int phase) {
        wait(bar, phase);
        ok = __all_sync(0xffffffffu, ok);
      };
      auto wait_load_warp = [&](int i) {
        wait_warp(&kv_full[stage_of(i)], (base + i) / C::kStages);
      };
      for (int k = 0;; ++k) {
        wait_warp(&item_full[k & 1], k >> 1);
        if (!ok) break;
        const PreItem* item = &s_item[k & 1];
        const int nt = x ? item->n_tiles[1] : item->n_tiles[0], n = item->n;
        const bool stop = item->kind == kStop;
        item_done(k);
        if (stop) break;
        if (n == 0) continue;
        wait_load_warp(0);
        if (nt > 0) {
          wait_warp(&q_full[x], q_uses++);
          tmem_fence_after_sync();
          if (ok) qk(0, nt == 1, false);  // S is free: the last P V ran before
        }
        release(0);
        for (int j = 0; j < n && ok; ++j, ++steps) {
          wait_load_warp(2 * j + 1);
          if (j + 1 < n) wait_load_warp(2 * j + 2);
          if (x == 1 || steps > 0) wait_warp(&turn[x], x == 1 ? steps : steps - 1);
          // (P of a new item also says that its rows' last results are read from O)
          if (j < nt) wait_warp(&p_full[2 * x], p_uses);
          tmem_fence_after_sync();
          if (!ok) break;
          if (j < nt) {
            const uint64_t b = umma_desc_at(v_desc, (uint32_t)stage_of(2 * j + 1) * C::kTileBytes);
#pragma unroll
            for (int kk = 0; kk < kKeys / 16; ++kk) {
              if (kk == kPart / 16) {
                wait_warp(&p_full[2 * x + 1], p_uses);
                tmem_fence_after_sync();
                if (!ok) break;
              }
              umma_f16_ta_warp(o_col, s_col + kk * 8, umma_desc_at(b, kk * 2048), kIdPV,
                               ((j & take) != 0 || kk > 0) ? 1u : 0u);
            }
            if (!ok) break;
            ++p_uses;
            if (j == nt - 1) umma_commit_warp(&o_full[x]);
            if (j + 1 < nt) qk(j + 1, j + 2 == nt, true);  // over P (j): a warp's MMAs run in order
            else pass_turn();
          } else {
            pass_turn();
          }
          release(2 * j + 1);
          if (j + 1 < n) release(2 * j + 2);
        }
        base += 2 * n;
      }
      umma_commit_warp(mma_done);
      mbar_drain(mma_done, 0);  // every MMA is done before tensor memory is freed
    } else {
      // ---- V tiles with masked keys ----------------------------------------------
      const int ct = tid - kCleanWarp * 32;
      int cleaned = 0;
      for (int k = 0; next_item(k, 2, 1, kCleaners); ++k) {
        const PreItem& w = s_item[k & 1];
        const int n = w.n, first_masked = w.first_masked, lk = w.at.lk;
        uint32_t* flags = s_flags + (k & 1) * kMaskedTiles * 4;
        if (w.check) check_seqlens(p, ct, kCleaners, err);  // beside the first loads
        for (int j = first_masked; j < n; ++j, ++cleaned) {
          wait(&raw_full[cleaned % kMaskedTiles], cleaned / kMaskedTiles);
          if (ok) {
            uint8_t* tile = smem + C::kOffKV + stage_of(2 * j + 1) * C::kTileBytes;
            const int valid = min(lk - j * kKeys, kKeys);
            for (int r = ct; r < C::kChunks * kKeys; r += kCleaners) {  // a 128-byte row each
              const int key = r % kKeys;
              uint4* row = reinterpret_cast<uint4*>(tile + r * 128);
              if (key >= valid) {
#pragma unroll
                for (int u = 0; u < 8; ++u) row[u] = make_uint4(0, 0, 0, 0);
                continue;
              }
              uint32_t any = 0u;
#pragma unroll
              for (int u = 0; u < 8; ++u) {
                const uint4 v = row[(u + r) & 7];  // lanes on different banks
                any |= times_zero(v.x, T()) | times_zero(v.y, T()) | times_zero(v.z, T()) |
                       times_zero(v.w, T());
              }
              if ((any & 0x7fff7fffu) == 0u) continue;  // every value finite
              for (int u = 0; u < 8; ++u) {
                uint4 v = row[u];
                v.x &= ~nonfinite_mask(v.x, T());
                v.y &= ~nonfinite_mask(v.y, T());
                v.z &= ~nonfinite_mask(v.z, T());
                v.w &= ~nonfinite_mask(v.w, T());
                row[u] = v;
              }
              atomicOr(&flags[(j - first_masked) * 4 + key / 32], 1u << (key & 31));
            }
            fence_proxy_async_smem();  // an MMA operand
          }
          named_barrier(1, kCleaners);
          if (ct == 0) mbar_arrive(&kv_full[stage_of(2 * j + 1)]);
        }
        base += 2 * n;
        item_done(k);
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
    const int row_tok = row / p.group;
    const int take = LONG ? s_take[0] : 0x7fffffff;
    const uint32_t o2_addr = o_addr + 64;  // of head_dim up to 64
    auto sums = [&]() {  // the row's, 4 channels every 128
      return p.sums + ((int64_t)s_take[1] * 2 + x) * (DP / 4) * kRows + row;
    };
    const uint32_t inv_group = (65536u + p.group - 1) / p.group;  // exact below 128 * 128
    int s_uses = 0, o_uses = 0;
    for (int k = 0; next_item(k, x, 2 + x, 128); ++k) {
      // Its fields are read where they are needed: the loop below has no register
      // to spare.
      const PreItem& w = s_item[k & 1];
      if (w.kind == kNone) {
        item_done(k);
        continue;
      }
      const int nt = x ? w.n_tiles[1] : w.n_tiles[0];
      // keys below `limit` are seen; columns of tiles from `first_masked` on are tested
      const int first_masked = w.first_masked;
      int limit = 0;
      bool valid;
      {
        const int tok = w.at.t0 + x * p.tile_tokens + row_tok, lq = w.at.lq, lk = w.at.lk;
        valid = row_tok < p.tile_tokens && tok < lq && x < p.item_tiles;
        if (valid) limit = p.causal ? min(tok + lk - lq + 1, lk) : lk;
      }
      float m = -INFINITY, l = 0.0f;
      for (int j = 0; j < nt; ++j) {
        wait(&s_full[x], s_uses++);
        __syncwarp();
        tmem_fence_after_sync();
        if (LONG && j > 0 && (j & take) == 0) {  // O has the products of all tiles before j
          float4* sum = sums();
#pragma unroll 1
          for (int c = 0; c < DP; c += 16) {
            alignas(16) uint32_t o[16], was[16];
            tmem_load<16>(o_addr + c, o);
            if (j == take + 1) {
#pragma unroll
              for (int e = 0; e < 16; ++e) was[e] = 0u;
            } else if (DP == 64) {
              tmem_load<16>(o2_addr + c, was);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                *reinterpret_cast<float4*>(&was[4 * e]) = sum[(c / 4 + e) * kRows];
            }
            tmem_wait_load();
#pragma unroll
            for (int e = 0; e < 16; ++e)
              o[e] = __float_as_uint(__uint_as_float(was[e]) + __uint_as_float(o[e]));
            if (DP == 64) {
              tmem_store<16>(o2_addr + c, o);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                sum[(c / 4 + e) * kRows] = *reinterpret_cast<const float4*>(&o[4 * e]);
            }
          }
          tmem_wait_store();
        }
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
          if (j > 0) {  // seldom: small pieces, since the scores are in registers
            const bool taken = LONG && j > take;  // there is a sum
            float4* sum = sums();
#pragma unroll 1
            for (int c = 0; c < (DP == 64 && taken ? 2 * DP : DP); c += 16) {
              uint32_t o[16];
              tmem_load<16>(o_addr + c, o);  // (a sum's columns follow O's)
              tmem_wait_load();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_store<16>(o_addr + c, o);
            }
            if (DP > 64 && taken) {
#pragma unroll 1
              for (int c = 0; c < DP / 4; ++c) {
                float4 v = sum[c * kRows];
                v.x *= alpha, v.y *= alpha, v.z *= alpha, v.w *= alpha;
                sum[c * kRows] = v;
              }
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
        wait(&o_full[x], o_uses++);
        __syncwarp();
        tmem_fence_after_sync();
      }
      const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
      const uint32_t* flags = s_flags + (k & 1) * kMaskedTiles * 4;
      uint32_t flagged = 0u;
      if (first_masked < w.n)
        for (int f = 0; f < kMaskedTiles * 4; ++f) flagged |= flags[f];
      // The rows leave in whole lines, 64 channels at a time, through a buffer
      // whose 16-byte pieces are swizzled against bank conflicts.
      uint8_t* stage = smem + C::kOffOut + x * C::kStageBytes;
      uint8_t* mine = stage + row * 128;
      const int tok0 = w.at.t0 + x * p.tile_tokens;
      const int rows =
          x < p.item_tiles ? min(p.tile_tokens, max(w.at.lq - tok0, 0)) * p.group : 0;
#pragma unroll 1
      for (int c0 = 0; c0 < DP; c0 += 64) {
        named_barrier(2 + x, 128);  // the buffer is free
#pragma unroll 1
        for (int c = c0; c < c0 + 64; c += 32) {
          uint32_t o[32];
          if (nt > 0) {
            tmem_load<32>(o_addr + c, o);
            tmem_wait_load();
          }
          if (LONG && nt - 1 > take) {  // and what was taken before
            alignas(16) uint32_t was[32];
            if (DP == 64) {
              tmem_load<32>(o2_addr + c, was);
              tmem_wait_load();
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                *reinterpret_cast<float4*>(&was[4 * e]) = sums()[(c / 4 + e) * kRows];
            }
#pragma unroll
            for (int e = 0; e < 32; ++e)
              o[e] = __float_as_uint(__uint_as_float(was[e]) + __uint_as_float(o[e]));
          }
          const bool none = nt == 0 || l == 0.0f;
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint32_t r[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
              r[u] = none ? 0u : pack2(__uint_as_float(o[e + 2 * u]) * inv,
                                       __uint_as_float(o[e + 2 * u + 1]) * inv, T());
            *reinterpret_cast<uint4*>(mine + ((((c & 32) + e) / 8) ^ (row & 7)) * 16) =
                make_uint4(r[0], r[1], r[2], r[3]);
          }
        }
        if (flagged != 0u && valid) {  // non-finite values of keys that this row sees
#pragma unroll 1
          for (int i = 0; i < kMaskedTiles * kKeys; ++i) {
            const int key = first_masked * kKeys + i;
            if (!(flags[i / 32] >> (i & 31) & 1u) || key >= limit) continue;
            const T* vr = static_cast<const T*>(p.v) + (int64_t)(w.at.k0 + key) * p.v_tok +
                          (int64_t)w.kvh * p.v_head;
#pragma unroll 1
            for (int d = c0; d < min(c0 + 64, p.dim); ++d) {
              const float v = widen(vr[d]);
              if (isfinite(v)) continue;
              T* at = reinterpret_cast<T*>(mine + (((d & 63) / 8) ^ (row & 7)) * 16) + (d & 7);
              const uint32_t sum = pack2(widen(*at) + v, 0.0f, T());
              *reinterpret_cast<uint16_t*>(at) = (uint16_t)sum;
            }
          }
        }
        named_barrier(2 + x, 128);
        const int piece = row & 7;
        if (ok && c0 + piece * 8 < p.dim)
          for (int r = row >> 3; r < rows; r += 16) {
            const int rt = (int)(((uint32_t)r * inv_group) >> 16);
            const int64_t to = (int64_t)(w.at.q0 + tok0 + rt) * p.heads + w.kvh * p.group +
                               (r - rt * p.group);
            *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + to * p.dim + c0 + piece * 8) =
                *reinterpret_cast<const uint4*>(stage + r * 128 + (piece ^ (r & 7)) * 16);
          }
      }
      if (ok && valid && p.lse != nullptr)
        p.lse[(int64_t)(w.at.q0 + tok0 + row_tok) * p.heads + w.kvh * p.group + row -
              row_tok * p.group] =
            l == 0.0f ? -INFINITY : fmaf(m, p.scale, logf(l));
      item_done(k);
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

constexpr int kSumSlots = 148;  // one CTA an SM

template <typename T, int DP, bool LONG>
int launch_prefill_t(const PrefillArgs& a, void* workspace, cudaStream_t stream) {
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
  p.sums = nullptr;
  p.ticket = nullptr;
  p.slots = kSumSlots;
  if (LONG && DP > 64) {
    uint8_t* ws = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(workspace) + 255) &
                                             ~(uintptr_t)255);
    p.ticket = reinterpret_cast<int*>(ws);
    p.sums = reinterpret_cast<float4*>(ws + 256);
    cudaMemsetAsync(p.ticket, 0, sizeof(int), stream);
  }
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
  auto kern = prefill_kernel<T, DP, LONG>;
  static std::atomic<uint64_t> done{0};
  allow_shared_memory(reinterpret_cast<const void*>(kern), C::kSmemBytes, done);
  // at most so many items over so many sequences
  auto items = [&](int tiles, int64_t seqs) {
    return (a.total_q / (tiles * p.tile_tokens) + std::min(seqs, a.total_q)) * a.kv_heads;
  };
  // While half of the 148 SMs have no item, an item is one row tile: 1,500 tokens of
  // 8 heads take 30.5 us a call, 34.5 in pairs; 100 tokens behind 4,900 keys, 32 / 8
  // heads, 77.5 us and 84.6.
  p.item_tiles = items(2, (int64_t)a.num_seqs + 1) <= 148 / 2 ? 1 : 2;
  // (with the rows behind and in front of all sequences)
  kern<<<(unsigned)items(p.item_tiles, (int64_t)a.num_seqs + 2), kPreThreads, C::kSmemBytes, stream>>>(
      mq, mk, mv, p, device_error_word());
  return kOk;
}

}  // namespace

size_t prefill_workspace_size(const PrefillArgs& a) {
  if (a.total_q == 0 || a.dim <= 64 || a.total_k <= (int64_t)kStretch * kKeys) return 0;
  return 256 + 256 + (size_t)kSumSlots * 2 * kRows * 128 * sizeof(float);
}

int launch_prefill(const PrefillArgs& a, void* workspace, size_t workspace_bytes,
                   cudaStream_t stream) {
  if (a.total_q == 0) return kOk;
  if (workspace != nullptr && workspace_bytes < prefill_workspace_size(a)) {
    set_error("workspace too small for prefill_attention: need " +
              std::to_string(prefill_workspace_size(a)) + " bytes");
    return kWorkspace;
  }
  auto with = [&](auto t, auto dp) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value;
    const bool more = a.total_k > (int64_t)kStretch * kKeys;  // than one stretch
    return more && (DP == 64 || workspace != nullptr)
               ? launch_prefill_t<T, DP, true>(a, workspace, stream)
               : launch_prefill_t<T, DP, false>(a, workspace, stream);
  };
  auto with_dim = [&](auto t) {
    return a.dim <= 64 ? with(t, std::integral_constant<int, 64>{})
                       : with(t, std::integral_constant<int, 128>{});
  };
  const int rc = a.dtype == 1 ? with_dim(__half()) : with_dim(__nv_bfloat16());
  if (rc != kOk) return rc;
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_error(std::string("prefill launch failed: ") + cudaGetErrorString(e));
    return kCudaError;
  }
  return kOk;
}

}  // namespace pkv
