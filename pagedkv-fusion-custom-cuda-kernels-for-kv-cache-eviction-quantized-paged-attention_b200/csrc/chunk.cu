// Attention of new tokens over the INT8 paged cache that holds them: one token of a
// sequence, a few drafted ones, or a chunk of a prompt behind what was cached before.
//
//   out[i, h] = sum_j softmax_j(scale q[i, h] . k_j) v_j,   j <= i + L - Lq
//
// k_j and v_j are codes times the scale of their (page, head).  The codes are exact
// in fp16; the products run on the tensor cores with fp32 sums, the K scales on the
// scores and the V scales on the probabilities.
//
//   plan_kernel   one CTA (one more for chunk_tc.cu's units): the sequences' rows and
//                 lengths, checked, and where in all of the work each sequence's begins;
//   rows_kernel   a unit is 8 query rows of a KV head and its sequence's keys; each
//                 warp takes an equal share of the units' steps of 16 keys;
//   join_kernel   units that more than 8 warps share.
// Sequences of many rows go to chunk_tc.cu (kFewRows).
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>
#include <string>
#include <type_traits>

#include "cache_mma.cuh"
#include "chunk.h"
#include "pkv_internal.h"

namespace pkv {
namespace {

constexpr int kPlanThreads = 256;
constexpr int kPlanWarps = kPlanThreads / 32;

// Inclusive scans over the CTA's threads; `all` is the result over all of them.
__device__ __forceinline__ int scan_max(int v, int* shared, int* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v = max(v, x);
  }
  if (lane == 31) shared[warp] = v;
  __syncthreads();
  int front = 0, most = 0;
#pragma unroll
  for (int w = 0; w < kPlanWarps; ++w) {
    if (w < warp) front = max(front, shared[w]);
    most = max(most, shared[w]);
  }
  *all = most;
  return max(v, front);
}
__device__ __forceinline__ int64_t scan_sum(int64_t v, int64_t* shared, int64_t* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  if (lane == 31) shared[warp] = v;
  __syncthreads();
  int64_t sum = 0;
#pragma unroll
  for (int w = 0; w < kPlanWarps; ++w) {
    if (w == warp) v += sum;
    sum += shared[w];
  }
  *all = sum;
  return v;
}

__global__ void __launch_bounds__(kPlanThreads)
    plan_kernel(const PlanArgs first_plan, const PlanArgs second_plan, int plans, const ZeroArgs z,
                int* err) {
  launch_the_next();
  if ((int)blockIdx.x >= plans) {
    const int64_t per_seq = (int64_t)z.width * z.block_size, slots = per_seq * z.seqs;
    const int64_t step = (int64_t)(gridDim.x - plans) * kPlanThreads;
    for (int64_t i = (int64_t)(blockIdx.x - plans) * kPlanThreads + threadIdx.x; i < slots; i += step) {
      const int64_t s = i / per_seq;
      const int at = (int)(i - s * per_seq), page = at / z.block_size;
      if (at >= z.lens[s]) continue;
      const int phys = z.tables[s * z.width + page];
      if (phys >= 0 && (int64_t)phys < z.num_blocks)
        z.sums[(int64_t)phys * z.block_size + at - page * z.block_size] = 0;
    }
    return;
  }
  const PlanArgs p = blockIdx.x == 0 ? first_plan : second_plan;
  __shared__ int s_max[kPlanWarps];
  __shared__ int64_t s_sum[kPlanWarps];
  __shared__ int s_end[kPlanThreads];
  const int tid = threadIdx.x;
  for (int i = tid; i < p.counts; i += kPlanThreads) p.counters[i] = 0;
  const int64_t room = (int64_t)p.width * p.block_size;
  // an entry of cu below an earlier one counts as the largest before it
  const int first = p.cu[0];
  int end = min(max(first, 0), p.total_q);
  const int q_begin = end;
  bool bad = first < 0 || first > p.total_q, longer = false;
  // units of a sequence that this plan has
  const auto units_of = [&](const PlanSeq& q) {
    const int64_t rows = q.lq * (int64_t)p.group;
    const bool few = rows <= p.few_rows ||
                     (rows + 7) / 8 * p.kv_heads * (int64_t)((q.len + 15) / 16) <= p.few_steps;
    return p.which == kPlanAll || few == (p.which == kPlanFew) ? (rows + p.rows - 1) / p.rows * p.kv_heads : 0;
  };
  int64_t in_shares = 0, in_parts[2] = {};  // places
  PlanSeq q = {};
  for (int s0 = 0; s0 < p.seqs; s0 += kPlanThreads) {
    const int s = s0 + tid;
    int q1 = 0, len = 0;
    if (s < p.seqs) {
      const int c = p.cu[s + 1], given = p.lens[s];
      q1 = min(max(c, 0), p.total_q);
      bad |= c < p.cu[s] || c > p.total_q;
      longer |= given > room;
      len = (int)min((int64_t)max(given, 0), room);
    }
    int most;
    const int incl = max(scan_max(q1, s_max, &most), end);
    s_end[tid] = incl;
    __syncthreads();
    q.q0 = tid > 0 ? s_end[tid - 1] : end;
    q.lq = incl - q.q0;
    q.len = len;
    q.steps = max((len + p.step - 1) / p.step, 1);
    q.pitch = q.steps + p.over;
    if (s < p.seqs) {
      p.seq[s] = q;
      const int64_t units = units_of(q);
      in_shares += units * q.pitch;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        in_parts[i] += units * ((q.steps + (kPartSteps << i) - 1) & -(kPartSteps << i));
    }
    end = max(end, most);
    __syncthreads();
  }
  PlanHead h = {};
  int part = 0;  // steps
  if (p.workers > 0) {
    int64_t all, parts[2];
    scan_sum(in_shares, s_sum, &all);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      scan_sum(in_parts[i], s_sum, &parts[i]);
      __syncthreads();
    }
    part = parts[0] <= (int64_t)p.workers * kPartSteps       ? kPartSteps
           : parts[1] <= (int64_t)p.workers * 2 * kPartSteps ? 2 * kPartSteps
                                                             : 0;
    h.share = part > 0 ? part : max((all + p.workers - 1) / p.workers, (int64_t)p.least);
    h.over = part > 0 ? 0 : p.over;
  }
  int64_t base = 0;
  for (int s0 = 0; s0 < p.seqs; s0 += kPlanThreads) {
    const int s = s0 + tid;
    if (p.seqs > kPlanThreads && s < p.seqs) q = p.seq[s];
    if (part > 0) q.pitch = (q.steps + part - 1) & -part;  // (a power of two)
    const int64_t mine = s < p.seqs ? units_of(q) * q.pitch : 0;
    int64_t all;
    q.first = base + scan_sum(mine, s_sum, &all) - mine;
    if (s < p.seqs) p.seq[s] = q;
    base += all;
    __syncthreads();
  }
  if (bad) record_error(err, kDevBadSeqlens);
  if (longer) record_error(err, kDevSeqTooLong);
  if (tid == 0) {
    h.places = base;
    h.q_begin = q_begin;
    h.q_end = end;
    *p.head = h;
  }
}

// ---------------------------------------------------------------------------
// 8 rows of a KV head over a part of the keys, by mma.sync
// ---------------------------------------------------------------------------
//
// Keys are the products' M and rows their N: one decoded token's 4 or 8 heads fill an
// n8 tile, where they would leave most of an m16 tile empty, and a lane's accumulators
// for 128 channels of V are 32 instead of 64.  S comes with a lane's keys in rows of
// the fragment; movmatrix turns the probabilities for the second product.
//
// Warps work alone, each with a ring of stages of 16 keys that is filled two steps ahead
// (by TMA, two boxes a step; by cp.async where steps are not within a page).  Each has the
// same share of all units' steps, so that they end together, and while one of them waits
// for the first pages of its next unit the others go on.  (CTAs of 8 warps on one unit met
// at its start and end and took 94 us for 64 sequences of 2,050 tokens, 75 us with equal
// shares.)  Calls of few steps are cut into parts of 4 or 8 steps, a warp each, since a
// warp alone takes about 2,000 clocks a step (7 sequences of 40 to 4,000 tokens: 28 us in
// shares of 16, 12 us in parts of 4).
//
// What bounds it: instructions, 440 a step, a third of them the codes' way to fp16, and their
// latencies (0.55 a clock and scheduler, 3.6 warps each), and what warps wait for at their
// start, 14,000 clocks of 115,000.  64 sequences of 2,050 tokens, 32 / 8 heads (260 MB): 60 us,
// 4.3 TB/s; 24 sequences of 1 to 8 tokens behind 100 to 4,000: 61 us.  (Units of 16 rows, 8 warps an
// SM: 78 us for the latter.)

constexpr int kStep = 16;      // keys of a step
constexpr int kRows = 8;
constexpr int kRowWarps = 8;   // of a CTA
constexpr int kOver = 6;       // steps that a unit's start and end cost
constexpr int kLeast = 2 * kPartSteps;  // places of a warp's share
constexpr int kJoinHere = 8;   // parts that the last of them joins; more are left to join_kernel
// A row's maximum moves when a step exceeds it by more than 2^kLazy, and p is kept times
// 2^kPShift, at most 2^15 in fp16, times its key's V scale over a power of two above the
// warp's largest: fp16's smallest step, 2^-24, is then 2^-37 of the row's largest p.
constexpr float kLazy = 2.0f;
constexpr float kPShift = 13.0f;
// The tensor cores cut the bits that an fp32 sum cannot hold, and a sum of many exponentials drops
// those below its last place: V of one sign lost 1.5e-4 to 2.3e-4 over 32,768 keys of a warp, the
// log denominator up to 4e-5.  Every so many keys a warp's O and l therefore join those of the
// keys before, rounded to nearest, which wait in its slot: 3.3e-6 and 1e-5 at any length, and with
// 16-bit queries 2.2e-5 of O, a tenth of the results' rounding to fp16.  (fp32, 64 sequences of
// 8,192 tokens, 8 heads: 216 -> 224 us; of 2,050, 32 / 8 heads: 71.8 -> 73.5.  16 bits: no change.)
constexpr int kSumKeysF32 = 512, kSumKeys16 = 4096;

template <int DP, bool PV, bool WHOLE>
struct RowsCfg {
  static constexpr int kStages = PV || DP > 128 ? 3 : 5;
  static constexpr int kCodeBytes = (PV ? 2 : 1) * kStep * DP;  // of a stage: K, then V
  // behind all stages' codes: the K and V scales, of the step, or of each key with the
  // mask of those that count
  static constexpr int kScaleBytes = WHOLE ? 8 : 2 * kStep * 4 + 16;
  static constexpr int kRingBytes = kStages * kCodeBytes;  // of a warp
  static constexpr int kOffScale = kRowWarps * kRingBytes;
  static constexpr int kOffBar = kOffScale + kRowWarps * kStages * kScaleBytes;
  static constexpr int kSmemBytes = kOffBar + (WHOLE ? kRowWarps * kStages * 8 : 0);
  static constexpr int kCtas = PV && DP > 128 ? 1 : 2;  // per SM
  static_assert(kCtas * (kSmemBytes + 1024) <= 228 * 1024, "shared memory");
};

// The key in row g (of 8) of a step's fragments.  With rows of 128 bytes it is such that
// the lanes that read K at once (two g, pieces t or t + 4) and V at once (pieces g, keys of
// four even or four odd rows) meet no bank twice under the copies' 128-byte swizzle.
template <int DP, bool WHOLE>
__device__ __forceinline__ int key_of_row(int g) {
  return DP == 128 && WHOLE ? (0x37621540 >> (4 * g)) & 7 : g;
}

// A part of a unit: rows of O, then (m, l) of each.
template <int DP, bool PV>
struct Slot {
  static constexpr int kMl = PV ? kRows * DP * 4 : 0;
  static constexpr int kBytes = kMl + kRows * 8;
};

struct RowsParams {
  const void* q;
  const int8_t* k_cache;
  const float* k_scale;
  const int8_t* v_cache;
  const float* v_scale;
  const int32_t* tables;
  void* out;
  float* lse;  // nullable
  float* logits;  // nullable, without PV: [total_q * heads][logit_pitch], in powers of two
  int64_t logit_pitch;
  const PlanHead* head;
  const PlanSeq* seq;
  int* counters;   // per warp: of the unit that begins in it and goes on behind it
  CutUnit* cuts;   // per eight warps: the unit of more than kJoinHere parts that begins in them
  uint8_t* slots;  // per warp two: of the unit that it begins with, and that it ends with
  int64_t q_tok, q_head;  // strides, elements
  int64_t num_blocks;
  int seqs, total_q, heads, kv_heads, group, dim, bs, width;
  int warps;       // of the grid
  float qk_scale;  // sm_scale log2e 2^24
};

// A unit as the warps that share it see it.
struct RowsUnit {
  PlanSeq seq;
  int s, unit;      // sequence, and which of its units
  int64_t at;       // its first place
  int kvh, block;
  int rows;
  int warp0, parts; // the warps that have steps of it

  __device__ __forceinline__ void find(const RowsParams& p, const PlanHead& plan, int64_t place) {
    for (;;) {  // (sequences that are not this kernel's have no places)
      seq = p.seq[s];
      const int64_t all = (seq.lq * (int64_t)p.group + kRows - 1) / kRows * p.kv_heads;
      unit = (int)min((place - seq.first) / seq.pitch, all);
      const int64_t next = s + 1 < p.seqs ? p.seq[s + 1].first : plan.places;
      if (place < next) break;
      ++s;
    }
    at = seq.first + (int64_t)unit * seq.pitch;
    kvh = unit % p.kv_heads;
    block = unit / p.kv_heads;
    rows = (int)min((int64_t)kRows, seq.lq * (int64_t)p.group - (int64_t)block * kRows);
    warp0 = (int)((at + plan.over) / plan.share);
    parts = (int)((at + plan.over + seq.steps - 1) / plan.share) - warp0 + 1;
  }
  // the keys that row r sees: those below its token's place, counted from the end
  __device__ __forceinline__ int limit(const RowsParams& p, int r) const {
    return r < rows ? (int)((uint32_t)(block * kRows + r) / (uint32_t)p.group) + 1 + seq.len - seq.lq : 0;
  }
  // row r as (token, head) of the packed tensors
  __device__ __forceinline__ int64_t token(const RowsParams& p, int r, int* head) const {
    const uint32_t i = block * kRows + r;  // (a call has less than 2^31 rows)
    const uint32_t tok = i / (uint32_t)p.group;
    *head = kvh * p.group + (int)(i - tok * (uint32_t)p.group);
    return seq.q0 + tok;
  }
  template <int BYTES>
  __device__ __forceinline__ uint8_t* slot(const RowsParams& p, int part) const {
    return p.slots + (int64_t)(2 * (warp0 + part) + (part == 0 ? 1 : 0)) * BYTES;
  }
};

__device__ __forceinline__ float row_scale(float l) { return l > 0.0f || l != l ? 1.0f / l : 0.0f; }
__device__ __forceinline__ float row_lse(float m, float l) {
  return l == 0.0f ? -INFINITY : (m + log2f(l)) * (1.0f / kLog2e);
}

// Without PV only the denominators are taken (p.lse).  WHOLE: pages of a multiple of 16
// tokens, so that a step's keys share their scales and are one box of the caches' maps.
template <typename T, int DP, int HALVES, bool PV, bool WHOLE>
__global__ void __launch_bounds__(kRowWarps * 32, RowsCfg<DP, PV, WHOLE>::kCtas)
    rows_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                const RowsParams p, int* err) {
  using C = RowsCfg<DP, PV, WHOLE>;
  constexpr int kStages = C::kStages;
  using S = Slot<DP, PV>;
  constexpr int kPieces = DP / 16;              // 16-byte pieces of a key's codes
  constexpr int kPasses = kPieces * kStep / 32; // copies a lane makes of K or V
  constexpr int kAhead = 32 / kPieces;          // keys between them
  constexpr int kTiles = PV ? DP / 16 : 1;      // accumulators of 16 channels
  constexpr int kSteps = DP / 16;
  constexpr int kV = kStep * DP;                // V of a stage
  constexpr int kRun = DP >= 128 ? 16 : 8;      // consecutive channels of a lane's results
  constexpr int kRuns = (DP + 127) / 128;
  constexpr int kSumKeys = HALVES == 2 ? kSumKeysF32 : kSumKeys16;
  // P times its V scale as one fp16 number or two, by what the result is rounded to anyway.  One
  // number's 2^-11 adds 0.8% to the error of bf16 results, and 43% to that of fp16 ones (3.0e-4
  // instead of 2.1e-4 of their root mean square; the second costs drafted tokens 66 -> 69 us).
  constexpr bool kSplitP = !std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int in_cta = threadIdx.x >> 5;
  uint8_t* ring = smem + in_cta * C::kRingBytes;
  uint8_t* ring_scale = smem + C::kOffScale + in_cta * kStages * C::kScaleBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kOffBar) + in_cta * kStages;
  uint32_t phases = 0;  // of the stages' barriers: the next wait's
  uint64_t hold = 0;
  if constexpr (WHOLE) {
    if (lane == 0) {
      if (p.num_blocks > 0) {  // (an empty cache has no maps)
        prefetch_tensormap(&map_k);
        if (PV) prefetch_tensormap(&map_v);
      }
      for (int i = 0; i < kStages; ++i) mbar_init(&full[i], 1);
      mbar_fence_init();
    }
    __syncwarp();
    hold = l2_policy_evict_first();
  }

  launch_the_next();
  behind_the_last();
  const PlanHead head = *p.head;
  // Of the grid.  Where there is work for few warps they are on all SMs; neighbours in
  // the plan, which read other heads of the same pages, are in the same CTA (64 sequences
  // of 2,050 tokens: 67 us where they were not).
  const int busy = (int)((head.places + head.share - 1) / head.share);
  const int of_cta = min(max((busy + (int)gridDim.x - 1) / (int)gridDim.x, 1), kRowWarps);
  const int warp = in_cta < of_cta ? (int)blockIdx.x * of_cta + in_cta : p.warps;
  // rows in front of the first and behind the last sequence become zero
  const int64_t front = (int64_t)head.q_begin * p.heads;
  const int64_t behind = (int64_t)head.q_end * p.heads;
  const int64_t outside = front + (int64_t)p.total_q * p.heads - behind;
  for (int64_t i = blockIdx.x * kRowWarps + in_cta; i < outside; i += p.warps) {
    const int64_t r = i < front ? i : behind + i - front;
    for (int c = lane * 4; PV && c < p.dim; c += 128)
      store4(static_cast<T*>(p.out) + r * p.dim + c, make_float4(0, 0, 0, 0));
    if (lane == 0 && p.lse != nullptr) p.lse[r] = -INFINITY;
  }

  // what a lane copies and reads of a stage
  const int64_t token_bytes = (int64_t)p.kv_heads * p.dim;
  const int piece = lane % kPieces, key_in = lane / kPieces;
  const bool on = piece * 16 < p.dim;
  // key, and its place in a stage, of a lane's rows g and g + 8, and of columns 2 t and
  // 2 t + 1 (and + 8) of the transposed probabilities
  const int kg = key_of_row<DP, WHOLE>(g);
  const int kv0 = key_of_row<DP, WHOLE>(2 * t), kv1 = key_of_row<DP, WHOLE>(2 * t + 1);
  const auto swizzle = [&](int k, int pc) {
    return DP == 128 && WHOLE ? pc ^ (k & 7) : piece_at<DP>(k, pc);
  };
  const uint32_t k_at = kg * DP + swizzle(kg, t) * 16;
  const auto v_place = [&](int k) {
    return (uint32_t)(DP >= 128 ? k * DP + swizzle(k, g) * 16
                                : k * DP + swizzle(k, g >> 1) * 16 + (g & 1) * 8);
  };
  const uint32_t v_at[2] = {v_place(kv0), v_place(kv1)};

  int64_t now = warp * head.share;
  const int64_t stop = min(now + head.share, head.places);
  RowsUnit u;
  if (now < stop) u.s = plan_find(p.seq, p.seqs, now);
  for (; now < stop; now = u.at + u.seq.pitch) {
    u.find(p, head, now);
    const int first_step = (int)max(now - u.at - head.over, (int64_t)0);
    const int end_step = (int)min((int64_t)u.seq.steps, stop - u.at - head.over);
    if (end_step <= first_step) continue;  // none of its steps
    const int kvh = u.kvh, rows = u.rows;
    const int k0 = first_step * kStep;
    const int k1 = min(min(u.seq.len, end_step * kStep), u.limit(p, rows - 1));
    const int32_t* table = p.tables + (int64_t)u.s * p.width;

    // Keys' pages are looked up a step ahead: entry and rem are those of the next step
    // to copy, of its first key (WHOLE) or of key lane % 16.
    const int step_pages = kStep / p.bs, step_rem = kStep - step_pages * p.bs;
    int key = k0 + (WHOLE ? 0 : lane & 15);
    int page = key / p.bs, rem = key - page * p.bs;
    int entry = key < k1 ? table[page] : -1;
    int next_left = k1 - k0;  // keys from the next step to copy on
    int copied = 0;           // its stage
    uint32_t gone = 0;        // WHOLE: stages whose page is outside the cache
    const int64_t col = kvh * p.dim + (on ? piece * 16 : 0);
    const int8_t* k_col = p.k_cache + col;
    const int8_t* v_col = PV ? p.v_cache + col : nullptr;
    const auto issue = [&]() {
      if (next_left > 0) {
        uint8_t* stage = ring + copied * C::kCodeBytes;
        uint8_t* scale = ring_scale + copied * C::kScaleBytes;
        if constexpr (WHOLE) {
          const bool good = entry >= 0 && (int64_t)entry < p.num_blocks;
          gone = good ? gone & ~(1u << copied) : gone | 1u << copied;
          if (good) {
            if (lane < (PV ? 2 : 1))
              copy4_if(true, smem_u32(scale) + lane * 4,
                       (lane == 0 ? p.k_scale : p.v_scale) + (int64_t)entry * p.kv_heads + kvh);
            if (lane == 0) {
              mbar_arrive_expect_tx(&full[copied], C::kCodeBytes);
              const int token = entry * p.bs + rem;
              tma_load_3d(stage, &map_k, &full[copied], 0, kvh, token, hold);
              if (PV) tma_load_3d(stage + kV, &map_v, &full[copied], 0, kvh, token, hold);
            }
          } else {
            record_error(err, kDevBadBlockId);
          }
        } else {
          const bool counts = (lane & 15) < next_left;
          const bool good = counts && entry >= 0 && (int64_t)entry < p.num_blocks;
          if (counts && !good) record_error(err, kDevBadBlockId);
          const uint32_t to = smem_u32(stage);
          if (PV || lane < 16)
            copy4_if(good, smem_u32(scale) + lane * 4,
                     (lane < 16 ? p.k_scale : p.v_scale) +
                         (good ? (int64_t)entry * p.kv_heads + kvh : 0));
          const unsigned mask = __ballot_sync(0xffffffffu, good) & 0xffffu;
          if (lane == 0) *reinterpret_cast<uint32_t*>(scale + 128) = mask;
          const uint32_t at = good ? (uint32_t)entry * p.bs + rem : 0xffffffffu;
#pragma unroll 1
          for (int c = 0; c < kPasses; ++c) {
            const int k = c * kAhead + key_in;
            const uint32_t row = __shfl_sync(0xffffffffu, at, k);
            const bool there = row != 0xffffffffu && on;
            const int64_t from = there ? row * token_bytes : 0;
            const uint32_t dst = to + k * DP + piece_at<DP>(k, piece) * 16;
            copy16_if(there, dst, k_col + from);
            if constexpr (PV) copy16_if(there, dst + kV, v_col + from);
          }
        }
        copied = copied + 1 == kStages ? 0 : copied + 1;
        next_left -= kStep;
        key += kStep;
        page += step_pages;
        rem += step_rem;
        if (rem >= p.bs) {
          rem -= p.bs;
          ++page;
        }
        entry = key < k1 ? table[page] : -1;
      }
      copies_commit();
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue();

    Raw4<T> raw[kSteps];  // row g's queries, on their way
    {
      int h;
      const int64_t tok = u.token(p, g, &h);
      load_queries<T, DP>(g < rows ? static_cast<const T*>(p.q) + tok * p.q_tok + h * p.q_head : nullptr,
                          p.dim, raw);
    }
    // a lane's rows are 2 t and 2 t + 1
    uint2 qr[HALVES][kSteps];
    float f[2], start[2];
    split_queries<T, DP, HALVES>(raw, qr, f, start);
    f[0] *= p.qk_scale;
    f[1] *= p.qk_scale;
    const int limit0 = u.limit(p, 2 * t), limit1 = u.limit(p, 2 * t + 1);
    const int clear = min(u.limit(p, 0), k1);  // every row sees the keys below
    float* logit[2] = {nullptr, nullptr};
    if constexpr (!PV) {
      if (p.logits != nullptr)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          int h;
          const int64_t tok = u.token(p, 2 * t + r, &h);
          if (2 * t + r < rows) logit[r] = p.logits + (tok * p.heads + h) * p.logit_pitch + kg;
        }
    }

    // p is 2^(score - base); base moves where a score is above most
    float o[kTiles][4];
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;
    float base[2] = {0.0f, 0.0f}, most[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    // O is in units of `unit_v`, a power of two above the V scales so far, so that p
    // times scale stays in fp16
    float unit_v = 0.0f, inv_v = 0.0f;

    // channels c * 128 + g * kRun + 4 x on of row 2 t + r
    const auto result = [&](int r, int c, int x, float by) {
      const int at = c * 8 + 2 * x;
      return make_float4(o[at][r] * by, o[at][r + 2] * by, o[at + 1][r] * by, o[at + 1][r + 2] * by);
    };
    const auto sum_over_lanes = [&]() {  // l of all the lanes of a row
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], x);
    };
    // The sums of earlier keys, in the slot as a part's: rows of O, then (base, l).
    uint8_t* slot = u.slot<S::kBytes>(p, warp - u.warp0);
    bool summed = false;
    const auto join_sums = [&](bool keep) {
      if (summed) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float2 was = reinterpret_cast<const float2*>(slot + S::kMl)[2 * t + r];
          const float f = was.y == 0.0f ? 0.0f : ex2(was.x - base[r]);
          if (g == 0) l[r] += was.y * f;
          if constexpr (PV) {
            const float* from = reinterpret_cast<const float*>(slot) + (2 * t + r) * DP;
            const float by = f * inv_v;
#pragma unroll
            for (int c = 0; c < kRuns; ++c)
#pragma unroll
              for (int x = 0; x < kRun / 4; ++x) {
                const float4 v = *reinterpret_cast<const float4*>(from + c * 128 + g * kRun + 4 * x);
                const int at = c * 8 + 2 * x;
                o[at][r] += v.x * by, o[at][r + 2] += v.y * by;
                o[at + 1][r] += v.z * by, o[at + 1][r + 2] += v.w * by;
              }
          }
        }
        __syncwarp();  // (base, l) are read
      }
      sum_over_lanes();
      if (!keep) return;
      summed = true;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        if constexpr (PV) {
          float* to = reinterpret_cast<float*>(slot) + (2 * t + r) * DP;
#pragma unroll
          for (int c = 0; c < kRuns; ++c)
#pragma unroll
            for (int x = 0; x < kRun / 4; ++x)
              *reinterpret_cast<float4*>(to + c * 128 + g * kRun + 4 * x) = result(r, c, x, unit_v);
        }
        if (g == 0) reinterpret_cast<float2*>(slot + S::kMl)[2 * t + r] = make_float2(base[r], l[r]);
        l[r] = 0.0f;
      }
      if constexpr (PV) {
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;
      }
      __syncwarp();
    };

    int used = 0;  // the stage
    for (int key_now = k0;; key_now += kStep) {
      const bool end = key_now >= k1;
      if (end || (key_now > k0 && (key_now - k0) % kSumKeys == 0)) join_sums(!end);
      if (end) break;
      copies_wait<kStages - 2>();
      __syncwarp();
      issue();
      const uint8_t* stage = ring + used * C::kCodeBytes;
      const float* scales = reinterpret_cast<const float*>(ring_scale + used * C::kScaleBytes);
      const int here = used;
      used = used + 1 == kStages ? 0 : used + 1;
      if constexpr (WHOLE) {
        if (gone >> here & 1u) continue;
        if (!mbar_wait_short(&full[here], phases >> here & 1u, err)) {
          record_error(err, kDevWaitTimeout);
          mbar_drain(&full[here], phases >> here & 1u);  // no copy outlives the CTA
        }
        phases ^= 1u << here;
        __syncwarp();
      }
      // scores: keys of rows g and g + 8, query rows as above: (g, first), (g, second), (g + 8, ...);
      // two sums, since a product waits 25 clocks for the one before it
      float sc[4] = {start[0], start[1], start[0], start[1]}, sd[4] = {};
#pragma unroll
      for (int pc = 0; pc < DP / 64; ++pc) {
        // (piece pc * 4 + t: bit 2 turned by odd pc)
        const uint32_t at = (k_at ^ ((pc & 1) * 64)) + pc / 2 * 128;
        const uint4 w0 = *reinterpret_cast<const uint4*>(stage + at);
        const uint4 w1 = *reinterpret_cast<const uint4*>(stage + at + 8 * DP);  // (the same swizzle)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint2 x = codes_plus_128(e == 0 ? w0.x : e == 1 ? w0.y : e == 2 ? w0.z : w0.w);
          const uint2 y = codes_plus_128(e == 0 ? w1.x : e == 1 ? w1.y : e == 2 ? w1.z : w1.w);
          const uint4 a = make_uint4(x.x, y.x, x.y, y.y);
          if constexpr (HALVES == 2) mma_f16(sd, a, qr[HALVES - 1][pc * 4 + e].x, qr[HALVES - 1][pc * 4 + e].y);
          if (HALVES == 1 && (e & 1)) mma_f16(sd, a, qr[0][pc * 4 + e].x, qr[0][pc * 4 + e].y);
          else mma_f16(sc, a, qr[0][pc * 4 + e].x, qr[0][pc * 4 + e].y);
        }
      }
      float ks[2], vs[2] = {0.0f, 0.0f};
      uint32_t mask = 0xffffu;
      if constexpr (WHOLE) {
        const float2 x = *reinterpret_cast<const float2*>(scales);
        ks[0] = ks[1] = x.x;
        if constexpr (PV) vs[0] = vs[1] = x.y;
      } else {
        ks[0] = scales[kg], ks[1] = scales[kg + 8];
        if constexpr (PV) vs[0] = scales[kStep + kg], vs[1] = scales[kStep + kg + 8];
        mask = reinterpret_cast<const uint32_t*>(scales)[2 * kStep];
      }
      const bool all = (WHOLE || mask == 0xffffu) && key_now + kStep <= clear;
      const auto seen = [&](int e) {  // e as in sc
        const int k = kg + (e >> 1) * 8;
        return (WHOLE ? key_now + k < k1 : mask >> k & 1u) &&
               key_now + k < ((e & 1) ? limit1 : limit0);
      };
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[e] = (sc[e] + sd[e]) * (ks[e >> 1] * f[e & 1]);
      if (!all) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!seen(e)) sc[e] = -INFINITY;
      }
      bool move = fmaxf(sc[0], sc[2]) > most[0] || fmaxf(sc[1], sc[3]) > most[1];
      if constexpr (PV) {
        const float v0 = fabsf(vs[0]), v1 = fabsf(vs[1]);
        move |= v0 > unit_v && v0 <= 3.0e38f;
        if constexpr (!WHOLE) move |= v1 > unit_v && v1 <= 3.0e38f;
      }
      if (__any_sync(0xffffffffu, move)) {
        float down = 1.0f;
        if constexpr (PV) {
          const auto finite = [](float v) {
            v = fabsf(v);
            return v <= 3.0e38f ? __float_as_uint(v) : 0u;
          };
          const uint32_t big = __reduce_max_sync(0xffffffffu, max(finite(vs[0]), finite(vs[1])));
          if (__uint_as_float(big) > unit_v) {
            const float unit_now = power_of_two(min(max((int)(big >> 23) - 126, -126), 126));
            inv_v = 1.0f / unit_now;
            down = unit_v * inv_v;
            unit_v = unit_now;
          }
        }
        float a[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float top = fmaxf(sc[r], sc[r + 2]);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
          a[r] = 1.0f;
          if (top > most[r]) {
            const float to = top - kPShift;
            a[r] = most[r] == -INFINITY ? 0.0f : ex2(base[r] - to);
            base[r] = to;
            most[r] = top + kLazy;
          }
          l[r] *= a[r];
          a[r] *= down;
        }
        if constexpr (PV) {
#pragma unroll
          for (int c = 0; c < kTiles; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[c][e] *= a[e & 1];
        }
      }
      if constexpr (!PV) {
#pragma unroll
        for (int r = 0; r < 2; ++r)
          if (logit[r] != nullptr) {
            if (key_now + kg < k1) logit[r][key_now] = sc[r];
            if (key_now + kg + 8 < k1) logit[r][key_now + 8] = sc[r + 2];
          }
      }
      uint32_t hi[2], lo[2];  // keys g, g + 8
      const float v0 = vs[0] * inv_v, v1 = vs[1] * inv_v;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float x0 = ex2(sc[2 * k] - base[0]), x1 = ex2(sc[2 * k + 1] - base[1]);
        l[0] += x0;
        l[1] += x1;
        if constexpr (PV) {
          float z0 = x0 * (k ? v1 : v0), z1 = x1 * (k ? v1 : v0);
          if (!all) {  // (a V scale that is not finite does not reach rows in front)
            if (!seen(2 * k)) z0 = 0.0f;
            if (!seen(2 * k + 1)) z1 = 0.0f;
          }
          const __half2 h = __floats2half2_rn(z0, z1);
          hi[k] = transpose_8x8(word_of(h));
          if constexpr (kSplitP) {
            const float2 b = __half22float2(h);
            lo[k] = transpose_8x8(word_of(__floats2half2_rn(z0 - b.x, z1 - b.y)));
          }
        }
      }
      if constexpr (PV) {
        // O: channels c * 128 + g * 16 + 4 w + e (of 64: g * 8 + 4 w + e) of lane (g, .)
        // are rows g (even e) and g + 8 (odd e) of accumulator c * 8 + 2 w + e / 2
        const uint8_t* vt = stage + kV;
        constexpr int kWords = DP >= 128 ? 4 : 2;
#pragma unroll
        for (int c = 0; c < kRuns; ++c) {
          uint32_t w[4][kWords];  // keys kv0, kv1, kv0 + 8, kv1 + 8
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t at = v_at[k & 1] + (k >> 1) * 8 * DP + c * 128;
            if constexpr (DP >= 128) {
              const uint4 x = *reinterpret_cast<const uint4*>(vt + at);
              w[k][0] = x.x, w[k][1] = x.y, w[k][2 % kWords] = x.z, w[k][3 % kWords] = x.w;
            } else {
              const uint2 x = *reinterpret_cast<const uint2*>(vt + at);
              w[k][0] = x.x, w[k][1] = x.y;
            }
          }
#pragma unroll
          for (int x = 0; x < kWords; ++x) {
            const uint2 b01 = codes_to_half(__byte_perm(w[0][x], w[1][x], 0x5140));
            const uint2 b23 = codes_to_half(__byte_perm(w[0][x], w[1][x], 0x7362));
            const uint2 c01 = codes_to_half(__byte_perm(w[2][x], w[3][x], 0x5140));
            const uint2 c23 = codes_to_half(__byte_perm(w[2][x], w[3][x], 0x7362));
            const uint4 a0 = make_uint4(b01.x, b01.y, c01.x, c01.y);
            const uint4 a1 = make_uint4(b23.x, b23.y, c23.x, c23.y);
            if constexpr (kSplitP) {
              mma_f16(o[c * 8 + 2 * x], a0, lo[0], lo[1]);
              mma_f16(o[c * 8 + 2 * x + 1], a1, lo[0], lo[1]);
            }
            mma_f16(o[c * 8 + 2 * x], a0, hi[0], hi[1]);
            mma_f16(o[c * 8 + 2 * x + 1], a1, hi[0], hi[1]);
          }
        }
      }
    }
    copies_wait<0>();
    __syncwarp();
    if (u.parts == 1) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        if (2 * t + r >= rows) continue;
        int h;
        const int64_t tok = u.token(p, 2 * t + r, &h);
        if constexpr (PV) {
          T* to = static_cast<T*>(p.out) + (tok * p.heads + h) * p.dim;
          const float by = row_scale(l[r]) * unit_v;
#pragma unroll
          for (int c = 0; c < kRuns; ++c)
#pragma unroll
            for (int x = 0; x < kRun / 4; ++x)
              if (c * 128 + g * kRun + 4 * x < p.dim)
                store4(to + c * 128 + g * kRun + 4 * x,
                       l[r] == 0.0f ? make_float4(0, 0, 0, 0) : result(r, c, x, by));
        }
        if (g == 0 && p.lse != nullptr) p.lse[tok * p.heads + h] = row_lse(base[r], l[r]);
      }
      continue;
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if (2 * t + r >= rows) continue;
      if constexpr (PV) {
        float* to = reinterpret_cast<float*>(slot) + (2 * t + r) * DP;
#pragma unroll
        for (int c = 0; c < kRuns; ++c)
#pragma unroll
          for (int x = 0; x < kRun / 4; ++x)
            *reinterpret_cast<float4*>(to + c * 128 + g * kRun + 4 * x) = result(r, c, x, unit_v);
      }
      if (g == 0) {
        // nothing attended: (-inf, 0); every score NaN: l is
        const float m = most[r] == -INFINITY && l[r] == l[r] ? -INFINITY : base[r];
        reinterpret_cast<float2*>(slot + S::kMl)[2 * t + r] = make_float2(m, l[r]);
      }
    }
    if (u.parts > kJoinHere) {
      if (lane == 0 && warp == u.warp0)
        p.cuts[warp / kRowWarps] = CutUnit{u.parts, u.rows, u.kvh, u.block, u.seq.q0, u.warp0};
      continue;
    }
    __syncwarp();
    int last = 0;
    if (lane == 0) last = atomic_add_acq_rel_gpu(&p.counters[u.warp0], 1) == u.parts - 1;
    if (!__shfl_sync(0xffffffffu, last, 0)) continue;
    // The last part to end joins all of them, in order: lane r has row r's factors, then a
    // lane four channels of all rows, so that a part's loads are under way together.
    float by[kJoinHere] = {}, m = -INFINITY, sum = 0.0f;
    {
      float2 ml[kJoinHere];
#pragma unroll
      for (int i = 0; i < kJoinHere; ++i) {
        ml[i] = make_float2(-INFINITY, 0.0f);
        if (i < u.parts && lane < rows)
          ml[i] = __ldcg(reinterpret_cast<const float2*>(u.slot<S::kBytes>(p, i) + S::kMl) + lane);
        m = fmaxf(m, ml[i].x);
      }
#pragma unroll
      for (int i = 0; i < kJoinHere; ++i) {
        by[i] = ml[i].x == -INFINITY ? 0.0f : ex2(ml[i].x - m);
        sum += ml[i].y * by[i];
      }
    }
    int h = 0;
    const int64_t tok = lane < rows ? u.token(p, lane, &h) : 0;
    if (lane < rows && p.lse != nullptr) p.lse[tok * p.heads + h] = row_lse(m, sum);
    if constexpr (PV) {
      const int64_t place = (tok * p.heads + h) * p.dim;
#pragma unroll
      for (int c = 0; c < (DP + 127) / 128; ++c) {
        const int at = c * 128 + lane * 4;
        float4 acc[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) acc[r] = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < kJoinHere; ++i) {
          if (i >= u.parts) break;
          const float* from = reinterpret_cast<const float*>(u.slot<S::kBytes>(p, i)) + at;
          float4 v[kRows];
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            v[r] = make_float4(0, 0, 0, 0);
            if (r < rows && at < DP) v[r] = __ldcg(reinterpret_cast<const float4*>(from + r * DP));
          }
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            const float k = __shfl_sync(0xffffffffu, by[i], r);  // (of a part of little weight 0: NaN stays)
            acc[r].x += v[r].x * k, acc[r].y += v[r].y * k, acc[r].z += v[r].z * k, acc[r].w += v[r].w * k;
          }
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const float l = __shfl_sync(0xffffffffu, sum, r), inv = row_scale(l);
          const int64_t to = __shfl_sync(0xffffffffu, place, r);
          if (r < rows && at < p.dim)
            store4(static_cast<T*>(p.out) + to + at,
                   l == 0.0f ? make_float4(0, 0, 0, 0)
                             : make_float4(acc[r].x * inv, acc[r].y * inv, acc[r].z * inv, acc[r].w * inv));
        }
      }
    }
  }
}

// Units of many parts (few long sequences): two CTAs for each eight warps, in which no more
// than one begins, each for 4 rows, of which a warp takes every fourth part.
constexpr int kJoinRows = 4, kJoinWarps = 16;
static_assert(kJoinHere >= kRowWarps, "one unit of more parts in so many warps");
template <typename T, int DP, bool PV>
__global__ void __launch_bounds__(kJoinWarps * 32, 2) join_kernel(const RowsParams p) {
  using S = Slot<DP, PV>;
  constexpr int kWide = (DP + 127) / 128, kSlices = kJoinWarps / kJoinRows;
  __shared__ float4 s_o[kJoinWarps][kWide * 32];
  __shared__ float2 s_ml[kJoinWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = blockIdx.y * kJoinRows + warp % kJoinRows, slice = warp / kJoinRows;
  launch_the_next();
  behind_the_last();
  const CutUnit cut = p.cuts[blockIdx.x];
  if (cut.parts == 0 || (int)blockIdx.y * kJoinRows >= cut.rows) return;
  RowsUnit u;
  u.warp0 = cut.first, u.parts = cut.parts, u.rows = cut.rows;
  u.kvh = cut.kvh, u.block = cut.block, u.seq.q0 = cut.q0;
  float m = -INFINITY, l = 0.0f;
  float4 acc[kWide];
#pragma unroll
  for (int c = 0; c < kWide; ++c) acc[c] = make_float4(0, 0, 0, 0);
  const auto add = [&](float2 ml, const float4 (&v)[kWide]) {
    if (ml.x == -INFINITY) return;
    const float big = fmaxf(m, ml.x), f = m == -INFINITY ? 0.0f : ex2(m - big), k = ex2(ml.x - big);
    m = big;
    l = l * f + ml.y * k;
#pragma unroll
    for (int c = 0; c < kWide; ++c) {
      acc[c].x = acc[c].x * f + v[c].x * k, acc[c].y = acc[c].y * f + v[c].y * k;
      acc[c].z = acc[c].z * f + v[c].z * k, acc[c].w = acc[c].w * f + v[c].w * k;
    }
  };
  constexpr int kBatch = DP > 128 ? 2 : 4;
  if (r < u.rows)
    for (int i = slice; i < u.parts; i += kBatch * kSlices) {
      float2 ml[kBatch];
      float4 v[kBatch][kWide];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const bool there = i + b * kSlices < u.parts;
        const uint8_t* from = u.slot<S::kBytes>(p, there ? i + b * kSlices : i);
        ml[b] = there ? __ldcg(reinterpret_cast<const float2*>(from + S::kMl) + r)
                      : make_float2(-INFINITY, 0.0f);
#pragma unroll
        for (int c = 0; c < kWide; ++c) {
          v[b][c] = make_float4(0, 0, 0, 0);
          if (PV && c * 128 + lane * 4 < DP)
            v[b][c] = __ldcg(reinterpret_cast<const float4*>(
                reinterpret_cast<const float*>(from) + r * DP + c * 128 + lane * 4));
        }
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) add(ml[b], v[b]);
    }
#pragma unroll
  for (int c = 0; c < kWide; ++c) s_o[warp][c * 32 + lane] = acc[c];
  if (lane == 0) s_ml[warp] = make_float2(m, l);
  __syncthreads();
  if (slice > 0 || r >= u.rows) return;
  for (int w = warp + kJoinRows; w < kJoinWarps; w += kJoinRows) {
    float4 v[kWide];
#pragma unroll
    for (int c = 0; c < kWide; ++c) v[c] = s_o[w][c * 32 + lane];
    add(s_ml[w], v);
  }
  int h;
  const int64_t tok = u.token(p, r, &h);
  const float inv = row_scale(l);
  if constexpr (PV) {
#pragma unroll
    for (int c = 0; c < kWide; ++c)
      if (c * 128 + lane * 4 < p.dim)
        store4(static_cast<T*>(p.out) + (tok * p.heads + h) * p.dim + c * 128 + lane * 4,
               l == 0.0f ? make_float4(0, 0, 0, 0)
                         : make_float4(acc[c].x * inv, acc[c].y * inv, acc[c].z * inv, acc[c].w * inv));
  }
  if (lane == 0 && p.lse != nullptr) p.lse[tok * p.heads + h] = row_lse(m, l);
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

}  // namespace

bool cache_map(CUtensorMap* map, const int8_t* cache, const ChunkArgs& a, int channels, int tokens,
               bool swizzle) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return false;
  if (a.num_blocks == 0) return true;  // (never used)
  cuuint64_t dims[3] = {(cuuint64_t)a.dim, (cuuint64_t)a.kv_heads,
                        (cuuint64_t)a.num_blocks * a.block_size};
  cuuint64_t strides[2] = {(cuuint64_t)a.dim, (cuuint64_t)a.dim * a.kv_heads};
  cuuint32_t box[3] = {(cuuint32_t)channels, 1, (cuuint32_t)tokens};
  cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<int8_t*>(cache), dims, strides, box,
            estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            !swizzle         ? CU_TENSOR_MAP_SWIZZLE_NONE
            : channels == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                             : CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

namespace {

constexpr int kMostWarps = 148 * 2 * kRowWarps;

// Which kernels a call's sequences go to: those of few rows to the warps of rows_kernel,
// the others to chunk_tc.cu, where it takes the shapes.  (24 sequences of 1 to 8 tokens in
// groups of 4: 60 us by the warps; 66 us by chunk_tc.cu, or 54 us there for those above 16
// rows and 28 us by the warps for the rest, since a unit there costs about 10 us to start
// and end.  What a unit costs does not grow with the keys: 24 sequences of 8 tokens, 32 rows,
// take the warps 55, 152, 603 and 1,160 us behind 1,000, 4,000, 16,000 and 32,000 keys, and
// chunk_tc.cu 55, 118, 325 and 621; of 4 tokens, 16 rows, 41, 88, 281 and 607 against 41, 89, 323 and
// 617.)  The lengths are on the device, so a call launches both unless its sizes tell.
constexpr int kFewRows = 32, kFewSteps = 4096;
struct Division {
  bool rows, tc;
};
Division division_of(const ChunkArgs& a) {
  const int group = a.heads / a.kv_heads;
  const int64_t most_rows = a.total_q * group;
  const int64_t units = (most_rows / kRows + std::min<int64_t>(a.seqs, a.total_q)) * a.kv_heads;
  const int64_t steps = (int64_t)a.width * a.block_size / kStep + 1;
  if (a.v_cache == nullptr || !chunk_tc_takes(a) || most_rows <= kFewRows ||
      (a.total_q <= a.seqs && group <= kFewRows) || units <= kFewSteps / steps)
    return {true, false};
  return {group <= kFewRows, true};
}

struct ChunkLayout {
  size_t head, seq, counters, slots, head2, seq2, tc, total;
};

ChunkLayout chunk_layout(const ChunkArgs& a) {
  const int dp = a.dim <= 64 ? 64 : a.dim <= 128 ? 128 : 256;
  ChunkLayout l;
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  const Division d = division_of(a);
  l.head = take(sizeof(PlanHead));
  l.seq = take(sizeof(PlanSeq) * (size_t)a.seqs);
  // (the counters and the cut units are zeroed together)
  l.counters = take(d.rows ? sizeof(int) * kMostWarps + sizeof(CutUnit) * (kMostWarps / kRowWarps) : 0);
  l.slots = take(d.rows ? (size_t)2 * kMostWarps * ((a.v_cache != nullptr ? kRows * dp * 4 : 0) + kRows * 8) : 0);
  l.head2 = take(d.tc ? sizeof(PlanHead) : 0);
  l.seq2 = take(d.tc ? sizeof(PlanSeq) * (size_t)a.seqs : 0);
  l.tc = take(d.tc ? chunk_tc_workspace_size(a) : 0);
  l.total = at + 256;
  return l;
}

// CTAs of a launch: no more warps than have their least part of the longest that the batch
// can be.
int64_t rows_ctas(const ChunkArgs& a, int per_sm) {
  const int64_t units =
      (a.total_q * (a.heads / a.kv_heads) / kRows + std::min<int64_t>(a.seqs, a.total_q) + 1) * a.kv_heads;
  const int64_t parts = ((int64_t)a.width * a.block_size + kStep * kPartSteps - 1) / (kStep * kPartSteps) + 1;
  const int64_t most = 148 * per_sm;
  return std::min(most, units >= most * kRowWarps ? most : (units * parts + kRowWarps - 1) / kRowWarps);
}

template <typename T, int DP, bool PV, bool WHOLE>
int launch_rows(const ChunkArgs& a, uint8_t* ws, cudaStream_t stream) {
  constexpr int HALVES = sizeof(T) == 4 ? 2 : 1;
  using C = RowsCfg<DP, PV, WHOLE>;
  const ChunkLayout lay = chunk_layout(a);
  RowsParams p;
  p.q = a.q;
  p.k_cache = a.k_cache;
  p.k_scale = a.k_scale;
  p.v_cache = a.v_cache;
  p.v_scale = a.v_scale;
  p.tables = a.tables;
  p.out = a.out;
  p.lse = a.lse;
  p.logits = a.logits;
  p.logit_pitch = (int64_t)a.width * a.block_size;
  p.head = reinterpret_cast<PlanHead*>(ws + lay.head);
  p.seq = reinterpret_cast<PlanSeq*>(ws + lay.seq);
  p.counters = reinterpret_cast<int*>(ws + lay.counters);
  p.cuts = reinterpret_cast<CutUnit*>(p.counters + kMostWarps);
  p.slots = ws + lay.slots;
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
  p.qk_scale = a.sm_scale * kLog2e * kCodeUnit;
  auto kern = rows_kernel<T, DP, HALVES, PV, WHOLE>;
  static std::atomic<uint64_t> done{0};
  allow_shared_memory(reinterpret_cast<const void*>(kern), C::kSmemBytes, done);
  const int64_t ctas = rows_ctas(a, C::kCtas);
  p.warps = (int)ctas * kRowWarps;
  CUtensorMap map_k = {}, map_v = {};
  if (WHOLE && (!cache_map(&map_k, a.k_cache, a, DP, kStep, true) ||
                (PV && !cache_map(&map_v, a.v_cache, a, DP, kStep, true)))) {
    set_error("cuTensorMapEncodeTiled failed for the caches");
    return kCudaError;
  }
  launch_behind(kern, dim3((unsigned)ctas), kRowWarps * 32, C::kSmemBytes, stream, map_k, map_v, p,
                device_error_word());
  // a unit of so many parts needs so many steps
  if (((int64_t)a.width * a.block_size + kStep - 1) / kStep > (int64_t)kPartSteps * kJoinHere)
    launch_behind(join_kernel<T, DP, PV>, dim3((unsigned)ctas, kRows / kJoinRows), kJoinWarps * 32, 0, stream, p);
  return kOk;
}

}  // namespace

int launch_plan(const PlanArgs& a, const PlanArgs* second, const ZeroArgs& zero, int* err,
                cudaStream_t stream) {
  const int plans = second != nullptr ? 2 : 1;
  const int64_t slots = zero.sums != nullptr ? (int64_t)zero.seqs * zero.width * zero.block_size : 0;
  const int64_t zeros = std::min<int64_t>((slots + 4 * kPlanThreads - 1) / (4 * kPlanThreads), 148 * 4);
  plan_kernel<<<(unsigned)(plans + zeros), kPlanThreads, 0, stream>>>(
      a, second != nullptr ? *second : a, plans, zero, err);
  return kOk;
}

const PlanSeq* chunk_plan(const ChunkArgs& a, void* workspace) {
  uint8_t* ws = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(workspace) + 255) &
                                           ~(uintptr_t)255);
  return reinterpret_cast<const PlanSeq*>(ws + chunk_layout(a).seq);
}

// (without a V cache only the denominators are taken)
size_t chunk_workspace_size(const ChunkArgs& a) {
  if (a.total_q == 0) return 0;
  return chunk_layout(a).total;
}

int launch_chunk(const ChunkArgs& a, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  if (a.total_q == 0) return kOk;
  if (workspace == nullptr || workspace_bytes < chunk_workspace_size(a)) {
    set_error("workspace too small for chunk_attention: need " +
              std::to_string(chunk_workspace_size(a)) + " bytes");
    return kWorkspace;
  }
  uint8_t* ws = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(workspace) + 255) &
                                           ~(uintptr_t)255);
  const ChunkLayout lay = chunk_layout(a);
  const Division d = division_of(a);
  PlanArgs plan;
  plan.cu = a.cu;
  plan.lens = a.lens;
  plan.seqs = a.seqs;
  plan.total_q = (int)a.total_q;
  plan.group = a.heads / a.kv_heads;
  plan.kv_heads = a.kv_heads;
  plan.block_size = a.block_size;
  plan.width = a.width;
  plan.rows = kRows;
  plan.step = kStep;
  plan.over = kOver;
  plan.workers = (int)rows_ctas(a, a.v_cache != nullptr && a.dim > 128 ? 1 : 2) * kRowWarps;
  plan.least = kLeast;
  plan.which = d.tc ? kPlanFew : kPlanAll;
  plan.few_rows = kFewRows;
  plan.few_steps = d.rows ? kFewSteps : 0;
  plan.head = reinterpret_cast<PlanHead*>(ws + lay.head);
  plan.seq = reinterpret_cast<PlanSeq*>(ws + lay.seq);
  plan.counters = reinterpret_cast<int*>(ws + lay.counters);
  plan.counts = kMostWarps + (int)sizeof(CutUnit) / 4 * (kMostWarps / kRowWarps);
  PlanArgs plan2 = chunk_tc_plan(plan);
  plan2.which = d.rows ? kPlanMany : kPlanAll;
  plan2.head = reinterpret_cast<PlanHead*>(ws + lay.head2);
  plan2.seq = reinterpret_cast<PlanSeq*>(ws + lay.seq2);
  launch_plan(d.rows ? plan : plan2, d.rows && d.tc ? &plan2 : nullptr, a.zero, device_error_word(),
              stream);
  int rc = kOk;
  if (d.tc) rc = launch_chunk_tc(a, plan2.head, plan2.seq, ws + lay.tc, !d.rows, stream);
  if (rc != kOk) return rc;
  const auto with_dim = [&](auto t) {
    using T = decltype(t);
    const auto with = [&](auto dp, auto pv) {
      constexpr int DP = decltype(dp)::value;
      constexpr bool PV = decltype(pv)::value;
      if constexpr (DP <= 128)
        if (a.block_size % kStep == 0) return launch_rows<T, DP, PV, true>(a, ws, stream);
      return launch_rows<T, DP, PV, false>(a, ws, stream);
    };
    const auto with_pv = [&](auto dp) {
      return a.v_cache != nullptr ? with(dp, std::true_type{}) : with(dp, std::false_type{});
    };
    return a.dim <= 64    ? with_pv(std::integral_constant<int, 64>{})
           : a.dim <= 128 ? with_pv(std::integral_constant<int, 128>{})
                          : with_pv(std::integral_constant<int, 256>{});
  };
  if (d.rows)
    rc = a.dtype == 0 ? with_dim(0.0f) : a.dtype == 1 ? with_dim(__half()) : with_dim(__nv_bfloat16());
  if (rc != kOk) return rc;
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_error(std::string("chunk attention launch failed: ") + cudaGetErrorString(e));
    return kCudaError;
  }
  return kOk;
}

}  // namespace pkv
