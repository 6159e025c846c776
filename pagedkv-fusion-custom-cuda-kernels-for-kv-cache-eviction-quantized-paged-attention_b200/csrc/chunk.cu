// Attention of new tokens over the INT8 paged cache that holds them: one token of a
// sequence, a few drafted ones, or a chunk of a prompt behind what was cached before.
//
//   out[i, h] = sum_j softmax_j(scale q[i, h] . k_j) v_j,   j <= i + L - Lq
//
// k_j and v_j are codes times the scale of their (page, head).  The codes are exact
// in fp16; the products run on the tensor cores with fp32 sums, the K scales on the
// scores and the V scales on the probabilities.
//
//   plan_kernel   one CTA: the sequences' rows and lengths, checked; how many parts
//                 each one's keys are split into; the items' numbers;
//   rows_kernel   an item is (sequence, 16 query rows of a KV head, part of the keys).
#include <cuda_runtime.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "cache_mma.cuh"
#include "pkv_internal.h"

namespace pkv {
namespace {

constexpr int kPlanThreads = 1024;

// Inclusive sum (or maximum) over the CTA; `carry` of the warps by shared memory.
template <typename V, typename Op>
__device__ __forceinline__ V scan_cta(V v, V* shared, Op op) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v = op(v, x);
  }
  __syncthreads();
  if (lane == 31) shared[warp] = v;
  __syncthreads();
  if (warp > 0) {
    V before = shared[0];
    for (int w = 1; w < warp; ++w) before = op(before, shared[w]);
    v = op(v, before);
  }
  return v;
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanArgs p, int* err) {
  __shared__ int64_t s_scan[kPlanThreads / 32];
  __shared__ int64_t s_carry[4];
  const int tid = threadIdx.x;
  for (int i = tid; i < p.counts; i += kPlanThreads) p.counters[i] = 0;
  const auto most = [](int64_t a, int64_t b) { return a > b ? a : b; };
  const auto sum = [](int64_t a, int64_t b) { return a + b; };
  // rows and lengths; an entry of cu below an earlier one counts as the largest
  // before it
  int64_t end = min(max(p.cu[0], 0), p.total_q), work = 0;
  const int q_begin = (int)end;
  bool bad = tid == 0 && (p.cu[0] < 0 || p.cu[0] > p.total_q), longer = false;
  for (int s0 = 0; s0 < p.seqs; s0 += kPlanThreads) {
    const int s = s0 + tid;
    int64_t q1 = 0;
    int len = 0;
    if (s < p.seqs) {
      const int c = p.cu[s + 1];
      q1 = min(max(c, 0), p.total_q);
      bad |= c < p.cu[s] || c > p.total_q;
      const int64_t room = (int64_t)p.width * p.block_size;
      len = max(p.lens[s], 0);
      longer |= len > room;
      len = (int)min((int64_t)len, room);
    }
    const int64_t incl = most(scan_cta(q1, s_scan, most), end);
    __syncthreads();
    if (tid < kPlanThreads && (tid & 31) == 31) s_scan[tid >> 5] = incl;
    int64_t before = __shfl_up_sync(0xffffffffu, incl, 1);
    __syncthreads();
    if ((tid & 31) == 0) before = tid > 0 ? s_scan[(tid >> 5) - 1] : end;
    if (s < p.seqs) {
      PlanSeq q;
      q.q0 = (int)before;
      q.lq = (int)(incl - before);
      q.len = len;
      p.seq[s] = q;
      work += (int64_t)((q.lq * (int64_t)p.group + p.rows - 1) / p.rows) * p.kv_heads * len;
    }
    end = s_scan[kPlanThreads / 32 - 1];
  }
  if (bad) record_error(err, kDevBadSeqlens);
  if (longer) record_error(err, kDevSeqTooLong);
  const int64_t mine = scan_cta(work, s_scan, sum);
  if (tid == kPlanThreads - 1) s_carry[0] = mine;
  __syncthreads();
  int64_t part = p.target > 0 ? (s_carry[0] + p.target - 1) / p.target : 0;
  part = (most(part, p.least) + p.round - 1) / p.round * p.round;
  const int split = (int)(part < (1 << 30) ? part : 1 << 30);
  int64_t items = 0, slots = 0, units = 0;
  for (int s0 = 0; s0 < p.seqs; s0 += kPlanThreads) {
    const int s = s0 + tid;
    int n = 0, u = 0, parts = 1;
    if (s < p.seqs) {
      const PlanSeq q = p.seq[s];
      u = (int)((q.lq * (int64_t)p.group + p.rows - 1) / p.rows) * p.kv_heads;
      if (q.len > split) parts = (q.len - 1) / split + 1;
      n = u * parts;
    }
    const int64_t a = scan_cta((int64_t)n, s_scan, sum);
    const int64_t b = scan_cta((int64_t)(parts > 1 ? n : 0), s_scan, sum);
    const int64_t c = scan_cta((int64_t)(parts > 1 ? u : 0), s_scan, sum);
    if (s < p.seqs) {
      PlanSeq* q = &p.seq[s];
      q->splits = parts;
      q->first = (int)(items + a - n);
      q->slot = (int)(slots + b - (parts > 1 ? n : 0));
      q->unit = (int)(units + c - (parts > 1 ? u : 0));
    }
    __syncthreads();
    if (tid == kPlanThreads - 1) s_carry[1] = a, s_carry[2] = b, s_carry[3] = c;
    __syncthreads();
    items += s_carry[1], slots += s_carry[2], units += s_carry[3];
  }
  if (tid == 0) {
    p.head->items = (int)items;
    p.head->split_keys = split;
    p.head->q_begin = q_begin;
    p.head->q_end = (int)end;
  }
}

// ---------------------------------------------------------------------------
// 16 rows of a KV head over a part of the keys, by mma.sync
// ---------------------------------------------------------------------------

constexpr int kStep = 16;      // keys of a warp's step
constexpr int kRowWarps = 8;
constexpr int kRowThreads = kRowWarps * 32;
constexpr int kRows = 16;
// A row's maximum moves when a step exceeds it by more than 2^kLazy, and p is kept times
// 2^kPShift, at most 2^15 in fp16, times its key's V scale over a power of two above the
// warp's largest: fp16's smallest step, 2^-24, is then 2^-37 of the row's largest p.
constexpr float kLazy = 2.0f;
constexpr float kPShift = 13.0f;

template <int DP, int HALVES, bool PV>
struct RowsCfg {
  static constexpr int kStages = 3;
  static constexpr int kCodeBytes = (PV ? 2 : 1) * kStep * DP;  // K, then V
  static constexpr int kStageBytes = kCodeBytes + 2 * kStep * 4 + 16;  // scales, which keys count
  static constexpr int kRingBytes = kStages * kStageBytes;             // of a warp
  static constexpr int kPitch = DP + 4;  // floats of a row of results
  static constexpr int kOffQ = kRowWarps * kRingBytes;
  static constexpr int kOffMl = kOffQ + HALVES * DP / 16 * 512;
  static constexpr int kOffMisc = kOffMl + kRowWarps * kRows * 8;
  static constexpr int kSmemBytes = kOffMisc + kRows * 4 + 16;
  static constexpr int kSlotO = PV ? kRows * DP * 4 : 0;
  static constexpr int kSlotBytes = kSlotO + kRows * 8;
  static_assert(!PV || kRows * kPitch * 4 <= kRingBytes, "results of a warp take its ring's place");
  static_assert(kSmemBytes <= 227 * 1024, "shared memory");
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
  const PlanHead* head;
  const PlanSeq* seq;
  int* counters;
  uint8_t* slots;
  int64_t q_tok, q_head;  // strides, elements
  int64_t num_blocks;
  int seqs, total_q, heads, kv_heads, group, dim, bs, width;
  float qk_scale;  // sm_scale log2e
};

// Without PV only the denominators are taken (p.lse).
template <typename T, int DP, int HALVES, bool PV>
__global__ void __launch_bounds__(kRowThreads, PV && DP > 128 ? 1 : 2)
    rows_kernel(const RowsParams p, int* err) {
  using C = RowsCfg<DP, HALVES, PV>;
  constexpr int kPieces = DP / 16;              // 16-byte pieces of a key's codes
  constexpr int kPasses = kPieces * kStep / 32; // copies a lane makes of K or V
  constexpr int kQuads = PV ? DP / 4 : 1;       // of a row's results
  constexpr int kTiles = PV ? DP / 8 : 0;       // accumulators of 8 channels
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * C::kRingBytes;
  uint4* s_q = reinterpret_cast<uint4*>(smem + C::kOffQ);
  float2* s_ml = reinterpret_cast<float2*>(smem + C::kOffMl);  // [warp][row]
  float* s_factor = reinterpret_cast<float*>(smem + C::kOffMisc);
  int* s_last = reinterpret_cast<int*>(smem + C::kOffMisc + kRows * 4);

  // rows in front of the first and behind the last sequence become zero
  const int64_t front = (int64_t)p.head->q_begin * p.heads;
  const int64_t behind = (int64_t)p.head->q_end * p.heads;
  const int64_t outside = front + (int64_t)p.total_q * p.heads - behind;
  for (int64_t i = blockIdx.x * kRowWarps + warp; i < outside; i += gridDim.x * kRowWarps) {
    const int64_t r = i < front ? i : behind + i - front;
    for (int c = lane * 4; PV && c < p.dim; c += 128)
      store4(static_cast<T*>(p.out) + r * p.dim + c, make_float4(0, 0, 0, 0));
    if (lane == 0 && p.lse != nullptr) p.lse[r] = -INFINITY;
  }

  const int items = p.head->items, split_keys = p.head->split_keys;
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const int s = plan_find(p.seq, p.seqs, item);
    const PlanSeq seq = p.seq[s];
    // KV heads next to one another share pages; then row blocks, then parts
    const int local = item - seq.first;
    const int kvh = local % p.kv_heads;
    const int blocks = (int)((seq.lq * (int64_t)p.group + kRows - 1) / kRows);
    const int unit = local % (p.kv_heads * blocks);
    const int block = unit / p.kv_heads, part = local / (p.kv_heads * blocks);
    const int rows = (int)min((int64_t)kRows, seq.lq * (int64_t)p.group - (int64_t)block * kRows);
    // keys that row r sees: those below its token's place, counted from the end
    const auto limit_of = [&](int r) {
      return r < rows ? (int)((block * (int64_t)kRows + r) / p.group) + 1 + seq.len - seq.lq : 0;
    };
    const int k0 = part * split_keys;
    const int k1 = min(min(seq.len, k0 + split_keys), limit_of(rows - 1));
    const int steps = k1 > k0 ? (k1 - k0 + kStep - 1) / kStep : 0;
    const int32_t* table = p.tables + (int64_t)s * p.width;

    // Step i of this warp is keys k0 + (i kRowWarps + warp) kStep and on.  Lanes 0-15 find
    // its keys' rows, a step ahead; entry and rem are those of the next step to copy.
    const int mine = steps > warp ? (steps - warp - 1) / kRowWarps + 1 : 0;
    const auto key_of = [&](int i) { return k0 + (i * kRowWarps + warp) * kStep; };
    int entry = -1, rem = 0;
    const auto look_up = [&](int i) {
      const int key = key_of(i) + (lane & 15);
      const int page = key / p.bs;
      rem = key - page * p.bs;
      entry = key < k1 ? table[page] : -1;
    };
    const auto issue = [&](int i) {
      if (i < mine) {
        uint8_t* stage = ring + (i % C::kStages) * C::kStageBytes;
        const bool counts = key_of(i) + (lane & 15) < k1;
        const bool good = counts && entry >= 0 && (int64_t)entry < p.num_blocks;
        if (counts && !good) record_error(err, kDevBadBlockId);
        const uint32_t at = good ? (uint32_t)entry * p.bs + rem : 0xffffffffu;
        const float* scale = lane < 16 ? p.k_scale : p.v_scale;
        if (PV || lane < 16) copy4_if(good, smem_u32(stage + C::kCodeBytes + lane * 4),
                 scale + (good ? (int64_t)entry * p.kv_heads + kvh : 0));
        const unsigned mask = __ballot_sync(0xffffffffu, good);
        if (lane == 0) *reinterpret_cast<uint32_t*>(stage + C::kCodeBytes + 128) = mask & 0xffffu;
#pragma unroll
        for (int c = 0; c < kPasses; ++c) {
          const int key = (c * 32 + lane) / kPieces, piece = lane % kPieces;
          const uint32_t row = __shfl_sync(0xffffffffu, at, key);
          const bool on = row != 0xffffffffu && piece * 16 < p.dim;
          const int64_t from =
              on ? ((int64_t)row * p.kv_heads + kvh) * p.dim + piece * 16 : 0;
          const uint32_t to = smem_u32(stage + key * DP + piece_at<DP>(key, piece) * 16);
          copy16_if(on, to, p.k_cache + from);
          if constexpr (PV) copy16_if(on, to + kStep * DP, p.v_cache + from);
        }
        if (i + 1 < mine) look_up(i + 1);
      }
      copies_commit();
    };
    if (mine > 0) look_up(0);
#pragma unroll
    for (int i = 0; i < C::kStages - 1; ++i) issue(i);

    stage_queries<T, DP, HALVES>(s_q, s_factor, p.dim, warp, kRowWarps, [&](int r) -> const T* {
      if (r >= rows) return nullptr;
      const int64_t i = block * (int64_t)kRows + r;
      const int tok = (int)(i / p.group);
      return static_cast<const T*>(p.q) + (seq.q0 + tok) * p.q_tok +
             (kvh * p.group + (int)(i - (int64_t)tok * p.group)) * p.q_head;
    });
    __syncthreads();
    const float f0 = s_factor[g] * p.qk_scale, f1 = s_factor[g + 8] * p.qk_scale;
    const int limit0 = limit_of(g), limit1 = limit_of(g + 8);
    const int clear = limit_of(0);  // every row sees the keys below

    float o[PV ? kTiles : 1][4];
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
    int unit_e = -127;  // O is in units of 2^unit_e (of V scales) / 2^kPShift

    for (int i = 0; i < mine; ++i) {
      copies_wait<C::kStages - 2>();
      __syncwarp();
      issue(i + C::kStages - 1);
      const uint8_t* stage = ring + (i % C::kStages) * C::kStageBytes;
      const float* scales = reinterpret_cast<const float*>(stage + C::kCodeBytes);
      const uint32_t mask = *reinterpret_cast<const uint32_t*>(stage + C::kCodeBytes + 128);
      // scores: rows g, g + 8; keys 8 n + 2 t, 8 n + 2 t + 1
      float sc[2][HALVES][4] = {};
#pragma unroll
      for (int pc = 0; pc < DP / 64; ++pc) {
        uint4 w[2];
#pragma unroll
        for (int n = 0; n < 2; ++n)
          w[n] = *reinterpret_cast<const uint4*>(stage + (n * 8 + g) * DP +
                                                 piece_at<DP>(n * 8 + g, pc * 4 + t) * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint2 b[2];
#pragma unroll
          for (int n = 0; n < 2; ++n)
            b[n] = codes_to_half(e == 0 ? w[n].x : e == 1 ? w[n].y : e == 2 ? w[n].z : w[n].w);
#pragma unroll
          for (int h = 0; h < HALVES; ++h) {
            const uint4 a = s_q[(h * (DP / 16) + pc * 4 + e) * 32 + lane];
#pragma unroll
            for (int n = 0; n < 2; ++n) mma_f16(sc[n][h], a, b[n].x, b[n].y);
          }
        }
      }
      float y[2][4];
      float vs[2][2];
      const int key0 = key_of(i) + 2 * t;
      const bool all = mask == 0xffffu && key_of(i) + kStep <= clear;
      uint32_t vmax = 0u;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float2 ks = *reinterpret_cast<const float2*>(scales + n * 8 + 2 * t);
        float2 v = make_float2(0.0f, 0.0f);
        if constexpr (PV) v = *reinterpret_cast<const float2*>(scales + kStep + n * 8 + 2 * t);
        vs[n][0] = v.x;
        vs[n][1] = v.y;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = sc[n][0][e];
          if constexpr (HALVES == 2) x += sc[n][1][e];
          y[n][e] = x * ((e & 1) ? ks.y : ks.x) * (e < 2 ? f0 : f1);
        }
        const uint32_t a = __float_as_uint(fabsf(v.x)), b = __float_as_uint(fabsf(v.y));
        vmax = max(vmax, max(a < 0x7f800000u ? a : 0u, b < 0x7f800000u ? b : 0u));
      }
      const auto seen = [&](int n, int e) {
        const int key = n * 8 + (e & 1);  // + 2 t
        return (mask >> (key + 2 * t) & 1u) && key0 + key < (e < 2 ? limit0 : limit1);
      };
      if (!all) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!seen(n, e)) y[n][e] = -INFINITY;
      }
      if constexpr (PV) vmax = __reduce_max_sync(0xffffffffu, vmax);
      float t0 = fmaxf(fmaxf(y[0][0], y[0][1]), fmaxf(y[1][0], y[1][1]));
      float t1 = fmaxf(fmaxf(y[0][2], y[0][3]), fmaxf(y[1][2], y[1][3]));
#pragma unroll
      for (int x = 1; x <= 2; x <<= 1) {
        t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, x));
        t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, x));
      }
      // power of two above the V scales, so that p times scale stays in fp16
      const int e_now = (int)(vmax >> 23) - 126;
      const bool grow = vmax != 0u && e_now > unit_e;
      const bool move0 = t0 > m0 + kLazy || (m0 == -INFINITY && t0 > m0);
      const bool move1 = t1 > m1 + kLazy || (m1 == -INFINITY && t1 > m1);
      if (__any_sync(0xffffffffu, move0 || move1) || grow) {
        const float a0 = move0 ? ex2(m0 - t0) : 1.0f, a1 = move1 ? ex2(m1 - t1) : 1.0f;
        if (move0) m0 = t0;
        if (move1) m1 = t1;
        l0 *= a0;
        l1 *= a1;
        float down = 1.0f;
        if (grow) {
          down = unit_e - e_now < -126 ? 0.0f : power_of_two(unit_e - e_now);
          unit_e = e_now;
        }
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
          o[n][0] *= a0 * down;
          o[n][1] *= a0 * down;
          o[n][2] *= a1 * down;
          o[n][3] *= a1 * down;
        }
      }
      const float base0 = m0 == -INFINITY ? 0.0f : m0 - kPShift;
      const float base1 = m1 == -INFINITY ? 0.0f : m1 - kPShift;
      const float inv_unit = power_of_two(-max(unit_e, -126));
      uint32_t hi[2][2], lo[2][2] = {};  // [n][rows g, g + 8]
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float x0 = ex2(y[n][2 * r] - (r ? base1 : base0));
          const float x1 = ex2(y[n][2 * r + 1] - (r ? base1 : base0));
          (r ? l1 : l0) += x0 + x1;
          if constexpr (!PV) continue;
          float z0 = x0 * (vs[n][0] * inv_unit), z1 = x1 * (vs[n][1] * inv_unit);
          if (!all) {
            if (!seen(n, 2 * r)) z0 = 0.0f;
            if (!seen(n, 2 * r + 1)) z1 = 0.0f;
          }
          const __half2 h = __floats2half2_rn(z0, z1);
          hi[n][r] = word_of(h);
          if constexpr (HALVES == 2) {
            const float2 b = __half22float2(h);
            lo[n][r] = word_of(__floats2half2_rn(z0 - b.x, z1 - b.y));
          }
        }
      if constexpr (!PV) continue;
      const uint4 pa = make_uint4(hi[0][0], hi[0][1], hi[1][0], hi[1][1]);
      const uint4 pb = HALVES == 2 ? make_uint4(lo[0][0], lo[0][1], lo[1][0], lo[1][1]) : pa;
      // O: channel c * 128 + g * 16 + 4 w + e of V is column g of accumulator
      // c * 16 + 4 w + e (of 64 channels: g * 8 + 4 w + e)
      const uint8_t* vt = stage + kStep * DP;
      constexpr int kWords = DP >= 128 ? 4 : 2;
#pragma unroll
      for (int c = 0; c < (DP + 127) / 128; ++c) {
        uint32_t w[4][kWords];  // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int key = 2 * t + (k & 1) + (k >> 1) * 8;
          if constexpr (DP >= 128) {
            const uint4 x = *reinterpret_cast<const uint4*>(vt + key * DP +
                                                            piece_at<DP>(key, c * 8 + g) * 16);
            w[k][0] = x.x, w[k][1] = x.y, w[k][2 % kWords] = x.z, w[k][3 % kWords] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(
                vt + key * DP + piece_at<DP>(key, g >> 1) * 16 + (g & 1) * 8);
            w[k][0] = x.x, w[k][1] = x.y;
          }
        }
#pragma unroll
        for (int x = 0; x < kWords; ++x) {
          const uint2 b01 = codes_to_half(__byte_perm(w[0][x], w[1][x], 0x5140));
          const uint2 b23 = codes_to_half(__byte_perm(w[0][x], w[1][x], 0x7362));
          const uint2 c01 = codes_to_half(__byte_perm(w[2][x], w[3][x], 0x5140));
          const uint2 c23 = codes_to_half(__byte_perm(w[2][x], w[3][x], 0x7362));
          const int at = c * 16 + x * 4;
          mma_f16(o[at], pa, b01.x, c01.x);
          mma_f16(o[at + 1], pa, b01.y, c01.y);
          mma_f16(o[at + 2], pa, b23.x, c23.x);
          mma_f16(o[at + 3], pa, b23.y, c23.y);
          if constexpr (HALVES == 2) {
            mma_f16(o[at], pb, b01.x, c01.x);
            mma_f16(o[at + 1], pb, b01.y, c01.y);
            mma_f16(o[at + 2], pb, b23.x, c23.x);
            mma_f16(o[at + 3], pb, b23.y, c23.y);
          }
        }
      }
    }
    copies_wait<0>();
    __syncwarp();
    // The warps' results meet in shared memory, each in its own ring.
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, x);
      l1 += __shfl_xor_sync(0xffffffffu, l1, x);
    }
    if (t == 0) {
      s_ml[warp * kRows + g] = make_float2(m0, l0);
      s_ml[warp * kRows + g + 8] = make_float2(m1, l1);
    }
    if (PV && mine > 0) {
      const float up = power_of_two(max(unit_e, -126));
      float* mine_o = reinterpret_cast<float*>(ring);
      constexpr int kRun = DP >= 128 ? 16 : 8;  // consecutive channels of a column
#pragma unroll
      for (int c = 0; c < (DP + 127) / 128; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float* to = mine_o + (g + (e >> 1) * 8) * C::kPitch + c * 128 + (2 * t + (e & 1)) * kRun;
#pragma unroll
          for (int x = 0; x < kRun; x += 4)
            *reinterpret_cast<float4*>(to + x) =
                make_float4(o[c * 16 + x][e] * up, o[c * 16 + x + 1][e] * up,
                            o[c * 16 + x + 2][e] * up, o[c * 16 + x + 3][e] * up);
        }
    }
    __syncthreads();
    const bool whole = seq.splits == 1;
    uint8_t* slot = p.slots + (int64_t)(seq.slot + local) * C::kSlotBytes;
    // O, m, l of row r over the parts given by get(i) -> (m, l), at(i) -> O
    const auto store_row = [&](int r, int c, float4 acc, float m, float l) {
      const int64_t i = block * (int64_t)kRows + r;
      const int tok = (int)(i / p.group);
      const int64_t to = (int64_t)(seq.q0 + tok) * p.heads + kvh * p.group + (i - (int64_t)tok * p.group);
      const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
      if (PV && c < p.dim)
        store4(static_cast<T*>(p.out) + to * p.dim + c,
               l == 0.0f ? make_float4(0, 0, 0, 0)
                         : make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
      if (c == 0 && p.lse != nullptr)
        p.lse[to] = l == 0.0f ? -INFINITY : (m - kPShift + log2f(l)) * (1.0f / kLog2e);
    };
    const int live = min(kRowWarps, steps);
    for (int x = tid; x < rows * kQuads; x += kRowThreads) {
      const int r = x / kQuads, c = x % kQuads * 4;
      float m = -INFINITY, l = 0.0f;
      for (int w = 0; w < live; ++w) m = fmaxf(m, s_ml[w * kRows + r].x);
      float4 acc = make_float4(0, 0, 0, 0);
      for (int w = 0; w < live; ++w) {
        const float2 ml = s_ml[w * kRows + r];
        // (a warp without a score above -inf has l = 0 and O = 0, or a NaN)
        const float f = ml.x == -INFINITY ? 1.0f : ex2(ml.x - m);
        l += ml.y * f;
        if constexpr (PV) {
          const float4 v = *reinterpret_cast<const float4*>(
              reinterpret_cast<const float*>(smem + w * C::kRingBytes) + r * C::kPitch + c);
          acc.x += v.x * f, acc.y += v.y * f, acc.z += v.z * f, acc.w += v.w * f;
        }
      }
      if (whole) {
        store_row(r, c, acc, m, l);
      } else {
        if constexpr (PV) *reinterpret_cast<float4*>(slot + (r * DP + c) * 4) = acc;
        if (c == 0) *reinterpret_cast<float2*>(slot + C::kSlotO + r * 8) = make_float2(m, l);
      }
    }
    __syncthreads();  // the slot is written; the ring and s_q are free
    if (whole) continue;
    const int units = p.kv_heads * blocks;
    if (tid == 0)
      *s_last = atomic_add_acq_rel_gpu(&p.counters[seq.unit + unit], 1) == seq.splits - 1;
    __syncthreads();
    if (!*s_last) continue;
    // the last part to end joins all of them, in order
    const uint8_t* first = p.slots + (int64_t)(seq.slot + unit) * C::kSlotBytes;
    const int64_t pitch = (int64_t)units * C::kSlotBytes;
    for (int x = tid; x < rows * kQuads; x += kRowThreads) {
      const int r = x / kQuads, c = x % kQuads * 4;
      float m = -INFINITY, l = 0.0f;
      float4 acc = make_float4(0, 0, 0, 0);
      for (int i = 0; i < seq.splits; ++i) {
        const float2 ml =
            __ldcg(reinterpret_cast<const float2*>(first + i * pitch + C::kSlotO + r * 8));
        if (ml.x == -INFINITY && ml.y == 0.0f) continue;
        float4 v = make_float4(0, 0, 0, 0);
        if constexpr (PV)
          v = __ldcg(reinterpret_cast<const float4*>(first + i * pitch + (r * DP + c) * 4));
        const float big = fmaxf(m, ml.x);
        const float f = m == -INFINITY ? 1.0f : ex2(m - big);
        const float k = ml.x == -INFINITY ? 1.0f : ex2(ml.x - big);
        m = big;
        l = l * f + ml.y * k;
        acc.x = acc.x * f + v.x * k, acc.y = acc.y * f + v.y * k;
        acc.z = acc.z * f + v.z * k, acc.w = acc.w * f + v.w * k;
      }
      store_row(r, c, acc, m, l);
    }
    __syncthreads();
  }
}

// Items to aim at where sequences are split: a few for every place on the card, so
// that unequal ones even out.
constexpr int kTarget = 148 * 2 * 3;
constexpr int kLeast = 256;

struct ChunkLayout {
  size_t head, seq, counters, slots, total;
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
  l.head = take(sizeof(PlanHead));
  l.seq = take(sizeof(PlanSeq) * (size_t)a.seqs);
  l.counters = take(sizeof(int) * 2 * kTarget);
  // without a table wider than the smallest part nothing is split
  const bool splits = (int64_t)a.width * a.block_size > kLeast;
  const size_t slot = (a.v_cache != nullptr ? kRows * dp * 4 : 0) + kRows * 8;
  l.slots = take(splits ? (size_t)2 * kTarget * slot : 0);
  l.total = at + 256;
  return l;
}

template <typename T, int DP, bool PV>
int launch_rows(const ChunkArgs& a, uint8_t* ws, cudaStream_t stream) {
  constexpr int HALVES = sizeof(T) == 4 ? 2 : 1;
  using C = RowsCfg<DP, HALVES, PV>;
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
  p.head = reinterpret_cast<PlanHead*>(ws + lay.head);
  p.seq = reinterpret_cast<PlanSeq*>(ws + lay.seq);
  p.counters = reinterpret_cast<int*>(ws + lay.counters);
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
  p.qk_scale = a.sm_scale * kLog2e;
  PlanArgs plan;
  plan.cu = a.cu;
  plan.lens = a.lens;
  plan.seqs = a.seqs;
  plan.total_q = (int)a.total_q;
  plan.group = p.group;
  plan.kv_heads = a.kv_heads;
  plan.block_size = a.block_size;
  plan.width = a.width;
  plan.rows = kRows;
  plan.target = kTarget;
  plan.least = kLeast;
  plan.round = kStep;
  plan.head = reinterpret_cast<PlanHead*>(ws + lay.head);
  plan.seq = reinterpret_cast<PlanSeq*>(ws + lay.seq);
  plan.counters = p.counters;
  plan.counts = 2 * kTarget;
  int* err = device_error_word();
  const int rc = launch_plan(plan, err, stream);
  if (rc != kOk) return rc;
  auto kern = rows_kernel<T, DP, HALVES, PV>;
  static std::atomic<uint64_t> done{0};
  allow_shared_memory(reinterpret_cast<const void*>(kern), C::kSmemBytes, done);
  const int64_t units = (a.total_q * p.group / kRows + std::min<int64_t>(a.seqs, a.total_q) + 1) * a.kv_heads;
  const int64_t parts = (int64_t)a.width * a.block_size / kLeast + 1;
  const int64_t most = 148 * (PV && DP > 128 ? 1 : 2);
  kern<<<(unsigned)std::min(most, units * std::min<int64_t>(parts, most)), kRowThreads, C::kSmemBytes, stream>>>(p, err);
  return kOk;
}

}  // namespace

int launch_plan(const PlanArgs& a, int* err, cudaStream_t stream) {
  plan_kernel<<<1, kPlanThreads, 0, stream>>>(a, err);
  return kOk;
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
  const auto with_dim = [&](auto t) {
    using T = decltype(t);
    const auto with = [&](auto dp) {
      constexpr int DP = decltype(dp)::value;
      return a.v_cache != nullptr ? launch_rows<T, DP, true>(a, ws, stream)
                                  : launch_rows<T, DP, false>(a, ws, stream);
    };
    return a.dim <= 64    ? with(std::integral_constant<int, 64>{})
           : a.dim <= 128 ? with(std::integral_constant<int, 128>{})
                          : with(std::integral_constant<int, 256>{});
  };
  const int rc = a.dtype == 0 ? with_dim(0.0f) : a.dtype == 1 ? with_dim(__half()) : with_dim(__nv_bfloat16());
  if (rc != kOk) return rc;
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_error(std::string("chunk attention launch failed: ") + cudaGetErrorString(e));
    return kCudaError;
  }
  return kOk;
}

}  // namespace pkv
