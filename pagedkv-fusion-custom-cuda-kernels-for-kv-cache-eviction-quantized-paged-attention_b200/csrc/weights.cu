// Attention weights gathered per cached token: what the eviction statistics are made of.
//
//   weights[page(j), offset(j)] += 1/H sum over the call's tokens i and heads h of
//                                  exp(scale q[i, h] . k_j - lse[i, h]),  j <= i + L - Lq
//
// with lse as the attention gave it, or taken first by the attention's own kernels.
//
//   gather_tc_kernel  (weights_tc.cu) pages of a multiple of 16 tokens, head_dim up to 128;
//   gather_kernel     the others: an item is (sequence, KV head, 256 keys, at most 1,024
//                     query rows); a warp keeps 32 keys as fragments in registers and lets
//                     the rows pass, 16 at a time, from shared memory;
//   finish_kernel     few rows a sequence without lse: from the scores of the attention's
//                     pass;
//   spread_kernel     adds the sums to the weights.
//
// Sums of several items, and of sequences that share pages, meet as integers of 2^-37
// in a workspace, so that the order of their arrival changes nothing: a weight is then off
// by half a step for each of them, 2^-38.
#include <cuda_runtime.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "chunk.h"
#include "weights.h"

namespace pkv {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kWarpKeys = 32;
constexpr int kKeys = kWarps * kWarpKeys;  // of an item
constexpr int kItemRows = 1024;            // fp32 sums of 64 values a lane, then exact
struct GatherParams {
  const void* q;
  const int8_t* k_cache;
  const float* k_scale;
  const int32_t* tables;
  const float* lse;
  const PlanHead* head;
  const PlanSeq* seq;
  unsigned long long* sums;  // [num_blocks, block_size], zero for pages in the tables
  int64_t q_tok, q_head;
  int64_t num_blocks;
  int seqs, heads, kv_heads, group, dim, bs, width;
  float qk_scale;
};

template <typename T, int DP, int HALVES>
__global__ void __launch_bounds__(kThreads, DP > 128 ? 1 : 2) gather_kernel(const GatherParams p, int* err) {
  constexpr int kSteps = DP / 16;
  constexpr int kTiles = kWarpKeys / 16;
  constexpr int kPass = 16;  // rows at a time
  __shared__ uint2 s_q[kPass / 8 * HALVES * kSteps * 32];
  __shared__ float s_factor[kPass], s_start[kPass], s_lse[kPass];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  launch_the_next();
  behind_the_last();
  const int64_t items = p.head->places;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int s = plan_find(p.seq, p.seqs, item);
    const PlanSeq seq = p.seq[s];
    const int unit = (int)((item - seq.first) / seq.steps);
    const int part = (int)(item - seq.first) - unit * seq.steps;
    const int kvh = unit % p.kv_heads, chunk = unit / p.kv_heads;
    const int64_t all_rows = seq.lq * (int64_t)p.group;
    const int k0 = part * kKeys + warp * kWarpKeys;  // of this warp
    const int shift = seq.len - seq.lq;
    const int32_t* table = p.tables + (int64_t)s * p.width;
    // rows of this item that see the item's first key
    const int64_t r_end = min(all_rows, (chunk + 1) * (int64_t)kItemRows);
    const int64_t r_first = max((int64_t)(part * kKeys - shift), (int64_t)0) * p.group;
    const int64_t r_begin = max(chunk * (int64_t)kItemRows, r_first / kPass * kPass);

    // this warp's keys: lane = key, then fragments
    const int key = k0 + lane, page = key / p.bs;
    const bool counts = key < seq.len;
    const int phys = counts ? table[page] : -1;
    const bool good = counts && phys >= 0 && (int64_t)phys < p.num_blocks;
    if (counts && !good) record_error(err, kDevBadBlockId);
    const uint32_t at = good ? (uint32_t)phys * p.bs + (key - page * p.bs) : 0xffffffffu;
    const float ks = good ? p.k_scale[(int64_t)phys * p.kv_heads + kvh] * p.qk_scale : 0.0f;
    const unsigned mask = __ballot_sync(0xffffffffu, good);
    uint4 a[kTiles][kSteps];
    float scale[kTiles][2];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      uint4 w[2][DP / 64];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint32_t row = __shfl_sync(0xffffffffu, at, n * 16 + r * 8 + g);
        scale[n][r] = __shfl_sync(0xffffffffu, ks, n * 16 + r * 8 + g);
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
          const int piece = c * 4 + t;
          w[r][c] = make_uint4(0, 0, 0, 0);
          if (row != 0xffffffffu && piece * 16 < p.dim)
            w[r][c] = __ldg(reinterpret_cast<const uint4*>(
                p.k_cache + ((int64_t)row * p.kv_heads + kvh) * p.dim + piece * 16));
        }
      }
#pragma unroll
      for (int c = 0; c < DP / 64; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const auto word = [&](const uint4& v) { return e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w; };
          const uint2 x = codes_plus_128(word(w[0][c])), y = codes_plus_128(word(w[1][c]));
          a[n][c * 4 + e] = make_uint4(x.x, y.x, x.y, y.y);
        }
    }
    float sum[kTiles][2] = {};  // keys g and g + 8
    for (int64_t r0 = r_begin; r0 < r_end; r0 += kPass) {
      const int rows = (int)min((int64_t)kPass, r_end - r0);
      __syncthreads();  // the last rows are used
      stage_queries<T, DP, HALVES>(
          s_q, s_factor, s_start, p.dim, kPass, warp, kWarps, [&](int r) -> const T* {
            if (r >= rows) return nullptr;
            const int tok = (int)((r0 + r) / p.group);
            return static_cast<const T*>(p.q) + (seq.q0 + tok) * p.q_tok +
                   (kvh * p.group + (int)(r0 + r - (int64_t)tok * p.group)) * p.q_head;
          });
      if (tid < kPass) {
        float v = -INFINITY;
        if (tid < rows) {
          const int tok = (int)((r0 + tid) / p.group);
          v = p.lse[(int64_t)(seq.q0 + tok) * p.heads + kvh * p.group + (r0 + tid - (int64_t)tok * p.group)];
        }
        s_lse[tid] = v;
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < kPass / 8; ++u) {
        if (u * 8 >= rows) break;
        float d[kTiles][4];
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) d[n][e] = s_start[u * 8 + 2 * t + (e & 1)];
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
          for (int h = HALVES - 1; h >= 0; --h) {
            const uint2 b = s_q[((u * HALVES + h) * kSteps + k) * 32 + lane];
#pragma unroll
            for (int n = 0; n < kTiles; ++n) mma_f16(d[n], a[n][k], b.x, b.y);
          }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = u * 8 + 2 * t + e;
          const float lse = s_lse[row], f = s_factor[row];
          // a row without keys (lse -inf) adds nothing
          const bool none = row >= rows || lse == -INFINITY;
          const int limit = none ? 0 : (int)((r0 + row) / p.group) + 1 + shift;
          const float base = none ? 0.0f : lse * kLog2e;
#pragma unroll
          for (int n = 0; n < kTiles; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const int at_key = n * 16 + r * 8 + g;
              const float x = ex2(fmaf(d[n][2 * r + e], scale[n][r] * f, -base));
              sum[n][r] += (mask >> at_key & 1u) && k0 + at_key < limit ? x : 0.0f;
            }
        }
      }
    }
    // the lanes of a key, then one adds
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        sum[n][r] += __shfl_xor_sync(0xffffffffu, sum[n][r], 1);
        sum[n][r] += __shfl_xor_sync(0xffffffffu, sum[n][r], 2);
        const uint32_t slot = __shfl_sync(0xffffffffu, at, n * 16 + r * 8 + g);
        if (t == 0 && slot != 0xffffffffu && r_begin < r_end) {
          add_weight(p.sums + slot, sum[n][r]);
        }
      }
  }
}

// The scores that the attention's kernel left (in powers of two), to weights, for calls of few
// rows, whose scores are a small part of the keys' bytes.  A lane has N cached tokens next to
// one another (4 where a table's tokens are a multiple of it: 16 bytes a load), a warp every
// eighth row: what bounds it is how many loads are under way (a thread for a token and all
// rows took 16 us for the 34 MB of 64 sequences, this 8 us).
template <int N>
__global__ void __launch_bounds__(256) finish_kernel(const GatherParams p, const float* logits,
                                                     int64_t slots) {
  __shared__ float s_sum[8][32 * N];
  launch_the_next();
  behind_the_last();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t per_seq = (int64_t)p.width * p.bs;
  for (int64_t i0 = blockIdx.x * (32ll * N); i0 < slots; i0 += gridDim.x * (32ll * N)) {
    const int64_t i = i0 + lane * N;
    float sum[N] = {};
    if (i < slots) {
      const int s = slots <= 0x7fffffff ? (int)i / (int)per_seq : (int)(i / per_seq);
      const int at = (int)(i - s * per_seq);
      const PlanSeq seq = p.seq[s];
      if (at < seq.len) {
        // the token's rows, and of those the first that sees each of the N (rows are below 2^25)
        const int r0 = seq.q0 * p.heads, r1 = r0 + seq.lq * p.heads;
        int from[N];
#pragma unroll
        for (int e = 0; e < N; ++e)
          from[e] = (int)min((int64_t)r0 + max(at + e - (seq.len - seq.lq), 0) * (int64_t)p.heads, (int64_t)r1);
#pragma unroll 4
        for (int r = from[0] + warp; r < r1; r += 8) {
          const float lse = p.lse[r], base = lse * kLog2e;
          float x[N];
          if constexpr (N == 4) *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(logits + r * per_seq + at);
          else x[0] = logits[r * per_seq + at];
#pragma unroll
          for (int e = 0; e < N; ++e) sum[e] += r >= from[e] && lse != -INFINITY ? ex2(x[e] - base) : 0.0f;
        }
      }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) s_sum[warp][lane * N + e] = sum[e];
    __syncthreads();
    const int64_t mine = i0 + threadIdx.x;
    if (threadIdx.x < 32 * N && mine < slots) {
      const int64_t s = mine / per_seq;
      const int at = (int)(mine - s * per_seq);
      const PlanSeq seq = p.seq[s];
      const int page = at / p.bs, phys = at < seq.len && seq.lq > 0 ? p.tables[s * p.width + page] : -1;
      if (phys >= 0 && (int64_t)phys < p.num_blocks) {
        float all = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) all += s_sum[w][threadIdx.x];
        add_weight(p.sums + (int64_t)phys * p.bs + (at - page * p.bs), all);
      }
    }
    __syncthreads();
  }
}

// Adds the sums to the weights.  A page may be in several tables: whoever comes first
// takes its sum and leaves a zero.
__global__ void __launch_bounds__(256) spread_kernel(const int32_t* tables, const int32_t* lens,
                                                     unsigned long long* sums, float* weights,
                                                     int64_t num_blocks, int bs, int width,
                                                     int64_t slots, float inv_heads) {
  behind_the_last();
  const int64_t per_seq = (int64_t)width * bs;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < slots; i += gridDim.x * 256ll) {
    const int64_t s = i / per_seq;
    const int at = (int)(i - s * per_seq);
    if (at >= lens[s]) continue;
    const int page = at / bs, phys = tables[s * width + page];
    if (phys < 0 || (int64_t)phys >= num_blocks) continue;
    const int64_t slot = (int64_t)phys * bs + (at - page * bs);
    const unsigned long long u = atomicExch(sums + slot, 0ull);
    if (u != 0)
      weights[slot] += u & kNotFinite ? __int_as_float(0x7fffffff)
                                      : (float)((double)u * (1.0 / (double)kWeightUnit)) * inv_heads;
  }
}

// How a call's denominators and scores come.  Calls of few rows a sequence (decode) whose
// log denominators are not given leave their scores too, so that the keys are read once
// (64 sequences of 2,050 tokens, 32 / 8 heads: 131 MB of keys, 34 MB of scores written and
// read); the others' come from a pass of the attention (its V the keys', where that is the
// tensor-memory kernel: 512 tokens over 4,096 take 113 us, with their denominators 43).
constexpr int64_t kMostScores = 128ll << 20;  // bytes
bool by_scores(const ChunkArgs& a) {
  const int64_t pitch = (int64_t)a.width * a.block_size;
  return a.lse == nullptr && a.total_q * (a.heads / a.kv_heads) <= 8 * (int64_t)a.seqs &&
         pitch <= kMostScores / 4 / (a.total_q * a.heads);
}
// The call that gives lse.
ChunkArgs inner_call(const ChunkArgs& a, float* lse, float* logits, void* out) {
  ChunkArgs b = a;
  b.lse = lse;
  b.logits = logits;
  b.out = out;
  const bool all = !by_scores(a) && chunk_tc_takes(a);
  b.v_cache = all ? (a.num_blocks > 0 ? a.k_cache : reinterpret_cast<const int8_t*>(16)) : nullptr;
  b.v_scale = all ? a.k_scale : nullptr;
  return b;
}

struct Layout {
  size_t head, seq, lse, sums, logits, out, inner, total;
};

Layout layout(const ChunkArgs& a) {
  Layout l;
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  const bool scores = by_scores(a), inner = a.lse == nullptr;
  const size_t rows = (size_t)a.total_q * a.heads;
  l.head = take(sizeof(PlanHead));
  l.seq = take(sizeof(PlanSeq) * (size_t)a.seqs);
  l.sums = take((size_t)a.num_blocks * a.block_size * 8);
  l.lse = take(inner ? rows * 4 : 0);
  l.logits = take(scores ? rows * a.width * a.block_size * 4 : 0);
  l.out = take(inner && !scores && chunk_tc_takes(a) ? rows * a.dim * (a.dtype == 0 ? 4 : 2) : 0);
  l.inner = at;
  if (inner) at += chunk_workspace_size(inner_call(a, nullptr, nullptr, nullptr));
  l.total = at + 256;
  return l;
}

GatherParams gather_params(const ChunkArgs& a, const float* lse, uint8_t* ws, const Layout& lay) {
  GatherParams p;
  p.q = a.q;
  p.k_cache = a.k_cache;
  p.k_scale = a.k_scale;
  p.tables = a.tables;
  p.lse = lse;
  p.head = reinterpret_cast<PlanHead*>(ws + lay.head);
  p.seq = reinterpret_cast<PlanSeq*>(ws + lay.seq);
  p.sums = reinterpret_cast<unsigned long long*>(ws + lay.sums);
  p.q_tok = a.q_token_stride;
  p.q_head = a.q_head_stride;
  p.num_blocks = a.num_blocks;
  p.seqs = a.seqs;
  p.heads = a.heads;
  p.kv_heads = a.kv_heads;
  p.group = a.heads / a.kv_heads;
  p.dim = a.dim;
  p.bs = a.block_size;
  p.width = a.width;
  p.qk_scale = a.sm_scale * kLog2e * kCodeUnit;
  return p;
}

template <typename T, int DP>
void launch_gather(const ChunkArgs& a, const GatherParams& p, int* err, cudaStream_t stream) {
  constexpr int HALVES = sizeof(T) == 4 ? 2 : 1;
  const int64_t parts = ((int64_t)a.width * a.block_size + kKeys - 1) / kKeys;
  const int64_t chunks = a.total_q * p.group / kItemRows + std::min<int64_t>(a.seqs, a.total_q);
  const int64_t most = 148 * (DP > 128 ? 1 : 2);
  const int64_t grid = std::min(most, std::min(most, parts) * chunks * a.kv_heads);
  launch_behind(gather_kernel<T, DP, HALVES>, dim3((unsigned)grid), kThreads, 0, stream, p, err);
}

}  // namespace

size_t accumulate_workspace_size(const ChunkArgs& a) {
  if (a.total_q == 0 || a.seqs == 0 || a.width == 0) return 0;
  return layout(a).total;
}

int launch_accumulate(const ChunkArgs& a, float* weights, void* workspace, size_t workspace_bytes,
                      cudaStream_t stream) {
  if (a.total_q == 0 || a.seqs == 0 || a.width == 0) return kOk;
  const Layout lay = layout(a);
  if (workspace == nullptr || workspace_bytes < lay.total) {
    set_error("workspace too small for accumulate_attention: need " + std::to_string(lay.total) +
              " bytes");
    return kWorkspace;
  }
  uint8_t* ws = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(workspace) + 255) &
                                           ~(uintptr_t)255);
  int* err = device_error_word();
  auto* sums = reinterpret_cast<unsigned long long*>(ws + lay.sums);
  const int64_t slots = (int64_t)a.seqs * a.width * a.block_size;
  ZeroArgs zero;
  zero.tables = a.tables;
  zero.lens = a.lens;
  zero.sums = sums;
  zero.num_blocks = a.num_blocks;
  zero.seqs = a.seqs;
  zero.block_size = a.block_size;
  zero.width = a.width;
  const float* lse = a.lse;
  const bool scores = by_scores(a);
  if (lse == nullptr) {
    float* logits = reinterpret_cast<float*>(ws + lay.logits);
    ChunkArgs b = inner_call(a, reinterpret_cast<float*>(ws + lay.lse), scores ? logits : nullptr,
                             ws + lay.out);
    if (scores) b.zero = zero;
    lse = b.lse;
    const int rc = launch_chunk(b, ws + lay.inner, chunk_workspace_size(b), stream);
    if (rc != kOk) return rc;
    if (scores) {
      GatherParams p = gather_params(a, lse, ws, lay);
      p.seq = chunk_plan(b, ws + lay.inner);
      const int n = (int64_t)a.width * a.block_size % 4 == 0 ? 4 : 1;
      const unsigned grid = (unsigned)std::min<int64_t>((slots + 32 * n - 1) / (32 * n), 148 * 8);
      launch_behind(n == 4 ? finish_kernel<4> : finish_kernel<1>, dim3(grid), 256, 0, stream, p, logits, slots);
    }
  }
  if (!scores) {
    PlanArgs plan;
    plan.cu = a.cu;
    plan.lens = a.lens;
    plan.seqs = a.seqs;
    plan.total_q = (int)a.total_q;
    plan.group = a.heads / a.kv_heads;
    plan.kv_heads = a.kv_heads;
    plan.block_size = a.block_size;
    plan.width = a.width;
    plan.rows = kItemRows;
    plan.step = kKeys;
    plan.over = 0;
    plan.workers = plan.least = 0;
    plan.which = kPlanAll;
    plan.few_rows = plan.few_steps = 0;
    plan.head = reinterpret_cast<PlanHead*>(ws + lay.head);
    plan.seq = reinterpret_cast<PlanSeq*>(ws + lay.seq);
    plan.counters = nullptr;
    plan.counts = 0;
    const bool tc = chunk_tc_takes(a);
    int rc = launch_plan(tc ? chunk_tc_plan(plan) : plan, nullptr, zero, err, stream);
    if (rc != kOk) return rc;
    const GatherParams p = gather_params(a, lse, ws, lay);
    const auto with_dim = [&](auto t) {
      using T = decltype(t);
      if (a.dim <= 64) launch_gather<T, 64>(a, p, err, stream);
      else if (a.dim <= 128) launch_gather<T, 128>(a, p, err, stream);
      else launch_gather<T, 256>(a, p, err, stream);
    };
    if (tc) rc = launch_gather_tc(a, lse, plan.head, plan.seq, sums, stream);
    else if (a.dtype == 0) with_dim(0.0f);
    else if (a.dtype == 1) with_dim(__half());
    else with_dim(__nv_bfloat16());
    if (rc != kOk) return rc;
  }
  const unsigned grid = (unsigned)std::min<int64_t>((slots + 255) / 256, 148 * 8);
  launch_behind(spread_kernel, dim3(grid), 256, 0, stream, a.tables, a.lens, sums, weights, a.num_blocks,
                a.block_size, a.width, slots, 1.0f / a.heads);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_error(std::string("accumulate launch failed: ") + cudaGetErrorString(e));
    return kCudaError;
  }
  return kOk;
}

}  // namespace pkv
