// Eviction of single tokens from the INT8 paged cache by the weights that they gathered.
//
// A sequence of more than `keep` tokens keeps its first `sinks`, its last `recent` and
// the heaviest of the others (of equal weights the earlier), `keep` in all, in order, at
// the front of its pages.  A page's new scale is the largest of its tokens' old ones, per
// KV head and for K and V apart; codes become rint(code (old / new)) where the old scale
// was smaller, and move as they are else.  The weights move along; the slots behind the
// last token that were in use get weight 0.
//
//   pick_kernel   a CTA per sequence: the weights' sort keys, the key that the last
//                 kept token has (radix, 8 bits a pass), the kept tokens in order;
//   move_kernel   a cluster per (sequence, K or V, KV head), and one per sequence for
//                 the weights.
//
// A kept token never moves back: those of the new pages [a, b) come from token a * bs
// or later.  The cluster therefore takes the new pages in rounds, reads all of a round's
// tokens, meets, and writes them: nothing that a later round reads is overwritten.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <string>

#include "pkv_common.cuh"
#include "pkv_internal.h"

namespace pkv {
namespace {

constexpr int kPickThreads = 1024;
constexpr int kKeysOnChip = 48 * 1024;  // sort keys of a sequence in shared memory

struct PickParams {
  const float* weights;
  const int32_t* tables;
  const int32_t* lens;
  int32_t* lens_out;
  int32_t* kept;
  int64_t num_blocks;
  int bs, width, keep, sinks, recent;
};

// Both sums of the CTA's threads in front of this one, and in all.
__device__ __forceinline__ int2 before_me(int2 v, int2* shared, int2* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int2 incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, incl.x, o), b = __shfl_up_sync(0xffffffffu, incl.y, o);
    if (lane >= o) incl.x += a, incl.y += b;
  }
  __syncthreads();
  if (lane == 31) shared[warp] = incl;
  __syncthreads();
  int2 sum = make_int2(0, 0), front = make_int2(0, 0);
  for (int w = 0; w < kPickThreads / 32; ++w) {
    if (w == warp) front = sum;
    sum.x += shared[w].x;
    sum.y += shared[w].y;
  }
  *all = sum;
  return make_int2(front.x + incl.x - v.x, front.y + incl.y - v.y);
}

template <bool ON_CHIP>
__global__ void __launch_bounds__(kPickThreads) pick_kernel(const PickParams p, int* err) {
  extern __shared__ uint32_t s_keys[];  // ON_CHIP: key i at i + i / 32
  __shared__ int s_count[256];
  __shared__ int2 s_scan[kPickThreads / 32];
  __shared__ int s_bad, s_digit, s_above;
  const int tid = threadIdx.x, s = blockIdx.x;
  const int32_t* table = p.tables + (int64_t)s * p.width;
  const int64_t room = (int64_t)p.width * p.bs;
  const int given = max(p.lens[s], 0);
  const int len = (int)min((int64_t)given, room);
  if (tid == 0) {
    s_bad = 0;
    if (given > len) record_error(err, kDevSeqTooLong);
  }
  __syncthreads();
  int32_t* kept = p.kept + (int64_t)s * p.keep;
  if (len > p.keep) {
    const int pages = (len - 1) / p.bs + 1;
    for (int i = tid; i < pages; i += kPickThreads) {
      const int phys = table[i];
      if (phys < 0 || (int64_t)phys >= p.num_blocks) s_bad = 1;
    }
  }
  __syncthreads();
  if (len <= p.keep || s_bad) {  // stays as it is
    if (tid == 0) {
      p.lens_out[s] = len;
      if (s_bad) record_error(err, kDevBadBlockId);
    }
    for (int i = tid; i < p.keep; i += kPickThreads) kept[i] = !s_bad && i < len ? i : -1;
    return;
  }
  // Tokens [sinks, sinks + n) compete for `want` places; the largest key wins.
  const int n = len - p.sinks - p.recent, want = p.keep - p.sinks - p.recent;
  const auto key_of = [&](int i) {
    const int at = p.sinks + i, page = at / p.bs;
    return orderable_key(p.weights[(int64_t)table[page] * p.bs + (at - page * p.bs)]);
  };
  const auto key_at = [&](int i) { return ON_CHIP ? s_keys[i + i / 32] : key_of(i); };
  if (ON_CHIP)
    for (int i = tid; i < n; i += kPickThreads) s_keys[i + i / 32] = key_of(i);
  uint32_t prefix = 0;  // of the key that the last kept token has
  int left = want;      // places for keys that begin with prefix
  for (int shift = 24; shift >= 0 && want > 0; shift -= 8) {
    __syncthreads();
    if (tid < 256) s_count[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kPickThreads) {
      const uint32_t k = key_at(i);
      if (shift == 24 || (k ^ prefix) >> (shift + 8) == 0) atomicAdd(&s_count[k >> shift & 255u], 1);
    }
    __syncthreads();
    if (tid < 32) {  // from the top: 8 digits a lane
      int mine = 0;
      for (int d = 0; d < 8; ++d) mine += s_count[255 - (tid * 8 + d)];
      int incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, incl, o);
        if (tid >= o) incl += x;
      }
      int above = incl - mine;
      if (above < left && incl >= left) {
        int d = 0;
        while (above + s_count[255 - (tid * 8 + d)] < left) above += s_count[255 - (tid * 8 + d++)];
        s_digit = 255 - (tid * 8 + d);
        s_above = above;
      }
    }
    __syncthreads();
    prefix |= (uint32_t)s_digit << shift;
    left -= s_above;
  }
  __syncthreads();
  // Each thread has a run of tokens: how many of them are above the key, and at it.
  const int run = (n + kPickThreads - 1) / kPickThreads;
  const int i0 = min(tid * run, n), i1 = min(i0 + run, n);
  int2 v = make_int2(0, 0);
  if (want > 0)
    for (int i = i0; i < i1; ++i) {
      const uint32_t k = key_at(i);
      v.x += k > prefix;
      v.y += k == prefix;
    }
  int2 all;
  const int2 front = before_me(v, s_scan, &all);
  if (want > 0) {
    int equal = front.y, to = p.sinks + front.x + min(front.y, left);
    for (int i = i0; i < i1; ++i) {
      const uint32_t k = key_at(i);
      if (k > prefix || (k == prefix && equal < left)) kept[to++] = p.sinks + i;
      equal += k == prefix;
    }
  }
  for (int i = tid; i < p.sinks; i += kPickThreads) kept[i] = i;
  for (int i = tid; i < p.recent; i += kPickThreads) kept[p.keep - p.recent + i] = len - p.recent + i;
  if (tid == 0) p.lens_out[s] = p.keep;
}

// ---------------------------------------------------------------------------
// The move
// ---------------------------------------------------------------------------

constexpr int kMoveThreads = 256;
constexpr int kRound = 128;  // at most so many tokens of a CTA in a round
constexpr int kHeld = 4;     // pieces that a thread holds

struct MoveParams {
  int8_t* cache;
  float* scales;
  float* weights;
  const int32_t* tables;
  const int32_t* lens;
  const int32_t* lens_out;
  const int32_t* kept;
  int64_t num_blocks;
  int seqs, bs, kv_heads, dim, width, keep;
};

// 16, 4 or 1 codes.
template <int N>
struct Piece;
template <>
struct Piece<16> { using T = uint4; };
template <>
struct Piece<4> { using T = uint32_t; };
template <>
struct Piece<1> { using T = uint8_t; };

__device__ __forceinline__ uint32_t shrink4(uint32_t w, float ratio) {
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x = (float)(int8_t)(w >> (8 * i)) * ratio;
    const int c = (int)fminf(fmaxf(rintf(x), -127.0f), 127.0f);
    r |= (uint32_t)(c & 255) << (8 * i);
  }
  return r;
}
__device__ __forceinline__ uint4 shrink(uint4 v, float f) {
  return make_uint4(shrink4(v.x, f), shrink4(v.y, f), shrink4(v.z, f), shrink4(v.w, f));
}
__device__ __forceinline__ uint32_t shrink(uint32_t v, float f) { return shrink4(v, f); }
__device__ __forceinline__ uint8_t shrink(uint8_t v, float f) { return (uint8_t)shrink4(v, f); }

template <int VEC>
__global__ void __launch_bounds__(kMoveThreads) move_kernel(const MoveParams p, int ctas) {
  using V = typename Piece<VEC>::T;
  __shared__ int64_t s_from[kRound], s_to[kRound];  // token slots of the cache
  __shared__ float s_old[kRound], s_new[kRound];
  const int tid = threadIdx.x;
  const int rank = blockIdx.x % ctas;
  const int chain = blockIdx.x / ctas;
  const int per_seq = 2 * p.kv_heads + 1;
  const int s = chain / per_seq, kind = chain % per_seq;
  // (a cluster leaves together)
  const int len = (int)min((int64_t)max(p.lens[s], 0), (int64_t)p.width * p.bs);
  const int kept_n = p.lens_out[s];
  if (kept_n >= len) return;
  const int32_t* table = p.tables + (int64_t)s * p.width;
  const int32_t* kept = p.kept + (int64_t)s * p.keep;
  const auto meet = [&]() {
    if (ctas > 1) cooperative_groups::this_cluster().sync();
    else __syncthreads();
  };
  const auto slot_of = [&](int at) {
    const int page = at / p.bs;
    return (int64_t)table[page] * p.bs + (at - page * p.bs);
  };
  if (kind == 2 * p.kv_heads) {  // the weights
    const int round = kMoveThreads * ctas;
    for (int r0 = 0; r0 < kept_n; r0 += round) {
      const int i = r0 + rank * kMoveThreads + tid;
      float w = 0.0f;
      int64_t to = 0;
      if (i < kept_n) {
        w = p.weights[slot_of(kept[i])];
        to = slot_of(i);
      }
      meet();
      if (i < kept_n) p.weights[to] = w;
    }
    meet();
    for (int i = kept_n + rank * kMoveThreads + tid; i < len; i += round) p.weights[slot_of(i)] = 0.0f;
    return;
  }
  const int v = kind / p.kv_heads, kvh = kind % p.kv_heads;
  int8_t* cache = p.cache + (int64_t)v * p.num_blocks * p.bs * p.kv_heads * p.dim + (int64_t)kvh * p.dim;
  float* scales = p.scales + (int64_t)v * p.num_blocks * p.kv_heads + kvh;
  const int64_t token_bytes = (int64_t)p.kv_heads * p.dim;
  const int pieces = p.dim / VEC;
  // Whole pages a round, as many tokens as the threads hold, in several passes over the
  // channels where that is less than a page.
  const int fit = min(kRound, kMoveThreads * kHeld / pieces);
  const int round = max(fit / p.bs, 1) * p.bs;
  const int per = min(pieces, kMoveThreads * kHeld / round);
  for (int r0 = rank * round; r0 - rank * round < kept_n; r0 += round * ctas) {
    const int n = max(min(round, kept_n - r0), 0);
    for (int i = tid; i < n; i += kMoveThreads) {
      const int at = kept[r0 + i], page = at / p.bs;
      s_from[i] = (int64_t)table[page] * p.bs + (at - page * p.bs);
      s_to[i] = slot_of(r0 + i);
      s_old[i] = scales[(int64_t)table[page] * p.kv_heads];
    }
    __syncthreads();
    for (int i = tid * p.bs; i < n; i += kMoveThreads * p.bs) {
      float most = s_old[i];
      const int end = min(i + p.bs, n);
      for (int j = i + 1; j < end; ++j) {
        const float x = s_old[j];
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(most) : "f"(x));
      }
      for (int j = i; j < end; ++j) s_new[j] = most;
    }
    for (int c0 = 0; c0 < pieces; c0 += per) {
      const int m = min(per, pieces - c0);
      V held[kHeld];
#pragma unroll
      for (int u = 0; u < kHeld; ++u) {
        const int x = u * kMoveThreads + tid, i = x / m;
        if (i < n)
          held[u] = *reinterpret_cast<const V*>(cache + s_from[i] * token_bytes +
                                                (c0 + x - i * m) * VEC);
      }
      meet();
#pragma unroll
      for (int u = 0; u < kHeld; ++u) {
        const int x = u * kMoveThreads + tid, i = x / m;
        if (i < n) {
          const float old = s_old[i], now = s_new[i];
          V c = held[u];
          if (old < now) c = shrink(c, old / now);
          *reinterpret_cast<V*>(cache + s_to[i] * token_bytes + (c0 + x - i * m) * VEC) = c;
        }
      }
    }
    for (int i = tid * p.bs; i < n; i += kMoveThreads * p.bs)
      scales[s_to[i] / p.bs * p.kv_heads] = s_new[i];
    __syncthreads();
  }
}

template <int VEC>
int launch_move(const MoveParams& p, cudaStream_t stream) {
  const int64_t chains = (int64_t)p.seqs * (2 * p.kv_heads + 1);
  // A cluster of more CTAs where there are few chains.
  int ctas = 1;
  while (ctas < 8 && chains * ctas * 2 <= 148 * 4) ctas *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(chains * ctas));
  cfg.blockDim = dim3(kMoveThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ctas > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, move_kernel<VEC>, p, ctas) == cudaSuccess ? kOk : kCudaError;
}

}  // namespace

int launch_evict(const EvictArgs& a, cudaStream_t stream) {
  if (a.seqs == 0) return kOk;
  int* err = device_error_word();
  PickParams k;
  k.weights = a.weights;
  k.tables = a.tables;
  k.lens = a.lens;
  k.lens_out = a.lens_out;
  k.kept = a.kept;
  k.num_blocks = a.num_blocks;
  k.bs = a.block_size;
  k.width = a.width;
  k.keep = a.keep;
  k.sinks = a.sinks;
  k.recent = a.recent;
  const int64_t most = (int64_t)a.width * a.block_size;
  if (most <= kKeysOnChip) {
    const int bytes = (int)(most + most / 32 + 1) * 4;
    static std::atomic<uint64_t> done{0};
    allow_shared_memory(reinterpret_cast<const void*>(pick_kernel<true>),
                        (kKeysOnChip + kKeysOnChip / 32 + 1) * 4, done);
    pick_kernel<true><<<a.seqs, kPickThreads, bytes, stream>>>(k, err);
  } else {
    pick_kernel<false><<<a.seqs, kPickThreads, 0, stream>>>(k, err);
  }
  MoveParams m;
  m.cache = a.cache;
  m.scales = a.scales;
  m.weights = a.weights;
  m.tables = a.tables;
  m.lens = a.lens;
  m.lens_out = a.lens_out;
  m.kept = a.kept;
  m.num_blocks = a.num_blocks;
  m.seqs = a.seqs;
  m.bs = a.block_size;
  m.kv_heads = a.kv_heads;
  m.dim = a.dim;
  m.width = a.width;
  m.keep = a.keep;
  const bool aligned = reinterpret_cast<uintptr_t>(a.cache) % 16 == 0;
  const int rc = a.dim % 16 == 0 && aligned ? launch_move<16>(m, stream)
                 : a.dim % 4 == 0 && aligned ? launch_move<4>(m, stream)
                                             : launch_move<1>(m, stream);
  const cudaError_t e = cudaGetLastError();
  if (rc != kOk || e != cudaSuccess) {
    set_error(std::string("evict launch failed: ") + cudaGetErrorString(e));
    return kCudaError;
  }
  return kOk;
}

}  // namespace pkv
