// Eviction of single tokens from the INT8 paged cache by the weights that they gathered.
//
// A sequence of more than `keep` tokens keeps its first `sinks`, its last `recent` and
// the heaviest of the others (of equal weights the earlier), `keep` in all, in order, at
// the front of its pages.  A page's new scale is the largest of its tokens' old ones, per
// KV head and for K and V apart; codes become rint(code (old / new)) where the old scale
// was smaller (clamped to -127 .. 127 where it was negative), and move as they are else.  The
// weights move along; the slots behind the last token that were in use get weight 0.
//
//   pick_kernel   a CTA or a cluster per sequence: the weights' sort keys, the key that the last
//                 kept token has (radix, 8 bits a pass), the kept tokens in order;
//   move_kernel   a cluster per (sequence, K or V, KV head), and one per sequence for
//                 the weights.
//
// 64 sequences of 1,500 to 2,600 tokens cut to 1,024, 8 heads of 128: pick 10 us, move 73
// us (268 MB, 3.7 TB/s): pieces of 128 bytes, read and written in turns, and 150
// instructions for 16 codes (issue slots 61% busy).  32,768 tokens to 4,096: pick 16 us, a
// cluster's passes one behind the other, move 18 us.
//
// A kept token never moves back: those of the new pages [a, b) come from token a * bs
// or later.  The cluster therefore takes the new pages in rounds, reads all of a round's
// tokens, meets, and writes them: nothing that a later round reads is overwritten.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <string>

#include "cache_mma.cuh"
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

// A cluster of `ctas` CTAs per sequence, each with a part of its tokens in their order: of
// long sequences where there are few (one of 32,768 tokens: 30 us in one CTA).
template <bool ON_CHIP>
__global__ void __launch_bounds__(kPickThreads) pick_kernel(const PickParams p, int ctas, int* err) {
  extern __shared__ uint32_t s_keys[];  // ON_CHIP: key i at i + i / 32
  __shared__ int s_count[2][256], s_sum[256];
  __shared__ int2 s_scan[kPickThreads / 32], s_all;
  __shared__ int s_bad, s_digit, s_above;
  launch_the_next();
  const int tid = threadIdx.x, s = blockIdx.x / ctas, rank = blockIdx.x % ctas;
  auto cluster = cooperative_groups::this_cluster();
  const auto meet = [&]() {
    if (ctas > 1) cluster.sync();
    else __syncthreads();
  };
  const int32_t* table = p.tables + (int64_t)s * p.width;
  const int64_t room = (int64_t)p.width * p.bs;
  const int given = max(p.lens[s], 0);
  const int len = (int)min((int64_t)given, room);
  if (tid == 0) {
    s_bad = 0;
    if (given > len && rank == 0) record_error(err, kDevSeqTooLong);
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
  if (len <= p.keep || s_bad) {  // stays as it is (a cluster's CTAs all see that)
    if (rank > 0) return;
    if (tid == 0) {
      p.lens_out[s] = len;
      if (s_bad) record_error(err, kDevBadBlockId);
    }
    for (int i = tid; i < p.keep; i += kPickThreads) kept[i] = !s_bad && i < len ? i : -1;
    return;
  }
  // Tokens [sinks, sinks + n) compete for `want` places; the largest key wins.  This CTA
  // has `mine` of them from `from` on.
  const int n = len - p.sinks - p.recent, want = p.keep - p.sinks - p.recent;
  const int each = (n + ctas - 1) / ctas;
  const int from = min(rank * each, n), mine = min(each, n - from);
  const auto key_of = [&](int i) {
    const int at = p.sinks + from + i, page = at / p.bs;
    return orderable_key(__ldg(p.weights + (int64_t)__ldg(table + page) * p.bs + (at - page * p.bs)));
  };
  const auto key_at = [&](int i) { return ON_CHIP ? s_keys[i + i / 32] : key_of(i); };
  if (ON_CHIP) {
#pragma unroll 8
    for (int i = tid; i < mine; i += kPickThreads) s_keys[i + i / 32] = key_of(i);
  }
  uint32_t prefix = 0;  // of the key that the last kept token has
  int left = want;      // places for keys that begin with prefix
  for (int shift = 24; shift >= 0 && want > 0; shift -= 8) {
    // (two buffers: the others may still read the last pass's)
    int* count = s_count[shift / 8 & 1];
    __syncthreads();
    if (tid < 256) count[tid] = 0;
    __syncthreads();
    for (int i = tid; i < mine; i += kPickThreads) {
      const uint32_t k = key_at(i);
      if (shift == 24 || (k ^ prefix) >> (shift + 8) == 0) atomicAdd(&count[k >> shift & 255u], 1);
    }
    meet();
    if (ctas > 1) {
      if (tid < 256) {
        int sum = 0;
        for (int c = 0; c < ctas; ++c) sum += cluster.map_shared_rank(count, c)[tid];
        s_sum[tid] = sum;
      }
      __syncthreads();
      count = s_sum;
    }
    if (tid < 32) {  // from the top: 8 digits a lane
      int here = 0;
      for (int d = 0; d < 8; ++d) here += count[255 - (tid * 8 + d)];
      int incl = here;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, incl, o);
        if (tid >= o) incl += x;
      }
      int above = incl - here;
      if (above < left && incl >= left) {
        int d = 0;
        while (above + count[255 - (tid * 8 + d)] < left) above += count[255 - (tid * 8 + d++)];
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
  const int run = (mine + kPickThreads - 1) / kPickThreads;
  const int i0 = min(tid * run, mine), i1 = min(i0 + run, mine);
  int2 v = make_int2(0, 0);
  if (want > 0)
    for (int i = i0; i < i1; ++i) {
      const uint32_t k = key_at(i);
      v.x += k > prefix;
      v.y += k == prefix;
    }
  int2 all;
  int2 front = before_me(v, s_scan, &all);
  if (ctas > 1) {  // and of the parts in front
    if (tid == 0) s_all = all;
    cluster.sync();
    for (int c = 0; c < rank; ++c) {
      const int2 x = *cluster.map_shared_rank(&s_all, c);
      front.x += x.x;
      front.y += x.y;
    }
    cluster.sync();  // nobody leaves while the others read
  }
  if (want > 0) {
    int equal = front.y, to = p.sinks + front.x + min(front.y, left);
    for (int i = i0; i < i1; ++i) {
      const uint32_t k = key_at(i);
      if (k > prefix || (k == prefix && equal < left)) kept[to++] = p.sinks + from + i;
      equal += k == prefix;
    }
  }
  const int step = ctas * kPickThreads;
  for (int i = rank * kPickThreads + tid; i < p.sinks; i += step) kept[i] = i;
  for (int i = rank * kPickThreads + tid; i < p.recent; i += step)
    kept[p.keep - p.recent + i] = len - p.recent + i;
  if (tid == 0 && rank == 0) p.lens_out[s] = p.keep;
}

// ---------------------------------------------------------------------------
// The move
// ---------------------------------------------------------------------------

constexpr int kMoveThreads = 256;
constexpr int kIndex = 1024;  // tokens of a CTA whose places are looked up at once
constexpr int kHeld = 4;      // pieces that a thread holds

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

// rint(code ratio) of four codes.  A byte in the low mantissa of 2^23 is a number, and a
// number at 1.5 2^23 is rounded to an integer, to even as rint, whose low byte is there: the
// conversion instructions, 16 a clock and SM, would take 90 us of the 64 sequences' move.
// (Only where the old scale is negative can a code leave its range: the ratio is not 0 to 1 then.)
__device__ __forceinline__ uint32_t shrink4(uint32_t w, float ratio) {
  const uint32_t u = w ^ 0x80808080u;
  uint32_t x[4];
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const uint64_t code = add_f32x2(f32x2(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 + i)),
                                          __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441 + i))),
                                    f32x2(-8388736.0f, -8388736.0f));
    const float2 c = unpack_f32x2(code);  // (products rounded apart from the sums behind them)
    x[i] = __float_as_uint(__fadd_rn(__fmul_rn(c.x, ratio), 12582912.0f));
    x[i + 1] = __float_as_uint(__fadd_rn(__fmul_rn(c.y, ratio), 12582912.0f));
  }
  if (!(ratio >= 0.0f && ratio <= 1.0f))
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[i] = __float_as_uint(fminf(fmaxf(__uint_as_float(x[i]), 12582912.0f - 127.0f), 12582912.0f + 127.0f));
  return __byte_perm(__byte_perm(x[0], x[1], 0x0040), __byte_perm(x[2], x[3], 0x0040), 0x5410);
}
__device__ __forceinline__ uint4 shrink(uint4 v, float f) {
  return make_uint4(shrink4(v.x, f), shrink4(v.y, f), shrink4(v.z, f), shrink4(v.w, f));
}
__device__ __forceinline__ uint32_t shrink(uint32_t v, float f) { return shrink4(v, f); }
__device__ __forceinline__ uint8_t shrink(uint8_t v, float f) { return (uint8_t)shrink4(v, f); }

template <int VEC>
__global__ void __launch_bounds__(kMoveThreads) move_kernel(const MoveParams p, int ctas) {
  using V = typename Piece<VEC>::T;
  __shared__ int s_from[kIndex], s_to[kIndex];  // token slots of the cache
  __shared__ float s_old[kIndex], s_new[kIndex];
  behind_the_last();
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
    return table[page] * p.bs + (at - page * p.bs);
  };
  if (kind == 2 * p.kv_heads) {  // the weights
    const int round = kMoveThreads * ctas;
    for (int r0 = 0; r0 < kept_n; r0 += round) {
      const int i = r0 + rank * kMoveThreads + tid;
      float w = 0.0f;
      int to = 0;
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
  // channels where that is less than a page.  The rounds' places and scales are looked up
  // many at a time: a round that began with its own took 14 us (kept, table, scale and codes
  // one behind the other).
  const int fit = min(kIndex, kMoveThreads * kHeld / pieces);
  const int round = max(fit / p.bs, 1) * p.bs;
  const int per = min(pieces, kMoveThreads * kHeld / round);
  const int rounds = (kept_n + round * ctas - 1) / (round * ctas), at_once = kIndex / round;
  for (int g0 = 0; g0 < rounds; g0 += at_once) {
    const int some = min(at_once, rounds - g0);
    // the place among the kept ones of the CTA's i-th token of these rounds
    const auto token_of = [&](int i) {
      const int g = i / round;
      return ((g0 + g) * ctas + rank) * round + i - g * round;
    };
#pragma unroll 4
    for (int i = tid; i < some * round; i += kMoveThreads) {
      const int t = token_of(i);
      if (t < kept_n) {
        const int at = kept[t], page = at / p.bs, phys = table[page];
        s_from[i] = phys * p.bs + (at - page * p.bs);
        s_to[i] = slot_of(t);
        s_old[i] = scales[(int64_t)phys * p.kv_heads];
      }
    }
    __syncthreads();
    for (int i = tid * p.bs; i < some * round; i += kMoveThreads * p.bs) {
      const int n = min(p.bs, kept_n - token_of(i));
      if (n <= 0) continue;
      float most = s_old[i];
      for (int j = 1; j < n; ++j) {
        const float x = s_old[i + j];
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(most) : "f"(x));
      }
      s_new[i / p.bs] = most;
      // what the codes are multiplied by; 1: they move as they are
      for (int j = 0; j < n; ++j) s_old[i + j] = s_old[i + j] < most ? s_old[i + j] / most : 1.0f;
    }
    __syncthreads();
    for (int g = 0; g < some; ++g) {
      const int base = g * round;
      const int n = max(min(round, kept_n - token_of(base)), 0);
      for (int c0 = 0; c0 < pieces; c0 += per) {
        const int m = min(per, pieces - c0);
        const uint32_t over_m = ((1u << 20) + m - 1) / m;  // exact for x m below 2^20
        V held[kHeld];
        int token[kHeld], at[kHeld];
#pragma unroll
        for (int u = 0; u < kHeld; ++u) {
          const int x = u * kMoveThreads + tid;
          token[u] = (int)(x * over_m >> 20);
          at[u] = (c0 + x - token[u] * m) * VEC;
          if (token[u] < n)
            held[u] = *reinterpret_cast<const V*>(cache + s_from[base + token[u]] * token_bytes + at[u]);
        }
        meet();
#pragma unroll
        for (int u = 0; u < kHeld; ++u) {
          if (token[u] >= n) continue;
          const float ratio = s_old[base + token[u]];
          V c = held[u];
          if (ratio != 1.0f) c = shrink(c, ratio);
          *reinterpret_cast<V*>(cache + s_to[base + token[u]] * token_bytes + at[u]) = c;
        }
      }
    }
    // (every CTA of the cluster has met since it read its scales of these rounds)
    for (int i = tid * p.bs; i < some * round; i += kMoveThreads * p.bs)
      if (token_of(i) < kept_n) scales[(int64_t)(s_to[i] / p.bs) * p.kv_heads] = s_new[i / p.bs];
    __syncthreads();
  }
}

// (errors: cudaGetLastError, as after <<<>>>)
template <typename... Params, typename... Args>
void launch_clusters(void (*kernel)(Params...), int64_t grid, int threads, int ctas, size_t shared,
                     bool behind, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)grid);
  config.blockDim = dim3((unsigned)threads);
  config.dynamicSmemBytes = shared;
  config.stream = stream;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attr;
  config.numAttrs = behind ? 2 : 1;
  cudaLaunchKernelEx(&config, kernel, Params(args)...);
}

template <int VEC>
void launch_move(const MoveParams& p, cudaStream_t stream) {
  const int64_t chains = (int64_t)p.seqs * (2 * p.kv_heads + 1);
  // A cluster of more CTAs where there are few chains.
  int ctas = 1;
  while (ctas < 8 && chains * ctas * 2 <= 148 * 4) ctas *= 2;
  launch_clusters(move_kernel<VEC>, chains * ctas, kMoveThreads, ctas, 0, true, stream, p, ctas);
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
  // more CTAs a sequence where that leaves each of them some keys a thread
  int ctas = 1;
  while (ctas < 8 && a.seqs * ctas * 2 <= 148 && most > 4 * kPickThreads * ctas) ctas *= 2;
  const int64_t part = (most + ctas - 1) / ctas;
  const bool on_chip = part <= kKeysOnChip;
  const auto kern = on_chip ? pick_kernel<true> : pick_kernel<false>;
  static std::atomic<uint64_t> done{0};
  allow_shared_memory(reinterpret_cast<const void*>(pick_kernel<true>),
                      (kKeysOnChip + kKeysOnChip / 32 + 1) * 4, done);
  launch_clusters(kern, (int64_t)a.seqs * ctas, kPickThreads, ctas, on_chip ? (size_t)(part + part / 32 + 1) * 4 : 0,
                  false, stream, k, ctas, err);
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
  if (a.dim % 16 == 0 && aligned) launch_move<16>(m, stream);
  else if (a.dim % 4 == 0 && aligned) launch_move<4>(m, stream);
  else launch_move<1>(m, stream);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_error(std::string("evict launch failed: ") + cudaGetErrorString(e));
    return kCudaError;
  }
  return kOk;
}

}  // namespace pkv
