// Rotary positions: per-head RMS norm + rotation of queries and keys in one
// pass (qk_norm_rope), and the append of keys and values to the INT8 paged
// cache with the rotation applied on the way (append_kv).
//
// The rotation of one pair (a, b) at position p with table entry (c, s):
//   a' = a c - b s,   b' = b c + a s
// in 32 bits with each product and sum rounded on its own, so that the INT8
// codes of append_kv have one defined value.  Pairs are (i, i + R/2) (half
// layout) or (2i, 2i + 1) (interleaved); channels from R on pass unchanged.
// The table is float32 [P, R]: R/2 cosines, then R/2 sines per position.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "pkv_common.cuh"
#include "pkv_internal.h"
#include "quantize_math.cuh"

namespace pkv {
namespace {

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

__device__ __forceinline__ float rot_first(float a, float b, float c, float s) {
  return __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
}
__device__ __forceinline__ float rot_second(float a, float b, float c, float s) {
  return __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
}

// N consecutive values of T as 32-bit words (N * sizeof(T) = 4, 8 or 16
// bytes, or a single value), loaded and stored in one access.
template <typename T, int N>
struct alignas(N * sizeof(T)) Chunk {
  T e[N];
};

template <typename T, int N>
__device__ __forceinline__ Chunk<T, N> load_chunk(const T* p) {
  Chunk<T, N> c;
  if constexpr (N * sizeof(T) == 16) {
    *reinterpret_cast<uint4*>(c.e) = *reinterpret_cast<const uint4*>(p);
  } else if constexpr (N * sizeof(T) == 8) {
    *reinterpret_cast<uint2*>(c.e) = *reinterpret_cast<const uint2*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) c.e[i] = p[i];
  }
  return c;
}

// ---------------------------------------------------------------------------
// qk_norm_rope
// ---------------------------------------------------------------------------

template <typename T>
struct QkArgs {
  const T* q;
  const T* k;
  T* q_out;
  T* k_out;
  int64_t q_tok, q_head, k_tok, k_head;  // input strides in elements
  const int64_t* positions;
  const float* table;
  const void* q_weight;  // both null: no norm
  const void* k_weight;
  bool weight_f32;  // weights in float32, else in T
  int64_t tokens;
  int heads, kv_heads, dim, rot;
  int64_t table_rows;
  float eps;
};

// A group of LPR lanes (a power of two) owns RPG rows (token, head) of one
// token; lane l holds chunks l and (NC = 2) l + LPR of VEC channels, one
// 16-byte access each.  The partners of the half layout are R/2 channels
// away, in another lane: their raw words come by shuffle, so a row is read
// once.  The table entries of a lane are the same for all its rows.
// What bounds it: without norms HBM (a row is read and written once); RPG = 4
// keeps four independent loads in flight and reads the table a quarter as often.
// 16,384 tokens of 40 + 40 heads in fp16, head_dim 128: 115 us for 675 MB (5.9 TB/s,
// 0.90 of the copy rate).  With norms and weights the instructions for a value: 32 +
// 8 heads in bf16 116 us for 344 MB (floor 53 us; issue slots 73% busy, DRAM 31%).
// A decode step of 64 tokens, 32 + 8 heads with norms: 3.0 us.
template <typename T, int VEC, int LPR, int NC, int RPG, bool NORM, bool INTER>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(QkArgs<T> a, int* err) {
  const int rows = a.heads + a.kv_heads;
  const int per_token = (rows + RPG - 1) / RPG;
  const int lane = threadIdx.x & 31, gl = lane & (LPR - 1), g0 = lane - gl;
  const int64_t group = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const int64_t token = group / per_token;
  const int sub = (int)(group - token * per_token);
  const bool live = token < a.tokens;  // every lane stays for the shuffles
  const int chunks = a.dim / VEC, half = a.rot / 2;
  int64_t pos = live ? a.positions[token] : 0;
  const bool bad = pos < 0 || pos >= a.table_rows;
  if (bad) {
    if (gl == 0) record_error(err, kDevBadPosition);
    pos = 0;
  }
  const float* row = a.table + pos * a.rot;

  alignas(16) float cs[NC][VEC], sn[NC][VEC];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int d = (gl + i * LPR) * VEC;
    if (live && d < a.rot) {
      if constexpr (INTER) {
        const int p = d / 2;
#pragma unroll
        for (int e = 0; e < VEC / 2; ++e) {
          cs[i][e] = p + e < half ? row[p + e] : 1.0f;
          sn[i][e] = p + e < half ? row[half + p + e] : 0.0f;
        }
      } else {
        const int p = d < half ? d : d - half;
#pragma unroll
        for (int e = 0; e < VEC; e += 4) {
          *reinterpret_cast<float4*>(&cs[i][e]) = *reinterpret_cast<const float4*>(row + p + e);
          *reinterpret_cast<float4*>(&sn[i][e]) =
              *reinterpret_cast<const float4*>(row + half + p + e);
        }
      }
    }
  }

  Chunk<T, VEC> x[RPG][NC];
#pragma unroll
  for (int r = 0; r < RPG; ++r) {
    const int h = sub + r * per_token;
    if (live && h < rows) {
      const T* src = h < a.heads ? a.q + token * a.q_tok + (int64_t)h * a.q_head
                                 : a.k + token * a.k_tok + (int64_t)(h - a.heads) * a.k_head;
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if (gl + i * LPR < chunks) x[r][i] = load_chunk<T, VEC>(src + (gl + i * LPR) * VEC);
    }
  }

#pragma unroll
  for (int r = 0; r < RPG; ++r) {
    const int h = sub + r * per_token;
    const bool on = live && h < rows;
    if (RPG > 1 && !__any_sync(0xffffffffu, on)) break;
    const bool is_q = h < a.heads;
    float rstd = 1.0f;
    const void* w = is_q ? a.q_weight : a.k_weight;
    if constexpr (NORM) {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if (on && gl + i * LPR < chunks)
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float v = to_f32<T>(x[r][i].e[e]);
            ss = fmaf(v, v, ss);
          }
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      rstd = rsqrtf(ss / (float)a.dim + a.eps);
    }
    auto weight = [&](int d) {
      if constexpr (!NORM) {
        return 1.0f;
      } else {
        return a.weight_f32 ? static_cast<const float*>(w)[d]
                            : to_f32<T>(static_cast<const T*>(w)[d]);
      }
    };
    T* dst = is_q ? a.q_out + (token * a.heads + h) * (int64_t)a.dim
                  : a.k_out + (token * a.kv_heads + (h - a.heads)) * (int64_t)a.dim;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = gl + i * LPR, d = c * VEC;
      Chunk<T, VEC> other;
      if constexpr (!INTER) {
        // the partner chunk of a rotated chunk, from whichever lane and slot
        // holds it (every lane of the warp takes part in the shuffles)
        const int pc = d < half ? c + half / VEC : c - half / VEC;
        constexpr int W = VEC * sizeof(T) / 4;
        uint32_t* o32 = reinterpret_cast<uint32_t*>(other.e);
#pragma unroll
        for (int j = 0; j < NC; ++j) {
          const uint32_t* v32 = reinterpret_cast<const uint32_t*>(x[r][j].e);
#pragma unroll
          for (int u = 0; u < W; ++u) {
            const uint32_t v = __shfl_sync(0xffffffffu, v32[u], g0 + (pc & (LPR - 1)));
            if (NC == 1 || pc / LPR == j) o32[u] = v;
          }
        }
      }
      if (!on || c >= chunks) continue;
      float y[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        y[e] = to_f32<T>(x[r][i].e[e]);
        if constexpr (NORM) y[e] = y[e] * rstd * weight(d + e);
      }
      if (d < a.rot) {
        if constexpr (INTER) {
#pragma unroll
          for (int e = 0; e < VEC; e += 2) {
            const float p = y[e], q = y[e + 1];
            if (d + e < a.rot) {
              y[e] = rot_first(p, q, cs[i][e / 2], sn[i][e / 2]);
              y[e + 1] = rot_second(p, q, cs[i][e / 2], sn[i][e / 2]);
            }
          }
        } else {
          const int pd = d < half ? d + half : d - half;
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            float p = to_f32<T>(other.e[e]);
            if constexpr (NORM) p = p * rstd * weight(pd + e);
            y[e] = d < half ? rot_first(y[e], p, cs[i][e], sn[i][e])
                            : rot_second(p, y[e], cs[i][e], sn[i][e]);
          }
        }
      }
      Chunk<T, VEC> out;
#pragma unroll
      for (int e = 0; e < VEC; ++e) out.e[e] = from_f32<T>(bad ? 0.0f : y[e]);
      if constexpr (VEC * sizeof(T) == 16)
        *reinterpret_cast<uint4*>(dst + d) = *reinterpret_cast<const uint4*>(out.e);
    }
  }
}

// Any head_dim, rotary width, alignment and stride: one warp per row, one
// value per access, the partner value read from memory again.  Bound by its
// accesses: 16,384 tokens of 40 + 40 heads in fp16, 24 of 96 channels rotated, take
// 362 us for 503 MB (floor 77 us), 20 of 80 with norms 482 us for 419 MB (64 us).
template <typename T, bool NORM>
__global__ void __launch_bounds__(256)
    qk_norm_rope_scalar_kernel(QkArgs<T> a, bool interleaved, int* err) {
  const int rows = a.heads + a.kv_heads;
  const int lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int64_t token = unit / rows;
  if (token >= a.tokens) return;  // whole warps
  const int h = (int)(unit - token * rows);
  const bool is_q = h < a.heads;
  const int half = a.rot / 2;
  const int64_t pos = a.positions[token];
  const bool bad = pos < 0 || pos >= a.table_rows;
  if (bad && lane == 0) record_error(err, kDevBadPosition);
  const float* row = a.table + (bad ? 0 : pos) * a.rot;
  const T* src = is_q ? a.q + token * a.q_tok + (int64_t)h * a.q_head
                      : a.k + token * a.k_tok + (int64_t)(h - a.heads) * a.k_head;
  T* dst = is_q ? a.q_out + (token * a.heads + h) * (int64_t)a.dim
                : a.k_out + (token * a.kv_heads + (h - a.heads)) * (int64_t)a.dim;
  const void* w = is_q ? a.q_weight : a.k_weight;
  float rstd = 1.0f;
  if constexpr (NORM) {
    float ss = 0.0f;
    for (int d = lane; d < a.dim; d += 32) {
      const float v = to_f32<T>(src[d]);
      ss = fmaf(v, v, ss);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    rstd = rsqrtf(ss / (float)a.dim + a.eps);
  }
  auto value = [&](int d) {
    const float v = to_f32<T>(src[d]);
    if constexpr (!NORM) {
      return v;
    } else {
      return v * rstd * (a.weight_f32 ? static_cast<const float*>(w)[d]
                                      : to_f32<T>(static_cast<const T*>(w)[d]));
    }
  };
  for (int d = lane; d < a.dim; d += 32) {
    float y = value(d);
    if (d < a.rot) {
      const bool first = interleaved ? (d & 1) == 0 : d < half;
      const int i = interleaved ? d / 2 : (first ? d : d - half);
      const float p = value(interleaved ? d ^ 1 : (first ? d + half : d - half));
      y = first ? rot_first(y, p, row[i], row[half + i]) : rot_second(p, y, row[i], row[half + i]);
    }
    dst[d] = from_f32<T>(bad ? 0.0f : y);
  }
}

template <typename T, int VEC, int LPR, int NC, bool NORM, bool INTER>
void launch_qk_rows(const QkArgs<T>& a, cudaStream_t stream) {
  const int rows = a.heads + a.kv_heads;
  constexpr int kGroups = 256 / LPR;
  // Few rows: one row per group, so that the call spreads over the SMs.
  if (a.tokens * rows <= 148LL * 4 * kGroups) {
    const int64_t groups = a.tokens * rows;
    qk_norm_rope_kernel<T, VEC, LPR, NC, 1, NORM, INTER>
        <<<(unsigned)((groups + kGroups - 1) / kGroups), 256, 0, stream>>>(a, device_error_word());
  } else {
    const int64_t groups = a.tokens * ((rows + 3) / 4);
    qk_norm_rope_kernel<T, VEC, LPR, NC, 4, NORM, INTER>
        <<<(unsigned)((groups + kGroups - 1) / kGroups), 256, 0, stream>>>(a, device_error_word());
  }
}

template <typename T, bool NORM, bool INTER>
bool launch_qk_vec(const QkArgs<T>& a, cudaStream_t stream) {
  constexpr int VEC = 16 / sizeof(T);
  const int chunks = a.dim / VEC;
  if (chunks <= 4) launch_qk_rows<T, VEC, 4, 1, NORM, INTER>(a, stream);
  else if (chunks <= 8) launch_qk_rows<T, VEC, 8, 1, NORM, INTER>(a, stream);
  else if (chunks <= 16) launch_qk_rows<T, VEC, 16, 1, NORM, INTER>(a, stream);
  else if (chunks <= 32) launch_qk_rows<T, VEC, 32, 1, NORM, INTER>(a, stream);
  else if (chunks <= 64) launch_qk_rows<T, VEC, 32, 2, NORM, INTER>(a, stream);
  else return false;
  return true;
}

template <typename T>
int launch_qk_t(const QkNormRopeArgs& p, cudaStream_t stream) {
  QkArgs<T> a;
  a.q = static_cast<const T*>(p.q);
  a.k = static_cast<const T*>(p.k);
  a.q_out = static_cast<T*>(p.q_out);
  a.k_out = static_cast<T*>(p.k_out);
  a.q_tok = p.q_token_stride;
  a.q_head = p.q_head_stride;
  a.k_tok = p.k_token_stride;
  a.k_head = p.k_head_stride;
  a.positions = p.positions;
  a.table = p.table;
  a.q_weight = p.q_weight;
  a.k_weight = p.k_weight;
  a.weight_f32 = p.weight_f32;
  a.tokens = p.tokens;
  a.heads = p.heads;
  a.kv_heads = p.kv_heads;
  a.dim = p.dim;
  a.rot = p.rot;
  a.table_rows = p.table_rows;
  a.eps = p.eps;
  const bool norm = p.q_weight != nullptr;
  constexpr int VEC = 16 / sizeof(T);
  auto aligned = [](const void* x) { return reinterpret_cast<uintptr_t>(x) % 16 == 0; };
  const bool strides = a.q_tok % VEC == 0 && a.q_head % VEC == 0 && a.k_tok % VEC == 0 &&
                       a.k_head % VEC == 0;
  const bool rot_ok = p.interleaved ? a.rot % 2 == 0 : (a.rot % 8 == 0 && (a.rot / 2) % VEC == 0);
  const bool vec = a.dim % VEC == 0 && strides && rot_ok && aligned(a.q) && aligned(a.k) &&
                   aligned(a.q_out) && aligned(a.k_out) && aligned(a.table);
  if (vec) {
    const bool done = norm ? (p.interleaved ? launch_qk_vec<T, true, true>(a, stream)
                                            : launch_qk_vec<T, true, false>(a, stream))
                           : (p.interleaved ? launch_qk_vec<T, false, true>(a, stream)
                                            : launch_qk_vec<T, false, false>(a, stream));
    if (done) return kOk;
  }
  const int64_t units = a.tokens * (a.heads + a.kv_heads);
  const unsigned grid = (unsigned)((units + 7) / 8);
  if (norm)
    qk_norm_rope_scalar_kernel<T, true><<<grid, 256, 0, stream>>>(a, p.interleaved,
                                                                  device_error_word());
  else
    qk_norm_rope_scalar_kernel<T, false><<<grid, 256, 0, stream>>>(a, p.interleaved,
                                                                   device_error_word());
  return kOk;
}

// ---------------------------------------------------------------------------
// append_kv
// ---------------------------------------------------------------------------
//
// A work unit is a page touched by the call (its K or V half in small calls):
// the call's tokens in that page set its scale together.  Up to kAppendScan
// tokens every CTA finds its page's tokens by scanning the slots itself (one
// launch); above that, an index kernel first chains the runs of consecutive
// tokens per page.

constexpr int kAppendThreads = 256;
constexpr int kAppendWarps = kAppendThreads / 32;
constexpr int kAppendMaxPage = 64;  // largest block_size
constexpr int kAppendHold = 16;     // tokens of a head kept on chip

template <typename T>
struct AppendArgs {
  const T* key;
  const T* value;
  int64_t k_tok, k_head, v_tok, v_head;
  int8_t* cache;
  float* scales;
  const int64_t* slots;
  const int64_t* positions;  // null: no rotation
  const float* table;
  int64_t tokens, blocks, table_rows;
  int bs, kv_heads, dim, rot;
  bool interleaved;
};

// Slot of token t, or -1 where the token is not to be written: the padding
// slot -1, a slot outside the cache, a position outside the table.
template <typename T>
__device__ __forceinline__ int64_t append_slot(const AppendArgs<T>& a, int64_t t, int* err) {
  const int64_t slot = a.slots[t];
  if (slot == -1) return -1;
  if (slot < 0 || slot >= a.blocks * a.bs) {
    record_error(err, kDevBadSlot);
    return -1;
  }
  if (a.positions != nullptr) {
    const int64_t p = a.positions[t];
    if (p < 0 || p >= a.table_rows) {
      record_error(err, kDevBadPosition);
      return -1;
    }
  }
  return slot;
}

enum Rotation { kNoRotation = 0, kHalves = 1, kPairs = 2 };

// Rotates chunk c (VEC channels, raw words x) of one head in place of y.  The
// partner chunk of the half layout is another lane's when a head fits one
// chunk per lane (NC = 1), else it is read from `src` again.  Every lane of
// the warp calls.
template <typename T, int VEC, int NC, int ROT>
__device__ __forceinline__ void append_rotate(const AppendArgs<T>& a, const float* row,
                                              const T* src, const Chunk<T, VEC>& x, int c, bool on,
                                              float (&y)[VEC]) {
  const int half = a.rot / 2, d = c * VEC;
  if constexpr (ROT == kPairs && VEC > 1) {
#pragma unroll
    for (int e = 0; e + 1 < VEC; e += 2) {
      if (on && d + e < a.rot) {
        const float cc = row[(d + e) / 2], ss = row[half + (d + e) / 2];
        const float p = y[e], q = y[e + 1];
        y[e] = rot_first(p, q, cc, ss);
        y[e + 1] = rot_second(p, q, cc, ss);
      }
    }
  } else {
    const bool first = ROT == kPairs ? (d & 1) == 0 : d < half;
    Chunk<T, VEC> o;
    if constexpr (VEC > 1 && NC == 1) {
      constexpr int W = VEC * sizeof(T) / 4;
      const int pc = first ? c + half / VEC : c - half / VEC;
      const uint32_t* v32 = reinterpret_cast<const uint32_t*>(x.e);
      uint32_t* o32 = reinterpret_cast<uint32_t*>(o.e);
#pragma unroll
      for (int u = 0; u < W; ++u) o32[u] = __shfl_sync(0xffffffffu, v32[u], pc & 31);
    } else if (on && d < a.rot) {
      o = load_chunk<T, VEC>(src + (ROT == kPairs ? d ^ 1 : (first ? d + half : d - half)));
    }
    if (on && d < a.rot) {
      const int i = ROT == kPairs ? d / 2 : (first ? d : d - half);
      alignas(16) float cc[VEC], ss[VEC];
      if constexpr (VEC == 4) {
        *reinterpret_cast<float4*>(cc) = *reinterpret_cast<const float4*>(row + i);
        *reinterpret_cast<float4*>(ss) = *reinterpret_cast<const float4*>(row + half + i);
      } else {
        cc[0] = row[i];
        ss[0] = row[half + i];
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float p = to_f32<T>(o.e[e]);
        y[e] = first ? rot_first(y[e], p, cc[e], ss[e]) : rot_second(p, y[e], cc[e], ss[e]);
      }
    }
  }
}

// The call's tokens in one page, in ascending offsets.
struct AppendList {
  int off[kAppendMaxPage];
  int tok[kAppendMaxPage];
  int64_t pos[kAppendMaxPage];
  int count, lowest;
};

// Compacts s_tok (a page's token per offset, or -1) into the list; whole CTA.
template <typename T>
__device__ void append_list(const AppendArgs<T>& a, const int* s_tok, AppendList& list) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int n = 0, lowest = a.bs;
    for (int b = 0; b < a.bs; b += 32) {
      const int off = b + lane;
      const int t = off < a.bs ? s_tok[off] : -1;
      const unsigned m = __ballot_sync(0xffffffffu, t >= 0);
      if (t >= 0) {
        const int at = n + __popc(m & ((1u << lane) - 1u));
        list.off[at] = off;
        list.tok[at] = t;
        list.pos[at] = a.positions != nullptr ? a.positions[t] : 0;
      }
      if (m != 0 && lowest == a.bs) lowest = b + __ffs(m) - 1;
      n += __popc(m);
    }
    if (lane == 0) {
      list.count = n;
      list.lowest = lowest;
    }
  }
  __syncthreads();
}

// The page's scale from the new values' absmax; the earlier codes, `row_bytes`
// of them per offset below `lowest`, moved to it where it grew.
__device__ __forceinline__ float append_scale(float amax, float* scale, float old, int lowest,
                                              int8_t* head_base, int64_t tok_stride, int dim,
                                              bool words) {
  const int lane = threadIdx.x & 31;
  const float step = amax > 0.0f ? __fdiv_rn(amax, 127.0f) : 0.0f;
  const bool grow = step > old;
  const float sc = lowest == 0 ? (step > 0.0f ? step : 1.0f) : (grow ? step : old);
  __syncwarp();  // every lane has the old scale
  if (lane == 0) *scale = sc;
  if (lowest > 0 && grow) {
    const float ratio = __fdiv_rn(old, sc);
    auto move = [&](int8_t code) {
      return (uint32_t)(__float2int_rn(__fmul_rn((float)code, ratio)) & 255);
    };
    if (words) {
      // lane = (offset, word): short rows keep the warp busy
      const int per_row = dim / 4;
#pragma unroll 4
      for (int i = lane; i < lowest * per_row; i += 32) {
        uint32_t* p = reinterpret_cast<uint32_t*>(head_base + (i / per_row) * tok_stride) + i % per_row;
        const uint32_t w = *p;
        *p = move((int8_t)w) | move((int8_t)(w >> 8)) << 8 | move((int8_t)(w >> 16)) << 16 |
             move((int8_t)(w >> 24)) << 24;
      }
    } else {
      for (int off = 0; off < lowest; ++off)
        for (int d = lane; d < dim; d += 32) {
          int8_t* p = head_base + off * tok_stride + d;
          *p = (int8_t)move(*p);
        }
    }
  }
  return sc;
}

// One head of one page, K or V, by one warp, any shape: absmax of the new
// values, the page's scale, the earlier codes moved, the new codes.  Inputs
// are read twice.
template <typename T, int VEC, int NC, int ROT>
__device__ __noinline__ void append_head(const AppendArgs<T>& a, int64_t page, bool is_key,
                                            int h, const AppendList& list) {
  const int lane = threadIdx.x & 31;
  const int n = list.count, lowest = list.lowest, chunks = a.dim / VEC;
  const int64_t tok_stride = (int64_t)a.kv_heads * a.dim;
  int8_t* head_base = a.cache + (is_key ? 0 : a.blocks * a.bs * tok_stride) +
                      page * a.bs * tok_stride + (int64_t)h * a.dim;
  float* scale = a.scales + (is_key ? 0 : a.blocks * a.kv_heads) + page * a.kv_heads + h;
  const T* base = is_key ? a.key + (int64_t)h * a.k_head : a.value + (int64_t)h * a.v_head;
  const int64_t step_tok = is_key ? a.k_tok : a.v_tok;
  const float old = lowest > 0 ? *scale : 0.0f;

  uint32_t m = 0u;
  auto fold = [&](const float (&y)[VEC]) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) m = max(m, __float_as_uint(y[e]) & 0x7fffffffu);
  };
  auto load = [&](int i, int c, float (&y)[VEC]) {
    const T* src = base + list.tok[i] * step_tok;
    Chunk<T, VEC> x;
    if (c < chunks) x = load_chunk<T, VEC>(src + c * VEC);
#pragma unroll
    for (int e = 0; e < VEC; ++e) y[e] = c < chunks ? to_f32<T>(x.e[e]) : 0.0f;
    if constexpr (ROT != kNoRotation)
      append_rotate<T, VEC, NC, ROT>(a, a.table + list.pos[i] * a.rot, src, x, c, c < chunks, y);
  };
  for (int i = 0; i < n; ++i)
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      float y[VEC];
      load(i, lane + 32 * j, y);
      fold(y);
    }
  m = __reduce_max_sync(0xffffffffu, m);  // NaN bits exceed +inf: NaN wins
  const float amax = __uint_as_float(m);
  const float sc = append_scale(amax, scale, old, lowest, head_base, tok_stride, a.dim, VEC == 4);
  const float rcp = __frcp_rn(sc);
  const bool fast = isfinite(amax) && !isinf(rcp);
  for (int i = 0; i < n; ++i)
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int c = lane + 32 * j;
      float y[VEC];
      load(i, c, y);
      if (c >= chunks) continue;
      int8_t* dst = head_base + list.off[i] * tok_stride + c * VEC;
      if constexpr (VEC == 4)
        *reinterpret_cast<uint32_t*>(dst) = quantize_word(y, sc, rcp, fast);
      else
        *dst = (int8_t)quantize_one(y[0], sc);
    }
}

// The same for pages whose rows fit on chip, in 8-channel pieces: half a warp per
// token (a warp's instruction serves two), or a warp above 128 channels.  All
// rows of a head are copied to shared memory at once, so inputs are read once
// and a warp has 4 KB in flight; the rotation is cheap enough to be done
// again for the codes.  32,768 bf16 tokens of 8 heads in pages of 16: 79 us
// (201 MB, 31 us at the copy rate), issue slots 61% busy -- bound by the
// instructions for a value and the latencies of a page's steps (its tokens' list,
// its rows, the maximum, the codes), which 24 warps an SM do not hide.  Slower were:
// rows held in registers (one pair of tokens ahead left each step waiting for
// HBM, all sixteen tokens spilled; 158 to 420 us); half a warp per token with all
// heads, maxima exchanged by the CTA (135 us); the next page's list and rows read
// ahead (95 us).
__device__ __forceinline__ void copy16_async(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src)
               : "memory");
}
__device__ __forceinline__ void copies_group() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>  // all but the last N groups
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Starts the copies of one head's rows.
template <typename T, int ROW>
__device__ __forceinline__ void append_fetch8(const AppendArgs<T>& a, bool is_key, int h,
                                              const AppendList& list, T* raw) {
  constexpr int kPer = 16 / sizeof(T);  // values of a 16-byte access
  constexpr int kLanes = ROW / 8;  // of a token
  const int lane = threadIdx.x & 31, d = lane % kLanes * 8;
  const T* base = (is_key ? a.key + (int64_t)h * a.k_head : a.value + (int64_t)h * a.v_head) + d;
  const int64_t step_tok = is_key ? a.k_tok : a.v_tok;
  if (d < a.dim)
    for (int i = lane / kLanes; i < list.count; i += 32 / kLanes)
#pragma unroll
      for (int u = 0; u < 8 / kPer; ++u)
        copy16_async(raw + i * ROW + d + u * kPer, base + list.tok[i] * step_tok + u * kPer);
}

template <typename T, int ROT, int ROW>
__device__ __forceinline__ void append_head8(const AppendArgs<T>& a, int64_t page, bool is_key,
                                             int h, const AppendList& list, const T* raw,
                                             const float* table) {
  constexpr int kLanes = ROW / 8;  // of a token
  const int lane = threadIdx.x & 31, sub = lane / kLanes, d = lane % kLanes * 8;
  const int n = list.count, lowest = list.lowest;
  const bool on = d < a.dim;
  const int64_t tok_stride = (int64_t)a.kv_heads * a.dim;
  const int stride32 = (int)tok_stride;
  int8_t* head_base = a.cache + (is_key ? 0 : a.blocks * a.bs * tok_stride) +
                      page * a.bs * tok_stride + (int64_t)h * a.dim;
  float* scale = a.scales + (is_key ? 0 : a.blocks * a.kv_heads) + page * a.kv_heads + h;
  const float old = lowest > 0 ? *scale : 0.0f;

  // The lane's channels: two groups of 4, with the half layout a group and its
  // partners, so that a rotation needs no other lane.
  const int half = a.rot / 2;
  const bool turned = ROT != kNoRotation && d < a.rot;  // whole pieces: rot % 8 = 0
  const int d0 = ROT == kHalves && turned ? d / 2 : d;
  const int d1 = ROT == kHalves && turned ? half + d / 2 : d + 4;
  auto values = [&](int i, float (&y)[8]) {
    const Chunk<T, 4> x0 = load_chunk<T, 4>(raw + i * ROW + d0);
    const Chunk<T, 4> x1 = load_chunk<T, 4>(raw + i * ROW + d1);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      y[e] = to_f32<T>(x0.e[e]);
      y[4 + e] = to_f32<T>(x1.e[e]);
    }
    if (ROT == kNoRotation || !turned) return;
    const float4 c = *reinterpret_cast<const float4*>(table + i * ROW + d / 2);
    const float4 s = *reinterpret_cast<const float4*>(table + i * ROW + half + d / 2);
    constexpr int kStep = ROT == kPairs ? 2 : 1;  // between the pairs' first values
    constexpr int kOther = ROT == kPairs ? 1 : 4;
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      float* f = &y[e * kStep];
      const uint64_t cc = e == 0 ? f32x2(c.x, c.y) : f32x2(c.z, c.w);
      const uint64_t ss = e == 0 ? f32x2(s.x, s.y) : f32x2(s.z, s.w);
      const uint64_t u = f32x2(f[0], f[kStep]), v = f32x2(f[kOther], f[kOther + kStep]);
      // Packed products, scalar sums: of packed products and a packed sum the
      // assembler makes one fma, with one rounding less.
      const float2 uc = unpack_f32x2(mul_f32x2(u, cc)), us = unpack_f32x2(mul_f32x2(u, ss));
      const float2 vc = unpack_f32x2(mul_f32x2(v, cc)), vs = unpack_f32x2(mul_f32x2(v, ss));
      f[0] = __fsub_rn(uc.x, vs.x), f[kStep] = __fsub_rn(uc.y, vs.y);
      f[kOther] = __fadd_rn(vc.x, us.x), f[kOther + kStep] = __fadd_rn(vc.y, us.y);
    }
  };
  float big = 0.0f;
  if (on)
#pragma unroll 4
    for (int i = sub; i < n; i += 32 / kLanes) {
      float y[8];
      values(i, y);
#pragma unroll
      for (int e = 0; e < 8; e += 2) big = max3_nan(big, fabsf(y[e]), fabsf(y[e + 1]));
    }
  // NaN bits exceed +inf: NaN wins
  const float amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(big)));
  const float sc = append_scale(amax, scale, old, lowest, head_base, tok_stride, a.dim, true);
  const float rcp = __frcp_rn(sc);
  const bool fast = isfinite(amax) && !isinf(rcp);
  if (on)
#pragma unroll 4
    for (int i = sub; i < n; i += 32 / kLanes) {
      float y[8];
      values(i, y);
      const float lo[4] = {y[0], y[1], y[2], y[3]}, hi[4] = {y[4], y[5], y[6], y[7]};
      int8_t* dst = head_base + (int64_t)list.off[i] * stride32;
      const uint32_t w0 = quantize_word(lo, sc, rcp, fast), w1 = quantize_word(hi, sc, rcp, fast);
      if constexpr (ROT == kHalves) {
        *reinterpret_cast<uint32_t*>(dst + d0) = w0;
        *reinterpret_cast<uint32_t*>(dst + d1) = w1;
      } else {
        *reinterpret_cast<uint2*>(dst + d) = make_uint2(w0, w1);
      }
    }
}

// The heads of K, of V or of both by the CTA's warps.  With BUFS = 2 a warp's next
// head is on its way while it works on one.
template <typename T, int VEC, int NC, int HOLD, int BUFS>
__device__ __forceinline__ void append_heads(const AppendArgs<T>& a, int64_t page, bool key_part,
                                             bool value_part, const AppendList& list) {
  // of the CTA's group of heads (blockIdx.y)
  const int per = (a.kv_heads + gridDim.y - 1) / gridDim.y, h0 = blockIdx.y * per;
  const int heads = min(per, a.kv_heads - h0);
  if (heads <= 0) return;  // whole CTA
  const int rows = (key_part ? heads : 0) + (value_part ? heads : 0);
  const int warp = threadIdx.x >> 5;
  const bool turns = a.positions != nullptr;
  auto is_key = [&](int r) { return key_part && r < heads; };
  auto head = [&](int r) { return h0 + (r < heads ? r : r - heads); };
  if (VEC == 8 && list.count <= HOLD) {
    constexpr int ROW = NC * 128;
    extern __shared__ __align__(16) float s_rows[];  // table rows, then each warp's rows
    T* raw = reinterpret_cast<T*>(s_rows + HOLD * ROW) + warp * BUFS * HOLD * ROW;
    if (key_part && turns)  // the tokens' table rows, once for all heads
      for (int i = threadIdx.x; i < list.count * (ROW / 4); i += kAppendThreads) {
        const int tok = i / (ROW / 4), at = i % (ROW / 4) * 4;
        if (at < a.rot) copy16_async(s_rows + tok * ROW + at, a.table + list.pos[tok] * a.rot + at);
      }
    if (warp < rows) append_fetch8<T, ROW>(a, is_key(warp), head(warp), list, raw);
    copies_group();
    for (int r0 = 0, buf = 0; r0 < rows; r0 += kAppendWarps) {
      const int r = r0 + warp, next = r + kAppendWarps;
      if (BUFS == 2) {
        if (next < rows) append_fetch8<T, ROW>(a, is_key(next), head(next), list, raw + (buf ^ 1) * HOLD * ROW);
        copies_group();
        copies_wait<1>();
      } else {
        copies_wait<0>();
      }
      if (r0 == 0) __syncthreads();  // the table rows are every warp's copies
      else __syncwarp();
      if (r >= rows) continue;
      const T* rows_of = raw + buf * HOLD * ROW;
      if (!is_key(r) || !turns)
        append_head8<T, kNoRotation, ROW>(a, page, is_key(r), head(r), list, rows_of, s_rows);
      else if (a.interleaved)
        append_head8<T, kPairs, ROW>(a, page, true, head(r), list, rows_of, s_rows);
      else
        append_head8<T, kHalves, ROW>(a, page, true, head(r), list, rows_of, s_rows);
      __syncwarp();  // the rows are free for another head
      if (BUFS == 2) {
        buf ^= 1;
      } else if (next < rows) {
        append_fetch8<T, ROW>(a, is_key(next), head(next), list, raw);
        copies_group();
      }
    }
    return;
  }
  constexpr int kVec = VEC == 8 ? 4 : VEC;
  for (int r = warp; r < rows; r += kAppendWarps) {
    if (!is_key(r) || !turns)
      append_head<T, kVec, NC, kNoRotation>(a, page, is_key(r), head(r), list);
    else if (a.interleaved)
      append_head<T, kVec, NC, kPairs>(a, page, true, head(r), list);
    else
      append_head<T, kVec, NC, kHalves>(a, page, true, head(r), list);
  }
}

// Up to kAppendScan tokens: CTA (t, K/V; 8 heads) handles the page of token t if no
// earlier token of the call is in that page.
template <typename T, int VEC, int NC>
__global__ void __launch_bounds__(kAppendThreads) append_scan_kernel(AppendArgs<T> a, int* err) {
  __shared__ int s_tok[kAppendMaxPage];
  __shared__ AppendList s_list;
  __shared__ int s_taken;
  const int64_t t = blockIdx.x >> 1;
  const bool is_key = (blockIdx.x & 1) == 0;
  const int64_t slot = append_slot(a, t, err);
  if (slot < 0) return;  // whole CTA
  const int64_t page = slot / a.bs;
  if (t > 0) {  // most tokens of a prompt follow one in their page
    const int64_t before = append_slot(a, t - 1, err);
    if (before >= page * a.bs && before < (page + 1) * a.bs) return;
  }
  for (int i = threadIdx.x; i < a.bs; i += kAppendThreads) s_tok[i] = -1;
  if (threadIdx.x == 0) s_taken = 0;
  __syncthreads();
  for (int64_t u = threadIdx.x; u < a.tokens; u += kAppendThreads) {
    const int64_t su = append_slot(a, u, err);
    if (su < 0 || su / a.bs != page) continue;
    if (u < t) s_taken = 1;
    atomicMax(&s_tok[su % a.bs], (int)u);  // of equal slots the last token counts
  }
  __syncthreads();
  if (s_taken) return;  // whole CTA
  append_list(a, s_tok, s_list);
  append_heads<T, VEC, NC, kAppendHold, 1>(a, page, is_key, !is_key, s_list);
}

// Index of larger calls.  A run head (a token whose predecessor is not in the
// same page) pushes itself on its page's list: head[page] = last pushed + 1
// (0: none), next[t] = the one before.  The first to push lists the page and
// itself.
template <typename T>
__global__ void __launch_bounds__(256)
    append_index_kernel(AppendArgs<T> a, int* head, int* next, int2* pages, int* count, int* err) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= a.tokens) return;
  const int64_t slot = append_slot(a, t, err);
  if (slot < 0) return;
  const int64_t page = slot / a.bs;
  if (t > 0) {
    const int64_t before = append_slot(a, t - 1, err);
    if (before >= 0 && before / a.bs == page) return;
  }
  const int prev = atomicExch(&head[page], (int)t + 1);
  next[t] = prev;
  if (prev == 0) pages[atomicAdd(count, 1)] = make_int2((int)page, (int)t);
}

// Rows on chip, HOLD tokens of NC x 128 channels: two heads a warp where three CTAs
// of an SM can have them, else one.
template <typename T, int NC, int HOLD>
constexpr int kAppendBufs = HOLD * NC * (int)sizeof(T) <= 32 ? 2 : 1;
template <typename T, int NC, int HOLD>
constexpr int kAppendStage =
    HOLD * NC * 128 * (4 + kAppendWarps * kAppendBufs<T, NC, HOLD> * (int)sizeof(T));
constexpr int append_ctas(int bytes) { return bytes <= 75 * 1024 ? 3 : bytes <= 112 * 1024 ? 2 : 1; }

template <typename T, int VEC, int NC, int HOLD>
__global__ void __launch_bounds__(kAppendThreads,
                                  VEC == 8 ? append_ctas(kAppendStage<T, NC, HOLD>) : 1)
    append_pages_kernel(AppendArgs<T> a, const int* head, const int* next, const int2* pages,
                        const int* count, int* err) {
  __shared__ int s_tok[kAppendMaxPage];
  __shared__ AppendList s_list;
  const int units = *count;
  for (int u = blockIdx.x; u < units; u += gridDim.x) {
    const int2 entry = pages[u];
    const int64_t page = entry.x;
    __syncthreads();  // the previous unit is done with s_tok and s_list
    for (int i = threadIdx.x; i < a.bs; i += kAppendThreads) s_tok[i] = -1;
    __syncthreads();
    if (threadIdx.x < 32) {
      // the run of the token that listed the page, then the runs pushed after it
      int link = head[page];
      for (int64_t start = entry.y;;) {
        for (int64_t t0 = start; t0 < a.tokens; t0 += 32) {
          const int64_t t = t0 + threadIdx.x;
          const int64_t slot = t < a.tokens ? append_slot(a, t, err) : -1;
          const int64_t at = slot - page * a.bs;
          const bool in = slot >= 0 && at >= 0 && at < a.bs;
          // the run ends at the first token of another page
          const unsigned out = __ballot_sync(0xffffffffu, !in);
          const int len = out == 0 ? 32 : __ffs(out) - 1;
          if ((int)threadIdx.x < len) atomicMax(&s_tok[at], (int)t);
          if (len < 32) break;
        }
        start = link - 1;
        if (start == entry.y) break;
        link = next[start];
      }
    }
    __syncthreads();
    append_list(a, s_tok, s_list);
    append_heads<T, VEC, NC, HOLD, kAppendBufs<T, NC, HOLD>>(a, page, true, true, s_list);
  }
}

// Largest call that scans its slots in every CTA, a launch instead of three.  us on the
// device, scan and index (bf16, 128 channels, pages of 16), prompts: 8 heads, 256
// tokens 12.0 and 19.5, 512 15.2 and 20.8, 1,024 21.2 and 22.7, 2,048 34.8 and 23.6;
// 40 heads, 256 22.0 and 24.0, 512 37.1 and 27.9.  Single tokens of as many
// sequences: 8 heads, 256 11.1 and 12.9, 512 17.1 and 18.8, 768 24.4 and 21.6; 40 heads,
// 128 17.4 and 19.3, 256 31.4 and 29.8, 512 63.5 and 45.2.
constexpr int64_t kAppendScan = 512;

template <typename T, int VEC, int NC>
void launch_append_n(const AppendArgs<T>& a, int* ws, cudaStream_t stream) {
  int* err = device_error_word();
  if (a.tokens <= kAppendScan) {
    if constexpr (VEC == 8 && NC == 2) {
      return launch_append_n<T, 4, 2>(a, ws, stream);  // few tokens a page, more CTAs an SM
    } else {
      constexpr int kStage = VEC == 8 ? kAppendHold * 128 * (4 + kAppendWarps * (int)sizeof(T)) : 0;
      auto kernel = append_scan_kernel<T, VEC, NC>;
      static std::atomic<uint64_t> done{0};
      allow_shared_memory(reinterpret_cast<const void*>(kernel), kStage, done);
      // 8 heads a CTA: 500 tokens of 40 heads of 256 channels in pages of 64 take 150 us
      // a call, 548 with all heads in one (in pages of 16, 128 channels: 38 and 36).
      const dim3 grid((unsigned)(2 * a.tokens), (unsigned)((a.kv_heads + 7) / 8));
      kernel<<<grid, kAppendThreads, kStage, stream>>>(a, err);
      return;
    }
  }
  int* head = ws;
  int* count = ws + a.blocks;
  int* next = count + 1;
  int2* pages = reinterpret_cast<int2*>(next + a.tokens + ((a.blocks + 1 + a.tokens) & 1));  // ws is 8-byte aligned
  cudaMemsetAsync(head, 0, (size_t)(a.blocks + 1) * sizeof(int), stream);
  append_index_kernel<T><<<(unsigned)((a.tokens + 255) / 256), 256, 0, stream>>>(a, head, next,
                                                                                 pages, count, err);
  // Few pages are shared among CTAs by groups of 8 heads, up to three CTAs an SM: 2,000
  // tokens of 40 heads in pages of 32 take 53 us, 88 with a CTA per page.
  const int64_t full = std::max<int64_t>(a.tokens / a.bs, 1);
  const int64_t groups =
      std::max<int64_t>(std::min<int64_t>((a.kv_heads + 7) / 8, 3 * 148 / full), 1);
  const dim3 grid((unsigned)std::min<int64_t>(a.tokens, 8 * 148 / groups), (unsigned)groups);
  auto pages_of = [&](auto hold) {
    constexpr int kHold = decltype(hold)::value;
    constexpr int kStage = VEC == 8 ? kAppendStage<T, NC, kHold> : 0;
    static_assert(kStage <= 227 * 1024 - 4096, "shared memory");
    auto kernel = append_pages_kernel<T, VEC, NC, kHold>;
    static std::atomic<uint64_t> done{0};
    allow_shared_memory(reinterpret_cast<const void*>(kernel), kStage, done);
    kernel<<<grid, kAppendThreads, kStage, stream>>>(a, head, next, pages, count, err);
  };
  // Larger pages are kept whole as far as shared memory goes.  16,384 tokens of 8
  // heads, us a call, against rows read twice (append_head): bf16 in pages of 32 61
  // and 162, of 64 82 and 175; fp32 in pages of 32 84 and 168.
  if constexpr (VEC == 8 && sizeof(T) * NC <= 2) {
    if (a.bs > 32) return pages_of(std::integral_constant<int, 64>{});
  }
  if constexpr (VEC == 8 && sizeof(T) * NC <= 4) {
    if (a.bs > kAppendHold) return pages_of(std::integral_constant<int, 32>{});
  }
  pages_of(std::integral_constant<int, kAppendHold>{});
}

template <typename T>
int launch_append_t(const AppendKvArgs& p, int* ws, cudaStream_t stream) {
  AppendArgs<T> a;
  a.key = static_cast<const T*>(p.key);
  a.value = static_cast<const T*>(p.value);
  a.k_tok = p.k_token_stride;
  a.k_head = p.k_head_stride;
  a.v_tok = p.v_token_stride;
  a.v_head = p.v_head_stride;
  a.cache = p.cache;
  a.scales = p.scales;
  a.slots = p.slots;
  a.positions = p.positions;
  a.table = p.table;
  a.tokens = p.tokens;
  a.blocks = p.blocks;
  a.table_rows = p.table_rows;
  a.bs = p.block_size;
  a.kv_heads = p.kv_heads;
  a.dim = p.dim;
  a.rot = p.positions != nullptr ? p.rot : 0;
  a.interleaved = p.interleaved;
  auto aligned = [](const void* x, int n) { return reinterpret_cast<uintptr_t>(x) % n == 0; };
  auto rows_of = [&](int n, int bytes) {  // values and strides in pieces of n
    return a.dim % n == 0 && a.k_tok % n == 0 && a.k_head % n == 0 && a.v_tok % n == 0 &&
           a.v_head % n == 0 && aligned(a.key, bytes) && aligned(a.value, bytes);
  };
  // whole pieces are rotated, and table rows are read four values at a time
  const bool halves = a.rot > 0 && !a.interleaved;
  if (rows_of(8, 16) && aligned(a.cache, 8) && a.rot % 8 == 0 &&
      (a.rot == 0 || aligned(a.table, 16)))
    a.dim <= 128 ? launch_append_n<T, 8, 1>(a, ws, stream) : launch_append_n<T, 8, 2>(a, ws, stream);
  else if (rows_of(4, 4 * (int)sizeof(T)) && aligned(a.cache, 4) &&
           (!halves || (a.rot % 8 == 0 && aligned(a.table, 16))))
    launch_append_n<T, 4, 2>(a, ws, stream);
  else
    launch_append_n<T, 1, 8>(a, ws, stream);
  return kOk;
}

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return kOk;
  set_error(std::string(what) + " launch failed: " + cudaGetErrorString(e));
  return kCudaError;
}

}  // namespace

int launch_qk_norm_rope(const QkNormRopeArgs& a, cudaStream_t stream) {
  if (a.tokens == 0 || a.heads + a.kv_heads == 0) return kOk;
  switch (a.dtype) {
    case 0: launch_qk_t<float>(a, stream); break;
    case 1: launch_qk_t<__half>(a, stream); break;
    case 2: launch_qk_t<__nv_bfloat16>(a, stream); break;
    default: set_error("unknown dtype code"); return kInvalidArgument;
  }
  return launched("qk_norm_rope");
}

size_t append_kv_workspace_size(int64_t tokens, int64_t blocks) {
  if (tokens <= kAppendScan) return 0;
  // list heads, page count, links, (page, first token) on an 8-byte boundary
  return (size_t)(blocks + 1 + tokens + 1 + 2 * tokens) * sizeof(int) + 8;
}

int launch_append_kv(const AppendKvArgs& a, void* workspace, size_t workspace_bytes,
                     cudaStream_t stream) {
  if (a.tokens == 0) return kOk;
  if (append_kv_workspace_size(a.tokens, a.blocks) > workspace_bytes ||
      (a.tokens > kAppendScan && workspace == nullptr)) {
    set_error("workspace too small for append_kv");
    return kWorkspace;
  }
  int* ws = reinterpret_cast<int*>((reinterpret_cast<uintptr_t>(workspace) + 7) & ~(uintptr_t)7);
  switch (a.dtype) {
    case 0: launch_append_t<float>(a, ws, stream); break;
    case 1: launch_append_t<__half>(a, ws, stream); break;
    case 2: launch_append_t<__nv_bfloat16>(a, ws, stream); break;
    default: set_error("unknown dtype code"); return kInvalidArgument;
  }
  return launched("append_kv");
}

}  // namespace pkv
