// Appending rows to a paged cache with the position rotation on the way, and
// gathering them back (sm_100a).
//
// Token t of request b at position p writes, for every KV head,
//     K'(2 elements of RoPE pair i) = (x1 cos - x2 sin, x2 cos + x1 sin),
//     angle = p * inv_freq[i],
// and its V row to row (table[b][p / bs], p % bs); query rows are rotated
// beside it.  All three kernels move each byte once and are bound by HBM (by
// launch latency for a decode step): a CTA takes a few tokens, computes their
// angles once for all heads into shared memory, and its threads move two
// vectors of up to 16 bytes per row, the two halves the neox pairs lie in.
#include <algorithm>

#include "paged.cuh"
#include "prof.cuh"

namespace sb {
namespace {

using paged::find_block;
using paged::find_request;

constexpr int kThreads = 256;
constexpr int kMaxTokens = 4;  // tokens of a CTA

// Where a CTA's tokens go; filled by its first threads.
struct TokenSlot {
  int64_t position;
  int64_t offset;  // of the row inside the cache (kv 0, head 0), elements or code bytes; -1: none
  int64_t scale_offset;
  int active;      // 0: padding
};

__device__ __forceinline__ void resolve_token(const sb_paged_cache &C, const sb_paged_batch &B, int t,
                                              TokenSlot &s, unsigned long long *err) {
  s.offset = -1;
  s.scale_offset = 0;
  s.active = 0;
  const int b = find_request(B, t);
  if (b < 0) return;
  const int64_t p = paged::index_at(B.positions, t, B.pos_dtype);
  s.active = 1;
  s.position = p;
  const int64_t lb = p < 0 ? -1 : p / C.block_size;
  const int phys = find_block(B, b, lb, C.n_blocks);
  if (phys < 0) {
    if (err) atomicAdd(err, 1ull);
    return;
  }
  const int64_t in_block = p - lb * C.block_size;
  s.offset = phys * C.stride_block + in_block * C.stride_pos;
  s.scale_offset = phys * C.scale_block + in_block * C.scale_pos;
}

struct AppendParams {
  sb_paged_cache cache;
  sb_paged_batch batch;
  sb_token_rows key, value, query, query_out;
  const double *inv_freq;
  unsigned long long *err;
  int n_q_heads;
  int rows;  // rows per token: K heads, V heads, query heads
  int tokens_per_cta;
};

// cos and sin of p * f to fp32: the turn is reduced to [-1/2, 1/2] in 64 bits
// (positions reach millions of radians, where an fp32 angle has lost its
// fraction) and only the fraction is rounded.
__device__ __forceinline__ float2 turn(int64_t p, double f) {
  constexpr double kInvTwoPi = 0.15915494309189533577;
  double r = (double)p * f * kInvTwoPi;
  r -= rint(r);
  float2 cs;
  sincospif(2.f * (float)r, &cs.y, &cs.x);
  return cs;
}

template <typename T, int VEC, bool ROTATE, bool NEOX>
__device__ __forceinline__ void move_row(const T *src, T *dst, int lane, int half, const float2 *cs) {
  // two vectors of the row: its RoPE pairs lie across them (neox) or inside each (interleaved)
  const int d0 = (VEC == 1 && !NEOX) ? 2 * lane : lane * VEC;
  const int d1 = (VEC == 1 && !NEOX) ? 2 * lane + 1 : half + lane * VEC;
  Vec<T, VEC> a, b;
  load_vec(a, src + d0);
  load_vec(b, src + d1);
  if (ROTATE) {
    if (NEOX || VEC == 1) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float2 w = cs[lane * VEC + i];
        const float x = Elem<T>::to_f32(a.e[i]), y = Elem<T>::to_f32(b.e[i]);
        a.e[i] = Elem<T>::from_f32(x * w.x - y * w.y);
        b.e[i] = Elem<T>::from_f32(y * w.x + x * w.y);
      }
    } else {
#pragma unroll
      for (int i = 0; i + 1 < VEC; i += 2) {
        const float2 w = cs[(d0 + i) / 2], u = cs[(d1 + i) / 2];
        const float x = Elem<T>::to_f32(a.e[i]), y = Elem<T>::to_f32(a.e[i + 1]);
        const float p = Elem<T>::to_f32(b.e[i]), q = Elem<T>::to_f32(b.e[i + 1]);
        a.e[i] = Elem<T>::from_f32(x * w.x - y * w.y);
        a.e[i + 1] = Elem<T>::from_f32(y * w.x + x * w.y);
        b.e[i] = Elem<T>::from_f32(p * u.x - q * u.y);
        b.e[i + 1] = Elem<T>::from_f32(q * u.x + p * u.y);
      }
    }
  }
  store_vec(dst + d0, a);
  store_vec(dst + d1, b);
}

template <typename T, int VEC, bool NEOX>
__global__ void __launch_bounds__(kThreads) append_kernel(const AppendParams P) {
  __shared__ TokenSlot slot[kMaxTokens];
  __shared__ float2 cs[kMaxTokens][256];  // head_dim <= 512
  const int D = P.cache.head_dim, half = D / 2, H = P.cache.n_heads;
  const int t0 = blockIdx.x * P.tokens_per_cta;
  const int n = min(P.tokens_per_cta, P.batch.n_tokens - t0);
  if (threadIdx.x < n) resolve_token(P.cache, P.batch, t0 + threadIdx.x, slot[threadIdx.x], P.err);
  if (P.inv_freq != nullptr)
    for (int i = threadIdx.x; i < n * half; i += blockDim.x) {
      const int k = i / half, c = i - k * half;
      cs[k][c] = turn(paged::index_at(P.batch.positions, t0 + k, P.batch.pos_dtype), P.inv_freq[c]);
    }
  __syncthreads();
  const int lanes = half / VEC;  // threads a row
  const int lane = threadIdx.x % lanes, first = threadIdx.x / lanes, step = blockDim.x / lanes;
  if (first >= step) return;  // lanes does not divide the block: the last threads have no row
  for (int r = first; r < n * P.rows; r += step) {
    const int k = r / P.rows, row = r - k * P.rows;
    const TokenSlot &s = slot[k];
    if (!s.active) continue;
    const int64_t t = t0 + k;
    if (row < 2 * H) {
      if (s.offset < 0) continue;
      const int kv = row >= H, h = row - kv * H;
      const sb_token_rows &src = kv ? P.value : P.key;
      const T *from = reinterpret_cast<const T *>(src.data) + t * src.stride_token + h * src.stride_head;
      T *to = reinterpret_cast<T *>(P.cache.data) + s.offset + kv * P.cache.stride_kv + h * P.cache.stride_head;
      if (kv || P.inv_freq == nullptr) move_row<T, VEC, false, NEOX>(from, to, lane, half, cs[k]);
      else move_row<T, VEC, true, NEOX>(from, to, lane, half, cs[k]);
    } else {
      const int h = row - 2 * H;
      const T *from = reinterpret_cast<const T *>(P.query.data) + t * P.query.stride_token + h * P.query.stride_head;
      T *to = reinterpret_cast<T *>(P.query_out.data) + t * P.query_out.stride_token + h * P.query_out.stride_head;
      if (P.inv_freq == nullptr) move_row<T, VEC, false, NEOX>(from, to, lane, half, cs[k]);
      else move_row<T, VEC, true, NEOX>(from, to, lane, half, cs[k]);
    }
  }
}

// ---------------------------------------------------------------------------
// 4-bit cache
// ---------------------------------------------------------------------------
// A row belongs to head_dim / 16 threads; thread j holds elements [8j, 8j + 8)
// and [D/2 + 8j, D/2 + 8j + 8).  A group is then whole threads of one half, or
// (group == head_dim) both halves of all of the row's threads.
__device__ __forceinline__ uint32_t pack_codes(const float (&x)[8], float zero, float inv) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // one rounding each, so that the codes are a function of the fp32 values alone
    const float c = rintf(__fmul_rn(__fsub_rn(x[i], zero), inv));
    w |= (uint32_t)fminf(fmaxf(c, 0.f), 15.f) << (4 * i);
  }
  return w;
}

// NaN in, NaN out: a group that holds one reads back as NaN.
__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float saturate_half(float x) { return min_nan(max_nan(x, -65504.f), 65504.f); }

// step and zero of a group from its extremes, and 1 / step (0 for a group of equal values)
__device__ __forceinline__ __half2 group_scale(float lo, float hi, float &zero, float &inv) {
  const __half z = __float2half_rn(saturate_half(lo));
  const __half st = __float2half_rn(min_nan(__fdiv_rn(__fsub_rn(hi, lo), 15.f), 65504.f));
  zero = __half2float(z);
  const float s = __half2float(st);
  inv = s > 0.f ? __fdiv_rn(1.f, s) : 0.f;
  return __halves2half2(st, z);
}

template <typename T>
__device__ __forceinline__ void load8(float (&x)[8], const T *p, bool aligned) {
  if (aligned) {
    constexpr int kV = 16 / sizeof(T);
#pragma unroll
    for (int v = 0; v < 8 / kV; ++v) {
      Vec<T, kV> a;
      load_vec(a, p + v * kV);
#pragma unroll
      for (int i = 0; i < kV; ++i) x[v * kV + i] = Elem<T>::to_f32(a.e[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = Elem<T>::to_f32(p[i]);
  }
}

// Rotation in 64 bits, one rounding to fp32.
__device__ __forceinline__ void turn_pair(float &x, float &y, double2 w) {
  const double a = x, b = y;
  x = (float)(a * w.x - b * w.y);
  y = (float)(b * w.x + a * w.y);
}

template <typename T, bool NEOX>
__global__ void __launch_bounds__(kThreads) append4_kernel(const AppendParams P, const bool aligned) {
  __shared__ TokenSlot slot[kMaxTokens];
  __shared__ double2 cs[kMaxTokens][64];
  const int D = P.cache.head_dim, half = D / 2, H = P.cache.n_heads;
  const int t0 = blockIdx.x * P.tokens_per_cta;
  const int n = min(P.tokens_per_cta, P.batch.n_tokens - t0);
  if (threadIdx.x < n) resolve_token(P.cache, P.batch, t0 + threadIdx.x, slot[threadIdx.x], P.err);
  if (P.inv_freq != nullptr)
    for (int i = threadIdx.x; i < n * half; i += blockDim.x) {
      const int k = i / half, c = i - k * half;
      double2 w;
      sincos((double)paged::index_at(P.batch.positions, t0 + k, P.batch.pos_dtype) * P.inv_freq[c], &w.y, &w.x);
      cs[k][c] = w;
    }
  __syncthreads();
  const int lanes = D / 16;  // 4 or 8 threads a row: whole rows in a warp
  const int lane = threadIdx.x % lanes, first = threadIdx.x / lanes, step = kThreads / lanes;
  const int group = P.cache.group;
  const int total = n * P.rows;
  // every thread of a warp takes the same number of turns (the shuffles need all of them)
  for (int r0 = 0; r0 < total; r0 += step) {
    const int r = r0 + first;
    const int k = min(r / P.rows, n - 1), row = r - k * P.rows;
    const TokenSlot &s = slot[k];
    const bool live = r < total && s.active;
    const bool is_q = row >= 2 * H;
    const int kv = row >= H, h = is_q ? row - 2 * H : row - kv * H;
    const bool write = live && (is_q || s.offset >= 0);
    float a[8], b[8];
    const sb_token_rows &src = is_q ? P.query : kv ? P.value : P.key;
    if (write) {
      const T *from = reinterpret_cast<const T *>(src.data) + (int64_t)(t0 + k) * src.stride_token + h * src.stride_head;
      load8(a, from + lane * 8, aligned);
      load8(b, from + half + lane * 8, aligned);
      if (P.inv_freq != nullptr && (is_q || !kv)) {
        if (NEOX) {
#pragma unroll
          for (int i = 0; i < 8; ++i) turn_pair(a[i], b[i], cs[k][lane * 8 + i]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            turn_pair(a[i], a[i + 1], cs[k][(lane * 8 + i) / 2]);
            turn_pair(b[i], b[i + 1], cs[k][(half + lane * 8 + i) / 2]);
          }
        }
      }
      if (is_q) {
        T *to = reinterpret_cast<T *>(P.query_out.data) + (int64_t)(t0 + k) * P.query_out.stride_token +
                h * P.query_out.stride_head;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          to[lane * 8 + i] = Elem<T>::from_f32(a[i]);
          to[half + lane * 8 + i] = Elem<T>::from_f32(b[i]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = b[i] = 0.f;
    }
    float lo0 = a[0], hi0 = a[0], lo1 = b[0], hi1 = b[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      lo0 = min_nan(lo0, a[i]), hi0 = max_nan(hi0, a[i]);
      lo1 = min_nan(lo1, b[i]), hi1 = max_nan(hi1, b[i]);
    }
    if (group == D) {
      lo0 = lo1 = min_nan(lo0, lo1);
      hi0 = hi1 = max_nan(hi0, hi1);
    }
    const int span = group == D ? lanes : group / 8;
    for (int o = 1; o < span; o <<= 1) {
      lo0 = min_nan(lo0, __shfl_xor_sync(0xffffffffu, lo0, o)), hi0 = max_nan(hi0, __shfl_xor_sync(0xffffffffu, hi0, o));
      lo1 = min_nan(lo1, __shfl_xor_sync(0xffffffffu, lo1, o)), hi1 = max_nan(hi1, __shfl_xor_sync(0xffffffffu, hi1, o));
    }
    if (!write || is_q) continue;
    float zero0, inv0, zero1, inv1;
    const __half2 s0 = group_scale(lo0, hi0, zero0, inv0), s1 = group_scale(lo1, hi1, zero1, inv1);
    uint8_t *codes = reinterpret_cast<uint8_t *>(P.cache.data) + s.offset + kv * P.cache.stride_kv +
                     h * P.cache.stride_head;
    *reinterpret_cast<uint32_t *>(codes + lane * 4) = pack_codes(a, zero0, inv0);
    *reinterpret_cast<uint32_t *>(codes + half / 2 + lane * 4) = pack_codes(b, zero1, inv1);
    __half2 *scales = reinterpret_cast<__half2 *>(reinterpret_cast<__half *>(P.cache.scales) + s.scale_offset +
                                                  kv * P.cache.scale_kv + h * P.cache.scale_head);
    if (group == D) {
      if (lane == 0) scales[0] = s0;
    } else if (lane % span == 0) {
      scales[lane * 8 / group] = s0;
      scales[(half + lane * 8) / group] = s1;
    }
  }
}

// ---------------------------------------------------------------------------
// Gather
// ---------------------------------------------------------------------------
struct GatherParams {
  sb_paged_cache cache;
  sb_paged_batch batch;
  sb_token_rows out[2];
  unsigned long long *err;
  int tokens_per_cta;
};

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) gather_kernel(const GatherParams P) {
  __shared__ TokenSlot slot[kMaxTokens];
  const int H = P.cache.n_heads, rows = 2 * H;
  const int t0 = blockIdx.x * P.tokens_per_cta;
  const int n = min(P.tokens_per_cta, P.batch.n_tokens - t0);
  if (threadIdx.x < n) resolve_token(P.cache, P.batch, t0 + threadIdx.x, slot[threadIdx.x], P.err);
  __syncthreads();
  const int lanes = P.cache.head_dim / VEC;
  for (int i = threadIdx.x; i < n * rows * lanes; i += kThreads) {
    const int r = i / lanes, lane = i - r * lanes;
    const int k = r / rows, row = r - k * rows;
    const TokenSlot &s = slot[k];
    if (s.offset < 0) continue;
    const int kv = row >= H, h = row - kv * H;
    const T *from = reinterpret_cast<const T *>(P.cache.data) + s.offset + kv * P.cache.stride_kv + h * P.cache.stride_head;
    T *to = reinterpret_cast<T *>(P.out[kv].data) + (int64_t)(t0 + k) * P.out[kv].stride_token +
            h * P.out[kv].stride_head;
    Vec<T, VEC> v;
    load_vec(v, from + lane * VEC);
    store_vec(to + lane * VEC, v);
  }
}

// A thread expands 8 codes (4 bytes) of one group to 8 elements.
template <typename T>
__global__ void __launch_bounds__(kThreads) gather4_kernel(const GatherParams P, const bool aligned) {
  __shared__ TokenSlot slot[kMaxTokens];
  const int H = P.cache.n_heads, rows = 2 * H;
  const int t0 = blockIdx.x * P.tokens_per_cta;
  const int n = min(P.tokens_per_cta, P.batch.n_tokens - t0);
  if (threadIdx.x < n) resolve_token(P.cache, P.batch, t0 + threadIdx.x, slot[threadIdx.x], P.err);
  __syncthreads();
  const int lanes = P.cache.head_dim / 8;
  for (int i = threadIdx.x; i < n * rows * lanes; i += kThreads) {
    const int r = i / lanes, lane = i - r * lanes;
    const int k = r / rows, row = r - k * rows;
    const TokenSlot &s = slot[k];
    if (s.offset < 0) continue;
    const int kv = row >= H, h = row - kv * H;
    const uint8_t *codes = reinterpret_cast<const uint8_t *>(P.cache.data) + s.offset + kv * P.cache.stride_kv +
                           h * P.cache.stride_head;
    const __half2 *scales = reinterpret_cast<const __half2 *>(reinterpret_cast<const __half *>(P.cache.scales) +
                                                              s.scale_offset + kv * P.cache.scale_kv +
                                                              h * P.cache.scale_head);
    const uint32_t w = *reinterpret_cast<const uint32_t *>(codes + lane * 4);
    const float2 sz = __half22float2(scales[lane * 8 / P.cache.group]);
    T *to = reinterpret_cast<T *>(P.out[kv].data) + (int64_t)(t0 + k) * P.out[kv].stride_token +
            h * P.out[kv].stride_head + lane * 8;
    T v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = Elem<T>::from_f32(fmaf((float)((w >> (4 * j)) & 15u), sz.x, sz.y));
    if (aligned) {
      constexpr int kV = 16 / sizeof(T);
#pragma unroll
      for (int j = 0; j < 8; j += kV) store_vec(to + j, *reinterpret_cast<const Vec<T, kV> *>(v + j));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) to[j] = v[j];
    }
  }
}

// Tokens a CTA takes: one while that leaves SMs without work, else four (the angles of four
// tokens of head_dim 128 are one per thread).
int tokens_per_cta(int n_tokens) { return n_tokens >= 4 * kMaxTokens * paged::sm_count() ? kMaxTokens : 1; }

template <typename T, int VEC>
void launch_append(const AppendParams &P, bool neox, int grid, cudaStream_t st) {
  if (neox) append_kernel<T, VEC, true><<<grid, kThreads, 0, st>>>(P);
  else append_kernel<T, VEC, false><<<grid, kThreads, 0, st>>>(P);
}

// The widest vector every row of the call can be moved in: 16 bytes, or one element.
template <typename T>
int append_rows(const AppendParams &P, bool neox, int grid, cudaStream_t st) {
  constexpr int kV = 16 / (int)sizeof(T);
  const int es = (int)sizeof(T);
  const bool wide = (P.cache.head_dim / 2) % kV == 0 && paged::cache_aligned(P.cache, es, 16) &&
                    paged::rows_aligned(P.key, es, 16) && paged::rows_aligned(P.value, es, 16) &&
                    paged::rows_aligned(P.query, es, 16) && paged::rows_aligned(P.query_out, es, 16);
  const int slot = prof_before(st);
  if (wide) launch_append<T, kV>(P, neox, grid, st);
  else launch_append<T, 1>(P, neox, grid, st);
  prof_after(slot, st);
  return launch_status();
}

template <typename T>
int append_codes(const AppendParams &P, bool neox, int grid, cudaStream_t st) {
  const bool wide = paged::rows_aligned(P.key, sizeof(T), 16) && paged::rows_aligned(P.value, sizeof(T), 16) &&
                    paged::rows_aligned(P.query, sizeof(T), 16);
  const int slot = prof_before(st);
  if (neox) append4_kernel<T, true><<<grid, kThreads, 0, st>>>(P, wide);
  else append4_kernel<T, false><<<grid, kThreads, 0, st>>>(P, wide);
  prof_after(slot, st);
  return launch_status();
}

template <typename T>
int gather_rows(const GatherParams &P, int grid, cudaStream_t st) {
  constexpr int kV = 16 / (int)sizeof(T);
  const int es = (int)sizeof(T);
  const bool out_wide = paged::rows_aligned(P.out[0], es, 16) && paged::rows_aligned(P.out[1], es, 16);
  const int slot = prof_before(st);
  if (P.cache.group != 0) gather4_kernel<T><<<grid, kThreads, 0, st>>>(P, out_wide);
  else if (out_wide && P.cache.head_dim % kV == 0 && paged::cache_aligned(P.cache, es, 16))
    gather_kernel<T, kV><<<grid, kThreads, 0, st>>>(P);
  else gather_kernel<T, 1><<<grid, kThreads, 0, st>>>(P);
  prof_after(slot, st);
  return launch_status();
}

}  // namespace
}  // namespace sb

extern "C" SB_API int sb_paged_append(const sb_paged_cache *cache, const sb_paged_batch *batch, sb_token_rows key,
                                      sb_token_rows value, sb_token_rows query, sb_token_rows query_out,
                                      int32_t n_q_heads, int32_t dtype, const double *inv_freq,
                                      int32_t rotary_style, uint64_t *err_counter, void *stream) {
  using namespace sb;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int s = paged::check_cache(cache);
  if (s == SB_OK) s = paged::check_batch(batch);
  if (s != SB_OK) return s;
  if (!elem_bytes(dtype)) return SB_ERR_UNSUPPORTED;
  if (cache->group == 0 && cache->dtype != dtype) return SB_ERR_INVALID_ARGUMENT;
  if (rotary_style != SB_ROTARY_NEOX && rotary_style != SB_ROTARY_INTERLEAVED) return SB_ERR_INVALID_ARGUMENT;
  if (cache->head_dim % 2 || cache->head_dim > 512) return SB_ERR_UNSUPPORTED;
  if ((query.data == nullptr) != (query_out.data == nullptr) || (query.data && n_q_heads <= 0))
    return SB_ERR_INVALID_ARGUMENT;
  if (batch->batch == 0 || batch->n_tokens == 0) return SB_OK;
  if (!key.data || !value.data) return SB_ERR_INVALID_ARGUMENT;
  AppendParams P;
  P.cache = *cache, P.batch = *batch;
  P.key = key, P.value = value;
  if (query.data) P.query = query, P.query_out = query_out;
  else P.query = P.query_out = sb_token_rows{nullptr, 0, 0};
  P.inv_freq = inv_freq;
  P.err = reinterpret_cast<unsigned long long *>(err_counter);
  P.n_q_heads = query.data ? n_q_heads : 0;
  P.rows = 2 * cache->n_heads + P.n_q_heads;
  P.tokens_per_cta = tokens_per_cta(batch->n_tokens);
  const int grid = (batch->n_tokens + P.tokens_per_cta - 1) / P.tokens_per_cta;
  const bool neox = rotary_style == SB_ROTARY_NEOX;
  const bool codes = cache->group != 0;
  switch (dtype) {
    case SB_DTYPE_F32: return codes ? append_codes<float>(P, neox, grid, st) : append_rows<float>(P, neox, grid, st);
    case SB_DTYPE_F16: return codes ? append_codes<__half>(P, neox, grid, st) : append_rows<__half>(P, neox, grid, st);
    default:
      return codes ? append_codes<__nv_bfloat16>(P, neox, grid, st) : append_rows<__nv_bfloat16>(P, neox, grid, st);
  }
}

extern "C" SB_API int sb_paged_gather(const sb_paged_cache *cache, const sb_paged_batch *batch,
                                      sb_token_rows key_out, sb_token_rows value_out, int32_t dtype,
                                      uint64_t *err_counter, void *stream) {
  using namespace sb;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int s = paged::check_cache(cache);
  if (s == SB_OK) s = paged::check_batch(batch);
  if (s != SB_OK) return s;
  if (!elem_bytes(dtype)) return SB_ERR_UNSUPPORTED;
  if (cache->group == 0 && cache->dtype != dtype) return SB_ERR_INVALID_ARGUMENT;
  if (batch->batch == 0 || batch->n_tokens == 0) return SB_OK;
  if (!key_out.data || !value_out.data) return SB_ERR_INVALID_ARGUMENT;
  GatherParams P;
  P.cache = *cache, P.batch = *batch;
  P.out[0] = key_out, P.out[1] = value_out;
  P.err = reinterpret_cast<unsigned long long *>(err_counter);
  P.tokens_per_cta = tokens_per_cta(batch->n_tokens);
  const int grid = (batch->n_tokens + P.tokens_per_cta - 1) / P.tokens_per_cta;
  switch (dtype) {
    case SB_DTYPE_F32: return gather_rows<float>(P, grid, st);
    case SB_DTYPE_F16: return gather_rows<__half>(P, grid, st);
    default: return gather_rows<__nv_bfloat16>(P, grid, st);
  }
}
