// Shared by the paged-cache kernels: token -> request -> page addressing and
// the argument checks of their C entry points.
#pragma once

#include <atomic>

#include "common.cuh"

namespace sb {
namespace paged {

__host__ __device__ __forceinline__ int64_t index_at(const void *p, int64_t i, int dtype) {
  return dtype == SB_INDEX_I64 ? reinterpret_cast<const int64_t *>(p)[i]
                               : (int64_t) reinterpret_cast<const int32_t *>(p)[i];
}

// The request of token t: the last b with cu_seqlens[b] <= t (requests without
// tokens are passed over), or -1 for padding.  Any cu_seqlens gives an index
// inside [0, batch).
__host__ __device__ __forceinline__ int find_request(const sb_paged_batch &B, int t) {
  int lo = 0, hi = B.batch;  // cu[lo] <= t < cu[hi] once cu[batch] > t
  if (t >= B.n_tokens || t >= B.cu_seqlens[B.batch]) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (B.cu_seqlens[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// find_request by a whole warp: 32 borders at a time, so that a batch of any
// size takes two or three loads one after the other instead of a dozen.
__device__ __forceinline__ int find_request_warp(const sb_paged_batch &B, int t) {
  if (t >= B.n_tokens || t >= B.cu_seqlens[B.batch]) return -1;
  const int lane = threadIdx.x & 31;
  int lo = 0, n = B.batch;  // the request is one of lo .. lo + n - 1; borders above lo are still to be looked at
  while (n > 1) {
    const int step = (n + 31) / 32, i = lo + lane * step;
    const bool before = lane * step < n && (lane == 0 || B.cu_seqlens[i] <= t);
    const int k = 31 - __clz(__ballot_sync(0xffffffffu, before));
    n = min(step, n - k * step);
    lo += k * step;
  }
  return lo;
}

// Physical block of logical block lb of request b, or -1.
__host__ __device__ __forceinline__ int find_block(const sb_paged_batch &B, int b, int64_t lb, int n_blocks) {
  if (lb < 0 || lb >= B.max_blocks) return -1;
  const int64_t e = index_at(B.block_tables, (int64_t)b * B.table_stride + lb, B.table_dtype);
  return e >= 0 && e < n_blocks ? (int)e : -1;
}

// Positions are handled in 32 bits inside the kernels: anything outside
// int32 addresses no row of a table of 32-bit length times block size, so it is
// brought to -1 (no row, sees nothing) or the largest position.
__host__ __device__ __forceinline__ int load_position(const sb_paged_batch &B, int t) {
  const int64_t p = index_at(B.positions, t, B.pos_dtype);
  return p < 0 ? -1 : p > 0x7fffff00 ? 0x7fffff00 : (int)p;
}

// SMs of the current device, looked up once per device.
inline int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  int n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// log2 of a block size that is a power of two, else -1.
inline int page_shift(int block_size) {
  for (int i = 0; i < 31; ++i)
    if (block_size == 1 << i) return i;
  return -1;
}

inline bool index_ok(int dtype) { return dtype == SB_INDEX_I32 || dtype == SB_INDEX_I64; }

inline int check_batch(const sb_paged_batch *b) {
  if (b == nullptr || b->batch < 0 || b->n_tokens < 0 || b->max_blocks < 0) return SB_ERR_INVALID_ARGUMENT;
  if (b->batch == 0 || b->n_tokens == 0) return SB_OK;
  if (!b->cu_seqlens || !b->positions || !index_ok(b->table_dtype) || !index_ok(b->pos_dtype))
    return SB_ERR_INVALID_ARGUMENT;
  if (b->max_blocks > 0 && (!b->block_tables || (b->batch > 1 && b->table_stride < b->max_blocks)))
    return SB_ERR_INVALID_ARGUMENT;
  return SB_OK;
}

inline bool multiple(const void *p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
inline bool multiple(int64_t v, int n) { return v % n == 0; }

// Geometry and, for 4-bit caches, alignment.
inline int check_cache(const sb_paged_cache *c) {
  if (c == nullptr || c->n_blocks < 0 || c->block_size <= 0 || c->n_heads <= 0 || c->head_dim <= 0)
    return SB_ERR_INVALID_ARGUMENT;
  if (c->n_blocks > 0 && !c->data) return SB_ERR_INVALID_ARGUMENT;
  if (c->group == 0) return elem_bytes(c->dtype) ? SB_OK : SB_ERR_UNSUPPORTED;
  if (c->head_dim != 64 && c->head_dim != 128) return SB_ERR_UNSUPPORTED;
  if ((c->group != 32 && c->group != 64 && c->group != 128) || c->group > c->head_dim) return SB_ERR_UNSUPPORTED;
  if (c->n_blocks > 0 && !c->scales) return SB_ERR_INVALID_ARGUMENT;
  if (!multiple(c->data, 16) || !multiple(c->stride_block, 16) || !multiple(c->stride_kv, 16) ||
      !multiple(c->stride_head, 16) || !multiple(c->stride_pos, 16))
    return SB_ERR_UNSUPPORTED;
  if (!multiple(c->scales, 4) || !multiple(c->scale_block, 2) || !multiple(c->scale_kv, 2) ||
      !multiple(c->scale_head, 2) || !multiple(c->scale_pos, 2))
    return SB_ERR_UNSUPPORTED;
  return SB_OK;
}

// Whether every row of `r` starts at a multiple of `bytes`.
inline bool rows_aligned(const sb_token_rows &r, int es, int bytes) {
  return multiple(r.data, bytes) && multiple(r.stride_token * es, bytes) && multiple(r.stride_head * es, bytes);
}
inline bool cache_aligned(const sb_paged_cache &c, int es, int bytes) {
  return multiple(c.data, bytes) && multiple(c.stride_block * es, bytes) && multiple(c.stride_kv * es, bytes) &&
         multiple(c.stride_head * es, bytes) && multiple(c.stride_pos * es, bytes);
}

}  // namespace paged
}  // namespace sb
