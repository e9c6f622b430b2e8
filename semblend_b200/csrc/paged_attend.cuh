// Shared by the paged-attention kernels: parameters, what a token sees, tiles
// of query rows and their key blocks, and the pieces of the tensor-core paths.
#pragma once

#include "paged.cuh"

namespace sb {
namespace paged {

struct AttendParams {
  sb_paged_cache cache;
  sb_paged_batch batch;
  sb_token_rows q, out;
  int Hq, G;   // query heads, query heads per KV head
  int window;  // 0x7fffffff: none
  int sinks;   // 0 without a window
  float scale;
};

// Keys [0, sink_end) and [first, end) are those a token at position p may see.
struct Span {
  int sink_end, first, end;
};
__host__ __device__ __forceinline__ Span key_span(const AttendParams &P, int p) {
  const int64_t held = (int64_t)P.batch.max_blocks * P.cache.block_size;
  Span s;
  s.end = (int64_t)p + 1 < held ? p + 1 : (int)held;
  s.first = p - P.window + 1;  // at most 0 without a window
  s.first = s.first < 0 ? 0 : s.first > s.end ? s.end : s.first;
  s.sink_end = P.sinks < s.first ? P.sinks : s.first;
  return s;
}

// The query rows of one tile: `n` tokens from `tok` on, and the keys any of
// them may see, in blocks of `KB`: blocks [0, sink_blocks) and then [w0, ...),
// `n_blocks` in all, at least one (a tile that sees nothing still writes zeros).
struct TileKeys {
  Span span;
  int pmin, pmax;
  int sink_blocks, w0, n_blocks;
};
__host__ __device__ __forceinline__ TileKeys tile_keys(const AttendParams &P, int tok, int n, int KB) {
  TileKeys t;
  t.pmin = 0x7fffffff, t.pmax = -1;
  for (int i = 0; i < n; ++i) {
    const int p = load_position(P.batch, tok + i);
    t.pmin = p < t.pmin ? p : t.pmin;
    t.pmax = p > t.pmax ? p : t.pmax;
  }
  const int plow = t.pmin < 0 ? 0 : t.pmin;  // a token at -1 sees nothing and widens nothing
  t.span = key_span(P, t.pmax);
  const int first = key_span(P, plow).first;
  t.span.first = first < t.span.first ? first : t.span.first;
  t.span.sink_end = P.sinks < t.span.first ? P.sinks : t.span.first;
  t.w0 = t.span.first / KB;
  t.sink_blocks = (t.span.sink_end + KB - 1) / KB;
  t.sink_blocks = t.sink_blocks < t.w0 ? t.sink_blocks : t.w0;
  const int last = (int)(((int64_t)t.span.end + KB - 1) / KB);
  t.n_blocks = t.sink_blocks + (last > t.w0 ? last - t.w0 : 0);
  if (t.n_blocks < 1) t.n_blocks = 1;
  return t;
}
__host__ __device__ __forceinline__ int block_key(const TileKeys &t, int i, int KB) {
  return (i < t.sink_blocks ? i : t.w0 + (i - t.sink_blocks)) * KB;
}
__host__ __device__ __forceinline__ bool in_span(const Span &s, int key) {
  return key < s.end && (key >= s.first || key < s.sink_end);
}

// Tokens [lo, hi) of request b, inside [0, n_tokens) whatever cu_seqlens holds.
__host__ __device__ __forceinline__ void request_tokens(const sb_paged_batch &B, int b, int &lo, int &hi) {
  lo = B.cu_seqlens[b], hi = B.cu_seqlens[b + 1];
  lo = lo < 0 ? 0 : lo;
  hi = hi > B.n_tokens ? B.n_tokens : hi;
  const int end = B.cu_seqlens[B.batch];
  hi = hi > end ? end : hi;
  if (hi < lo) hi = lo;
}

// Decode path (csrc/paged_decode.cu): tiles of 8 or 16 query rows, keys split over CTAs.
bool decode_takes(const AttendParams &P, int dtype);
int64_t decode_workspace_bytes(const AttendParams &P);
int launch_decode(const AttendParams &P, int dtype, void *workspace, cudaStream_t st);

}  // namespace paged
}  // namespace sb
