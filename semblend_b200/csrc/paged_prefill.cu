// Paged attention for many query rows per request: prefill chunks and the
// recomputed rows of partial prefills, on tcgen05 tensor cores (sm_100a).
//
// A tile is the G query heads of a KV group at 128 / G tokens (up to 128 rows),
// two consecutive tiles of a request form a unit, and the unit's keys go by in
// blocks of 128: first the blocks of the sinks, then those from the first
// token's window to the last token.  Products, softmax and the order of the
// barriers are those of the dense partial-prefill kernel (attention.cu): S =
// Q K^T into TMEM, one softmax thread per row, P written back over S, O += P V
// in TMEM, two tiles in ping-pong.  What differs is where K and V come from
// and what a row sees:
//
//   16-bit rows   TMA boxes of one page (or 128 rows of a larger one) and 64
//                 columns, issued by the lanes of the producer warp, which look
//                 the page numbers up one block ahead; pages that no row of
//                 the unit sees are loaded from behind the pool, as zeros
//   4-bit codes   seven loader warps read the codes, expand them in registers
//                 to fp16 and store them in the layout a 128-byte-swizzled TMA
//                 load would have left; products then run in fp16, queries
//                 scaled by a power of two per row.  Element pairs (d, d + 4) of
//                 each eight stay side by side, as the masks leave them: the
//                 queries and the result's columns are ordered to match
//
// A key that a row does not see has its score replaced, and its V row is zeroed
// in shared memory where no row of the unit sees it (the rest of a last page
// may hold anything).  Where another row of the unit does see it and it holds
// an infinity or a NaN, the product with a probability of zero is a NaN: rows
// that come out infinite or NaN are computed again over their own keys alone.
// So are units with an unmapped page inside their keys.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <type_traits>

#include "paged_attend.cuh"
#include "prof.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace sb {
namespace paged {
namespace {

constexpr int kBM = 128, kBN = 128;
constexpr int kSoftmaxRegs = 200;
// About ten seconds: a role may wait while rows of the last unit are computed one by one.
constexpr long long kWaitCycles = 20000000000LL;

template <int D, bool CODES> struct Shape {
  static constexpr int kHalves = D / 64;                // 64-column halves of an operand tile
  static constexpr int kHalf = 128 * 128;               // bytes of one half: 128 rows of 128 bytes
  static constexpr int kTile = kHalves * kHalf;
  static constexpr int kStages = D == 128 ? 2 : 4;      // K and V rings
  // warps 0-3 and 4-7: softmax of tile 0 and 1; 8: units and (16-bit) loads; 9: MMA; 10: zeroes V rows;
  // 4-bit: 8 and 10-15 load
  static constexpr int kThreads = CODES ? 512 : 384;
  // the launch's registers a thread (65536 / threads, in eights) less what the softmax warps take
  static constexpr int kControlRegs = CODES ? 56 : 104;
  static_assert(2 * 128 * kSoftmaxRegs + (kThreads - 256) * kControlRegs == kThreads * (CODES ? 128 : 168),
                "register split");
  static constexpr int kLoaders = CODES ? 7 : 1;        // warps that fill K and V
  static constexpr int kBars = 1024;
  static constexpr int kSmem = 1024 + kTile * (2 + 2 * kStages) + kBars;
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

__host__ __device__ constexpr uint32_t tmem_s(int t) { return 256u * t; }
__host__ __device__ constexpr uint32_t tmem_o(int t) { return 256u * t + 128u; }

struct PrefillParams {
  AttendParams a;
  int Pt;            // tokens of a tile
  int slots;         // unit slots of a KV head: n_tokens / (2 Pt) + batch
  int64_t n_units;
  int pages, page_rows;  // pages of a block of 128 keys and the rows a box takes of one
  int dtype;
  unsigned *next;    // workspace, zeroed ahead of the launch
  int *status;
};

// One unit as its roles see it.
struct Unit {
  int b, g, tok, n0, n1;    // request, KV head, first token, tokens of the two tiles
  int nblk0, nblk1;         // blocks each tile goes through
  int sink_blocks, w0;
  int first, end, sink_end; // keys some row sees
  int plain;                // 1: an unmapped page among them, every row is computed on its own
  int stop;                 // 1: no more units
};
constexpr int kUnitInts = sizeof(Unit) / 4;

__device__ __forceinline__ int unit_block_key(const Unit &u, int i) {
  return (i < u.sink_blocks ? i : u.w0 + (i - u.sink_blocks)) * kBN;
}
// Blocks with keys that no row of the unit sees.
__device__ __forceinline__ bool unit_edge(const Unit &u, int key0) {
  return key0 + kBN > u.end || (key0 < u.first && key0 + kBN > u.sink_end);
}

template <typename T> struct Pack2;
template <> struct Pack2<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t *>(&v);
  }
};
template <> struct Pack2<__half> {
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t *>(&v);
  }
};
__device__ __forceinline__ float2 unpack_any(uint32_t x, int dtype) {
  if (dtype == SB_DTYPE_BF16) return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  return __half22float2(*reinterpret_cast<__half2 *>(&x));
}
__device__ __forceinline__ uint32_t pack_any(float a, float b, int dtype) {
  return dtype == SB_DTYPE_BF16 ? Pack2<__nv_bfloat16>::pack(a, b) : Pack2<__half>::pack(a, b);
}

// The next unit of this CTA, found by a whole warp (lanes share the scans).
__device__ __forceinline__ bool make_unit(const PrefillParams &P, int64_t u, Unit &w) {
  const AttendParams &A = P.a;
  const int lane = threadIdx.x & 31, two = 2 * P.Pt, Hkv = A.cache.n_heads;
  // later tokens, which see most without a window, first; the KV heads of a slot side by side
  const int slot = P.slots - 1 - (int)(u / Hkv);
  w.g = (int)(u % Hkv);
  // request b owns the slots from cu[b] / two + b on: enough for its tokens, whatever its neighbours have
  int lo = 0, hi = A.batch.batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (max(A.batch.cu_seqlens[mid], 0) / two + mid <= slot) lo = mid;
    else hi = mid;
  }
  w.b = lo;
  int tlo, thi;
  request_tokens(A.batch, w.b, tlo, thi);
  const int64_t tok = tlo + (int64_t)(slot - (max(A.batch.cu_seqlens[w.b], 0) / two + w.b)) * two;
  if (tok < tlo || tok >= thi) return false;
  w.tok = (int)tok;
  w.n0 = min(P.Pt, thi - w.tok);
  w.n1 = max(0, min(P.Pt, thi - w.tok - P.Pt));
  int pmin = 0x7fffffff, pmax0 = -1, pmax1 = -1;
  for (int i = lane; i < w.n0 + w.n1; i += 32) {
    const int p = load_position(A.batch, w.tok + i);
    if (p >= 0) pmin = min(pmin, p);
    if (i < w.n0) pmax0 = max(pmax0, p);
    else pmax1 = max(pmax1, p);
  }
  for (int o = 16; o > 0; o >>= 1) {
    pmin = min(pmin, __shfl_xor_sync(0xffffffffu, pmin, o));
    pmax0 = max(pmax0, __shfl_xor_sync(0xffffffffu, pmax0, o));
    pmax1 = max(pmax1, __shfl_xor_sync(0xffffffffu, pmax1, o));
  }
  const int e0 = key_span(A, pmax0).end, e1 = key_span(A, pmax1).end;
  w.end = max(e0, e1);
  w.first = pmin == 0x7fffffff ? 0 : min(key_span(A, pmin).first, w.end);
  w.sink_end = min(A.sinks, w.first);
  w.w0 = w.first / kBN;
  w.sink_blocks = min((w.sink_end + kBN - 1) / kBN, w.w0);
  // every tile goes through the blocks from the unit's first on; one that sees nothing through one block
  w.nblk0 = max(1, w.sink_blocks + max(0, (int)(((int64_t)e0 + kBN - 1) / kBN) - w.w0));
  w.nblk1 = w.n1 > 0 ? max(1, w.sink_blocks + max(0, (int)(((int64_t)e1 + kBN - 1) / kBN) - w.w0)) : 0;
  w.stop = 0;
  // pages the unit's keys lie in
  const int bs = A.cache.block_size;
  bool bad = false;
  for (int part = 0; part < 2; ++part) {
    const int k0 = part == 0 ? 0 : w.first, k1 = part == 0 ? w.sink_end : w.end;
    if (k1 <= k0) continue;
    const int p1 = (k1 - 1) / bs;
    for (int p = k0 / bs + lane; p <= p1; p += 32) bad |= find_block(A.batch, w.b, p, A.cache.n_blocks) < 0;
  }
  w.plain = __any_sync(0xffffffffu, bad);
  return true;
}

template <typename T, int D, bool CODES>
__global__ void __launch_bounds__(Shape<D, CODES>::kThreads, 1)
    prefill_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const PrefillParams P) {
  using S = Shape<D, CODES>;
  constexpr int kStages = S::kStages, kTile = S::kTile, kHalf = S::kHalf, kHalves = S::kHalves;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sQ = smem;
  uint8_t *sK = sQ + 2 * kTile;
  uint8_t *sV = sK + kStages * kTile;
  uint64_t *bars = reinterpret_cast<uint64_t *>(sV + kStages * kTile);
  uint64_t *k_full = bars, *k_empty = bars + 4, *v_full = bars + 8, *v_empty = bars + 12;
  uint64_t *q_full = bars + 16;     // [2]
  uint64_t *q_empty = bars + 18;
  uint64_t *s_full = bars + 19;     // [2]
  uint64_t *p_full = bars + 21;     // [2 tiles][2 key halves]
  uint64_t *o_final = bars + 25;    // [2]
  uint64_t *final_bar = bars + 27;
  uint64_t *unit_full = bars + 28;  // [2]
  uint64_t *unit_empty = bars + 30; // [2]
  uint64_t *v_clean = bars + 32;    // [kStages]
  uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(bars + 36);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(bars + 37);
  volatile int *unit_ring = reinterpret_cast<volatile int *>(bars + 38);  // [2][kUnitInts]
  static_assert(38 * 8 + 2 * sizeof(Unit) <= S::kBars, "barrier area");
  const AttendParams &A = P.a;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      tc::mbar_init(&k_full[s], S::kLoaders);
      tc::mbar_init(&v_full[s], S::kLoaders);
      tc::mbar_init(&k_empty[s], 1);
      tc::mbar_init(&v_empty[s], 1);
      tc::mbar_init(&v_clean[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      tc::mbar_init(&q_full[t], 4);
      tc::mbar_init(&s_full[t], 1);
      tc::mbar_init(&p_full[2 * t], 4);
      tc::mbar_init(&p_full[2 * t + 1], 4);
      tc::mbar_init(&o_final[t], 1);
    }
    tc::mbar_init(q_empty, 1);
    tc::mbar_init(final_bar, 1);
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&unit_full[i], 1);
      // MMA thread, 8 softmax warps, and warp 10 (V rows) or the six other loader warps
      tc::mbar_init(&unit_empty[i], 1 + 8 + (CODES ? S::kLoaders - 1 : 1));
    }
    *abort_flag = 0;
    tc::fence_mbar_init();
  }
  if (warp == 9) {
    tc::tmem_alloc(tmem_holder, 512);
    tc::tmem_relinquish();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_holder;
  const tc::Abort ab{abort_flag, P.status};
  volatile int never = 0;
  const tc::Abort drain{&never, nullptr};

  // The n-th unit of this CTA.  A whole warp reads the slot before lane 0 releases it; the MMA thread is alone.
  auto pop_unit = [&](uint32_t n, bool whole_warp, Unit &w) -> bool {
    if (!tc::mbar_wait(&unit_full[n & 1], (n >> 1) & 1, ab, 5, kWaitCycles)) return false;
    int *to = reinterpret_cast<int *>(&w);
#pragma unroll
    for (int i = 0; i < kUnitInts; ++i) to[i] = unit_ring[(n & 1) * kUnitInts + i];
    if (whole_warp) __syncwarp();
    if (!whole_warp || lane == 0) tc::mbar_arrive(&unit_empty[n & 1]);
    return !w.stop;
  };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kControlRegs));
    if (warp == 9) {
      if (lane == 0) {
        // ------------------------------ MMA issuer ------------------------------
        constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
        constexpr uint32_t idesc_qk = tc::idesc_f16(kBM, kBN, fmt, 0);
        constexpr uint32_t idesc_pv = tc::idesc_f16(kBM, D, fmt, 1);
        uint32_t gl = 0, qi = 0;
        uint32_t pc[2] = {0, 0};
        bool ok = true;
        const uint64_t dq0 = tc::desc_kmajor_sw128(sQ);
        const uint64_t dk0 = tc::desc_kmajor_sw128(sK);
        const uint64_t dv0 = tc::desc_mnmajor_sw128(sV, 0, kHalf);
        constexpr uint32_t kTileUnits = kTile >> 4, kHalfUnits = kHalf >> 4;
        auto issue_s = [&](int t, uint32_t st) {
          const uint64_t dq = dq0 + t * kTileUnits, dk = dk0 + st * kTileUnits;
#pragma unroll
          for (int kb = 0; kb < kHalves; ++kb)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              tc::mma_bf16_ss(tmem + tmem_s(t), dq + kb * kHalfUnits + kk * 2, dk + kb * kHalfUnits + kk * 2, idesc_qk,
                              (kb | kk) != 0);
          tc::mma_commit(&s_full[t]);
        };
        Unit w;
        for (uint32_t n = 0; ok; ++n) {
          if (!pop_unit(n, false, w)) break;
          if (w.plain) continue;
          const int nb = max(w.nblk0, w.nblk1);
          if (!tc::mbar_wait(&q_full[0], qi & 1, ab, 3, kWaitCycles) ||
              !tc::mbar_wait(&q_full[1], qi & 1, ab, 3, kWaitCycles))
            break;
          tc::fence_after_sync();
          {
            const uint32_t ks = gl % kStages;
            if (!tc::mbar_wait(&k_full[ks], (gl / kStages) & 1, ab, 3, kWaitCycles)) break;
            tc::fence_after_sync();
            issue_s(0, ks);
            if (w.nblk1 > 0) issue_s(1, ks);
            tc::mma_commit(&k_empty[ks]);
          }
          for (int j = 0; j < nb && ok; ++j) {
            const uint32_t g = gl + j;
            const uint32_t vs = g % kStages, vph = (g / kStages) & 1;
            const uint32_t ks1 = (g + 1) % kStages, kph1 = ((g + 1) / kStages) & 1;
            bool v_ready = false, k_ready = false;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const int nt = t == 0 ? w.nblk0 : w.nblk1;
              if (!ok || j >= nt) continue;
              // P.V in two halves of 64 keys: the first runs while the softmax writes the second
              if (!tc::mbar_wait(&p_full[2 * t], pc[t] & 1, ab, 3, kWaitCycles)) {
                ok = false;
                continue;
              }
              if (!v_ready) {
                if (!tc::mbar_wait(&v_full[vs], vph, ab, 3, kWaitCycles) ||
                    (!CODES && !tc::mbar_wait(&v_clean[vs], vph, ab, 3, kWaitCycles))) {
                  ok = false;
                  continue;
                }
                v_ready = true;
              }
              tc::fence_after_sync();
              const uint32_t p_tmem = tmem + tmem_s(t);
              const uint64_t dv = dv0 + vs * kTileUnits;
#pragma unroll
              for (int kk = 0; kk < kBN / 32; ++kk)
                tc::mma_bf16_ts(tmem + tmem_o(t), p_tmem + kk * 8, dv + kk * (2048 >> 4), idesc_pv,
                                (j == 0 && kk == 0) ? 0u : 1u);
              if (!tc::mbar_wait(&p_full[2 * t + 1], pc[t] & 1, ab, 3, kWaitCycles)) {
                ok = false;
                continue;
              }
              ++pc[t];
              tc::fence_after_sync();
#pragma unroll
              for (int kk = kBN / 32; kk < kBN / 16; ++kk)
                tc::mma_bf16_ts(tmem + tmem_o(t), p_tmem + kk * 8, dv + kk * (2048 >> 4), idesc_pv, 1u);
              if (j == nt - 1) tc::mma_commit(&o_final[t]);
              if (j + 1 < nt) {
                if (!k_ready) {
                  if (!tc::mbar_wait(&k_full[ks1], kph1, ab, 3, kWaitCycles)) {
                    ok = false;
                    continue;
                  }
                  tc::fence_after_sync();
                  k_ready = true;
                }
                issue_s(t, ks1);
              }
            }
            if (!ok) break;
            tc::mma_commit(&v_empty[vs]);
            if (j + 1 < nb) tc::mma_commit(&k_empty[ks1]);
          }
          if (!ok) break;
          gl += nb;
          tc::mma_commit(q_empty);
          ++qi;
        }
        tc::mma_commit(final_bar);
        tc::mbar_wait(final_bar, 0, drain, 0, kWaitCycles);
      }
    } else if (warp == 8 || CODES) {
      // ------------------------------ units, K and V ------------------------------
      const bool leader = warp == 8;
      uint32_t gl = 0, pushed = 0;
      bool ok = true, vfail = false;
      if (!CODES && lane == 0) {
        tc::tma_prefetch_desc(&tmK);
        tc::tma_prefetch_desc(&tmV);
      }
      auto push_unit = [&](const Unit &w) -> bool {
        const uint32_t slot = pushed & 1, use = pushed >> 1;
        if (use > 0 && !tc::mbar_wait(&unit_empty[slot], (use - 1) & 1, ab, 2, kWaitCycles)) return false;
        const int *from = reinterpret_cast<const int *>(&w);
        if (lane == 0) {
#pragma unroll
          for (int i = 0; i < kUnitInts; ++i) unit_ring[slot * kUnitInts + i] = from[i];
          tc::mbar_arrive(&unit_full[slot]);
        }
        __syncwarp();
        ++pushed;
        return true;
      };
      Unit w;
      for (uint32_t n = 0; ok;) {
        if (leader) {
          unsigned u = 0;
          if (lane == 0) u = atomicAdd(P.next, 1u);
          u = __shfl_sync(0xffffffffu, u, 0);
          if (u >= P.n_units) {
            w.stop = 1;
            push_unit(w);
            break;
          }
          if (!make_unit(P, u, w)) continue;
          if (!push_unit(w)) {
            ok = false;
            break;
          }
        } else {
          if (!pop_unit(n, true, w)) break;
          ++n;
        }
        if (w.plain) continue;
        const int nb = max(w.nblk0, w.nblk1);
        const int bs = A.cache.block_size;
        if constexpr (!CODES) {
          // lane -> box: page lane / halves of the block, 64-column half lane % halves
          const int page = lane / kHalves, half = lane % kHalves;
          const bool mine = page < P.pages;
          auto page_at = [&](int i, int &row) -> int {
            const int key = unit_block_key(w, i) + page * P.page_rows;
            const int lb = key / bs;
            row = key - lb * bs;
            // pages without a key that some row sees come from behind the pool, as zeros
            const bool any = key < w.end && (key + P.page_rows > w.first || key < w.sink_end);
            const int phys = any ? find_block(A.batch, w.b, lb, A.cache.n_blocks) : -1;
            return phys < 0 ? A.cache.n_blocks : phys;
          };
          int row = 0, blk = mine ? page_at(0, row) : 0;
          for (int j = 0; j < nb && ok; ++j) {
            const uint32_t st = gl % kStages, ph = (gl / kStages) & 1;
            int row1 = 0, blk1 = 0;
            if (mine && j + 1 < nb) blk1 = page_at(j + 1, row1);
            if (!tc::mbar_wait(&k_empty[st], ph ^ 1, ab, 2, kWaitCycles)) ok = false;
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const uint32_t to = st * kTile + half * kHalf + page * P.page_rows * 128;
            if (lane == 0) tc::mbar_arrive_expect_tx(&k_full[st], kTile);
            __syncwarp();
            if (mine) tc::tma_load_4d(sK + to, &tmK, &k_full[st], half * 64, row, w.g, blk);
            ++gl;
            if (!tc::mbar_wait(&v_empty[st], ph ^ 1, ab, 2, kWaitCycles)) ok = false;
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) {
              vfail = true;
              break;
            }
            if (lane == 0) tc::mbar_arrive_expect_tx(&v_full[st], kTile);
            __syncwarp();
            if (mine) tc::tma_load_4d(sV + to, &tmV, &v_full[st], half * 64, row, w.g, blk);
            row = row1, blk = blk1;
          }
        } else {
          // Rows of kLanes threads, 32 codes (16 bytes) each; this warp takes groups of rows
          // loader, loader + 7, ... of a block.  The next block's codes are on their way to registers
          // while this one waits for its slot.
          constexpr int kLanes = D / 32, kRows = 32 / kLanes, kGroups = kBN / kRows;
          constexpr int kMine = (kGroups + S::kLoaders - 1) / S::kLoaders;
          const int loader = leader ? 0 : warp - 9, chunk = lane % kLanes;
          const char *cbase = reinterpret_cast<const char *>(A.cache.data) + (int64_t)w.g * A.cache.stride_head + 16 * chunk;
          const char *sbase = reinterpret_cast<const char *>(A.cache.scales) + 2 * (int64_t)w.g * A.cache.scale_head +
                              4 * (32 * chunk / A.cache.group);
          uint4 code[2][kMine];
          uint32_t scale[2][kMine];  // (step, zero); both 0 where no row of the unit sees the key
          auto fetch = [&](int i, int kv) {
#pragma unroll
            for (int x = 0; x < kMine; ++x) {
              const int key = unit_block_key(w, i) + (loader + x * S::kLoaders) * kRows + lane / kLanes;
              code[kv][x] = make_uint4(0, 0, 0, 0);
              scale[kv][x] = 0u;
              int64_t row, srow;
              if (loader + x * S::kLoaders < kGroups && key < w.end && (key >= w.first || key < w.sink_end) &&
                  key_row(A, w.b, key, row, srow)) {
                code[kv][x] = *reinterpret_cast<const uint4 *>(cbase + row + kv * A.cache.stride_kv);
                scale[kv][x] = *reinterpret_cast<const uint32_t *>(sbase + 2 * (srow + kv * A.cache.scale_kv));
              }
            }
          };
          auto store = [&](uint8_t *tile, int kv) {
#pragma unroll
            for (int x = 0; x < kMine; ++x) {
              if (loader + x * S::kLoaders >= kGroups) continue;
              const int row = (loader + x * S::kLoaders) * kRows + lane / kLanes;
              const __half2 sz = *reinterpret_cast<const __half2 *>(&scale[kv][x]);
              const __half2 step = __low2half2(sz), zero = __high2half2(sz);
              const uint32_t word[4] = {code[kv][x].x, code[kv][x].y, code[kv][x].z, code[kv][x].w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                // 0x6400 | c is 1024 + c in fp16, 0x6400 | 16 c is 1024 + 16 c; both back to c exactly
                uint32_t out[4];
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                  const uint32_t b = (((y < 2 ? word[i] : word[i] >> 8) & (y & 1 ? 0x00F000F0u : 0x000F000Fu)) | 0x64006400u);
                  const __half2 raw = *reinterpret_cast<const __half2 *>(&b);
                  const __half2 c = y & 1 ? __hfma2(raw, __float2half2_rn(0.0625f), __float2half2_rn(-64.f))
                                          : __hsub2(raw, __float2half2_rn(1024.f));
                  const __half2 v = __hfma2(c, step, zero);
                  out[y] = *reinterpret_cast<const uint32_t *>(&v);
                }
                const int at = 4 * chunk + i;  // eight elements: one 16-byte piece of the row
                *reinterpret_cast<uint4 *>(tile + (at / 8) * kHalf + row * 128 + (((at % 8) ^ (row & 7)) << 4)) =
                    make_uint4(out[0], out[1], out[2], out[3]);
              }
            }
            tc::fence_proxy_async_smem();
            __syncwarp();
          };
          fetch(0, 0);
          fetch(0, 1);
          for (int j = 0; j < nb && ok; ++j) {
            const uint32_t st = gl % kStages, ph = (gl / kStages) & 1;
            ok = __all_sync(0xffffffffu, tc::mbar_wait(&k_empty[st], ph ^ 1, ab, 2, kWaitCycles));
            if (!ok) break;
            store(sK + st * kTile, 0);
            if (lane == 0) tc::mbar_arrive(&k_full[st]);
            if (j + 1 < nb) fetch(j + 1, 0);
            ok = __all_sync(0xffffffffu, tc::mbar_wait(&v_empty[st], ph ^ 1, ab, 2, kWaitCycles));
            if (!ok) break;
            store(sV + st * kTile, 1);
            if (lane == 0) tc::mbar_arrive(&v_full[st]);
            if (j + 1 < nb) fetch(j + 1, 1);
            ++gl;
          }
        }
      }
      if (!CODES && lane == 0) {
        // every load this warp issued lands before the CTA can exit (the V load of the last counted
        // block is missing when its slot wait gave up)
        const uint32_t nk = gl < (uint32_t)kStages ? gl : (uint32_t)kStages;
        for (uint32_t i = gl - nk; i < gl; ++i)
          tc::mbar_wait(&k_full[i % kStages], (i / kStages) & 1, drain, 0, kWaitCycles);
        const uint32_t gv = vfail ? gl - 1 : gl;
        const uint32_t nv = gv < (uint32_t)kStages ? gv : (uint32_t)kStages;
        for (uint32_t i = gv - nv; i < gv; ++i)
          tc::mbar_wait(&v_full[i % kStages], (i / kStages) & 1, drain, 0, kWaitCycles);
      }
    } else if (warp == 10) {
      // ------------------------------ V rows that no row of the unit sees ------------------------------
      uint32_t gl = 0;
      bool ok = true;
      Unit w;
      for (uint32_t n = 0; ok; ++n) {
        if (!pop_unit(n, true, w)) break;
        if (w.plain) continue;
        const int nb = max(w.nblk0, w.nblk1);
        for (int j = 0; j < nb; ++j, ++gl) {
          const int key0 = unit_block_key(w, j);
          const uint32_t st = gl % kStages;
          if (!tc::mbar_wait(&v_full[st], (gl / kStages) & 1, ab, 6, kWaitCycles)) {
            ok = false;
            break;
          }
          if (!unit_edge(w, key0)) {
            if (lane == 0) tc::mbar_arrive(&v_clean[st]);
            continue;
          }
          for (int i = lane; i < 128 * 8 * kHalves; i += 32) {
            const int row = (i / 8) % 128, key = key0 + row;
            if (key < w.end && (key >= w.first || key < w.sink_end)) continue;
            *reinterpret_cast<uint4 *>(sV + st * kTile + (i / 1024) * kHalf + row * 128 + (i % 8) * 16) =
                make_uint4(0, 0, 0, 0);
          }
          tc::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&v_clean[st]);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ------------------------------ softmax / epilogue ------------------------------
    const int t = warp >> 2, quarter = warp & 3;
    const int m = quarter * 32 + lane;  // tile row == TMEM lane
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
    const int hh = m / P.Pt, pi = m - hh * P.Pt;
    uint32_t sc = 0, oc = 0, qi = 0;
    bool ok = true;
    const bool neg_scale = A.scale < 0.f;
    Unit w;
    for (uint32_t n = 0; ok; ++n) {
      if (!pop_unit(n, true, w)) break;
      const int ntok = t == 0 ? w.n0 : w.n1;
      const bool valid = hh < A.G && pi < ntok;
      const int tok = w.tok + t * P.Pt + pi, head = w.g * A.G + hh;
      const int pos = valid ? load_position(A.batch, tok) : -1;
      const char *qrow = reinterpret_cast<const char *>(A.q.data) +
                         2 * (valid ? (int64_t)tok * A.q.stride_token + (int64_t)head * A.q.stride_head : 0);
      char *orow = reinterpret_cast<char *>(A.out.data) +
                   2 * (valid ? (int64_t)tok * A.out.stride_token + (int64_t)head * A.out.stride_head : 0);
      bool redo = w.plain && valid;
      if (!w.plain) {
        // gather this row of Q into the 128-byte-swizzled K-major tile (zeros for unused rows)
        if (qi > 0 && !tc::mbar_wait(q_empty, (qi - 1) & 1, ab, 4, kWaitCycles)) break;
        float scale_log2 = A.scale * 1.4426950408889634f;
        {
          uint8_t *q_tile = sQ + t * kTile;
          const uint4 *src = reinterpret_cast<const uint4 *>(qrow);
          uint4 v[D / 8];
#pragma unroll
          for (int c = 0; c < D / 8; ++c) v[c] = valid ? src[c] : make_uint4(0, 0, 0, 0);
          if constexpr (CODES) {
            // to fp16 with a largest magnitude in [2^11, 2^12): a power of two, undone in the scale
            float big = 0.f;
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
              const uint32_t x[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float2 f = unpack_any(x[i], P.dtype);
                big = fmaxf(big, fmaxf(fabsf(f.x), fabsf(f.y)));
              }
            }
            int e = (int)((__float_as_uint(big) >> 23) & 255) - 127;
            e = big > 0.f ? min(max(e, -110), 110) : 0;
            const float norm = __uint_as_float((uint32_t)(11 - e + 127) << 23);
            scale_log2 *= __uint_as_float((uint32_t)(e - 11 + 127) << 23);
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
              const float2 a = unpack_any(v[c].x, P.dtype), b = unpack_any(v[c].y, P.dtype);
              const float2 d = unpack_any(v[c].z, P.dtype), f = unpack_any(v[c].w, P.dtype);
              v[c].x = Pack2<T>::pack(a.x * norm, d.x * norm);  // elements (0, 4), (1, 5), (2, 6), (3, 7)
              v[c].y = Pack2<T>::pack(a.y * norm, d.y * norm);
              v[c].z = Pack2<T>::pack(b.x * norm, f.x * norm);
              v[c].w = Pack2<T>::pack(b.y * norm, f.y * norm);
            }
          }
#pragma unroll
          for (int c = 0; c < D / 8; ++c) {
            const int kb = c >> 3, cc = c & 7;
            *reinterpret_cast<uint4 *>(q_tile + kb * kHalf + m * 128 + ((cc ^ (m & 7)) << 4)) = v[c];
          }
        }
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&q_full[t]);
        ++qi;
        const int nb = t == 0 ? w.nblk0 : w.nblk1;
        float m_used = -INFINITY, l = 0.f;
        const uint32_t s_addr = tmem + lane_addr + tmem_s(t);
        for (int j = 0; j < nb; ++j) {
          if (!tc::mbar_wait(&s_full[t], sc & 1, ab, 4, kWaitCycles)) {
            ok = false;
            break;
          }
          ++sc;
          tc::fence_after_sync();
          const int key0 = unit_block_key(w, j);
          // this row does not see the whole block (unused rows, with a zero query, are never stored)
          const bool edge = valid && !(key0 + kBN - 1 <= pos && (key0 > pos - A.window || key0 + kBN <= A.sinks));
          const float masked = neg_scale ? INFINITY : -INFINITY;
          uint32_t sr[kBN];
#pragma unroll
          for (int c = 0; c < 4; ++c) tc::tmem_ld32(s_addr + c * 32, *reinterpret_cast<uint32_t(*)[32]>(sr + c * 32));
          tc::tmem_ld_wait();
          if (__any_sync(0xffffffffu, edge)) {
            const int hi = edge ? pos - key0 : kBN;                // columns above are later keys
            const int lo = edge ? max(pos - A.window, -1) - key0 : -1;  // columns up to it have left the window ...
            const int sk = A.sinks - key0;                         // ... unless they are sinks
#pragma unroll
            for (int c = 0; c < kBN; ++c)
              if (c > hi || (c <= lo && c >= sk)) sr[c] = __float_as_uint(masked);
          }
          float mx;
          {
            float a0 = masked, a1 = masked, a2 = masked, a3 = masked;
#pragma unroll
            for (int c = 0; c < kBN; c += 8) {
#define SB_X(i) __uint_as_float(sr[c + (i)])
              if (!neg_scale) {
                a0 = tc::max3(a0, SB_X(0), SB_X(1)), a1 = tc::max3(a1, SB_X(2), SB_X(3));
                a2 = tc::max3(a2, SB_X(4), SB_X(5)), a3 = tc::max3(a3, SB_X(6), SB_X(7));
              } else {
                a0 = tc::min3(a0, SB_X(0), SB_X(1)), a1 = tc::min3(a1, SB_X(2), SB_X(3));
                a2 = tc::min3(a2, SB_X(4), SB_X(5)), a3 = tc::min3(a3, SB_X(6), SB_X(7));
              }
#undef SB_X
            }
            mx = neg_scale ? fminf(fminf(a0, a1), fminf(a2, a3)) : fmaxf(fmaxf(a0, a1), fmaxf(a2, a3));
          }
          const float mx_s = mx * scale_log2;
          float m_new = m_used;
          bool need = false;
          if (mx_s > -INFINITY && (m_used == -INFINITY || mx_s > m_used + 8.f)) {
            need = m_used != -INFINITY;
            m_new = mx_s;
          }
          if (__any_sync(0xffffffffu, need)) {
            // O_t holds the blocks before this one (this S block's barrier says so): rescale it in TMEM
            const float alpha = need ? tc::ex2_approx(m_used - m_new) : 1.f;
            const uint32_t o_addr = tmem + lane_addr + tmem_o(t);
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t x[32];
              tc::tmem_ld32(o_addr + c, x);
              tc::tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * alpha);
              tc::tmem_st16(o_addr + c, *reinterpret_cast<const uint32_t(*)[16]>(x));
              tc::tmem_st16(o_addr + c + 16, *reinterpret_cast<const uint32_t(*)[16]>(x + 16));
            }
            tc::tmem_st_wait();
            l *= alpha;
          }
          m_used = m_new;
          const float neg_m = m_used != -INFINITY ? -m_used : -INFINITY;
          const float2 cc = make_float2(scale_log2, scale_log2), nm = make_float2(neg_m, neg_m);
          float2 sum2 = make_float2(0.f, 0.f);
#pragma unroll
          for (int c = 0; c < kBN; c += 32) {
            uint32_t x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 e = tc::fma2(make_float2(__uint_as_float(sr[c + 2 * i]), __uint_as_float(sr[c + 2 * i + 1])),
                                        cc, nm);
              const float2 pp = make_float2(tc::ex2_approx(e.x), tc::ex2_approx(e.y));
              sum2 = tc::add2(sum2, pp);
              x[i] = Pack2<T>::pack(pp.x, pp.y);
            }
            tc::tmem_st16(s_addr + c / 2, x);
            if (c % 64 == 32) {  // 64 keys of P are in TMEM: their P.V may start
              tc::tmem_st_wait();
              tc::fence_before_sync();
              __syncwarp();
              if (lane == 0) tc::mbar_arrive(&p_full[2 * t + c / 64]);
            }
          }
          l += sum2.x + sum2.y;
        }
        if (!ok) break;
        if (nb == 0) continue;
        if (!tc::mbar_wait(&o_final[t], oc & 1, ab, 4, kWaitCycles)) break;
        ++oc;
        tc::fence_after_sync();
        // l is 0 only where no key is seen (a NaN score makes it NaN)
        const float inv = l == 0.f ? 0.f : 1.f / l;
        bool odd = !isfinite(l);
        uint4 *dst = reinterpret_cast<uint4 *>(orow);
        const uint32_t o_addr = tmem + lane_addr + tmem_o(t);
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t x[32];
          tc::tmem_ld32(o_addr + c, x);
          tc::tmem_ld_wait();
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; ++i) odd |= !isfinite(__uint_as_float(x[i]));
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            // 4-bit: columns 8 k + (0, 1, 2, 3, ...) hold elements 8 k + (0, 4, 1, 5, 2, 6, 3, 7)
            const int k = i / 4 * 8, y = i % 4;
            const int p = CODES ? k + (y < 2 ? 4 * y : 4 * (y - 2) + 1) : 2 * i, q = CODES ? p + 2 : p + 1;
            pk[i] = pack_any(__uint_as_float(x[p]) * inv, __uint_as_float(x[q]) * inv, P.dtype);
          }
          if (valid) {
#pragma unroll
            for (int i = 0; i < 4; ++i) dst[c / 8 + i] = make_uint4(pk[4 * i], pk[4 * i + 1], pk[4 * i + 2], pk[4 * i + 3]);
          }
        }
        redo = valid && odd;
        tc::fence_before_sync();
      }
      // rows to compute on their own, one after the other by the whole warp
      uint32_t todo = __ballot_sync(0xffffffffu, redo);
      __syncwarp();
      while (todo) {
        const int who = __ffs(todo) - 1;
        todo &= todo - 1;
        const int p = __shfl_sync(0xffffffffu, pos, who);
        const char *q = reinterpret_cast<const char *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(qrow), who));
        char *o = reinterpret_cast<char *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(orow), who));
        attend_row<D>(A, P.dtype, w.b, w.g, p, q, o);
      }
    }
  }

  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (warp == 9) tc::tmem_dealloc(tmem, 512);
}

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
  return n > 0 ? n : 148;
}

PrefillParams plan(const AttendParams &A) {
  PrefillParams P;
  P.a = A;
  P.Pt = kBM / A.G;
  P.slots = A.batch.n_tokens / (2 * P.Pt) + A.batch.batch;
  P.n_units = (int64_t)P.slots * A.cache.n_heads;
  P.page_rows = std::min(A.cache.block_size, kBN);
  P.pages = kBN / P.page_rows;
  return P;
}

template <typename T, int D, bool CODES>
int run(PrefillParams &P, int32_t *status, void *workspace, cudaStream_t st) {
  using S = Shape<D, CODES>;
  CUtensorMap tk, tv;
  memset(&tk, 0, sizeof(tk)), memset(&tv, 0, sizeof(tv));
  if (!CODES) {
    const sb_paged_cache &c = P.a.cache;
    const CUtensorMapDataType dt =
        std::is_same<T, __nv_bfloat16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    // a dimension of one element may carry any stride: give it one a map accepts
    const uint64_t sp = c.block_size > 1 ? 2 * (uint64_t)c.stride_pos : 2 * D;
    const uint64_t sh = c.n_heads > 1 ? 2 * (uint64_t)c.stride_head : 2 * D;
    const uint64_t sb = c.n_blocks > 1 ? 2 * (uint64_t)c.stride_block : 2 * D;
    char *base = reinterpret_cast<char *>(c.data);
    if (!make_tmap_4d(&tk, dt, base, D, c.block_size, c.n_heads, c.n_blocks, sp, sh, sb, 64, P.page_rows) ||
        !make_tmap_4d(&tv, dt, base + 2 * c.stride_kv, D, c.block_size, c.n_heads, c.n_blocks, sp, sh, sb, 64,
                      P.page_rows))
      return SB_ERR_CUDA;
  }
  auto kernel = prefill_kernel<T, D, CODES>;
  if (ensure_dynamic_smem(reinterpret_cast<const void *>(kernel), S::kSmem) != SB_OK) return SB_ERR_CUDA;
  P.next = reinterpret_cast<unsigned *>(workspace);
  P.status = status ? status : reinterpret_cast<int *>(workspace) + 1;
  const cudaError_t e = cudaMemsetAsync(workspace, 0, kPrefillWorkspace, st);
  if (e != cudaSuccess) {
    set_last_cuda_error(e);
    return SB_ERR_CUDA;
  }
  const int grid = (int)std::min<int64_t>(sm_count(), P.n_units);
  const int slot = prof_before(st);
  kernel<<<grid, S::kThreads, S::kSmem, st>>>(tk, tv, P);
  prof_after(slot, st);
  return launch_status();
}

}  // namespace

// Enough rows per request to fill tiles of 128; pages that cut a block of 128 keys evenly, in whole
// swizzle groups of 8 rows.
bool prefill_takes(const AttendParams &P, int dtype) {
  if (!decode_takes(P, dtype) || P.G > kBM || P.scale == 0.f || P.cache.n_blocks == 0) return false;
  if (!rows_aligned(P.out, 2, 16)) return false;
  const int bs = P.cache.block_size;
  if (bs % 8 || (bs < kBN ? kBN % bs : bs % kBN)) return false;
  const PrefillParams p = plan(P);
  if (p.n_units >= (1ll << 31)) return false;
  return (int64_t)P.batch.n_tokens * P.G >= 64 * (int64_t)P.batch.batch;
}

int launch_prefill(const AttendParams &A, int dtype, int32_t *status, void *workspace, cudaStream_t st) {
  PrefillParams P = plan(A);
  P.dtype = dtype;
  const bool wide = A.cache.head_dim == 128;
  if (A.cache.group != 0)
    return wide ? run<__half, 128, true>(P, status, workspace, st) : run<__half, 64, true>(P, status, workspace, st);
  if (dtype == SB_DTYPE_BF16)
    return wide ? run<__nv_bfloat16, 128, false>(P, status, workspace, st)
                : run<__nv_bfloat16, 64, false>(P, status, workspace, st);
  return wide ? run<__half, 128, false>(P, status, workspace, st) : run<__half, 64, false>(P, status, workspace, st);
}

}  // namespace paged
}  // namespace sb
