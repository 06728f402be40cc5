// Attention of prompts and prompt chunks over a paged cache on the 5th-generation tensor cores (tcgen05 + TMEM): the
// rows of a sequence that brings more than a few tokens, behind any cached past, 16-bit pages or e4m3 codes.
//
// The rows of a CTA are (token, query head of the group) pairs, so that heads which share a key / value head share its
// tiles too: 256 rows, two row tiles of 128, walk the visible keys in tiles of 128, half a tile (64 keys) at a time,
//   S  = Q K^T   (128 x 64)      in tensor memory, two buffers of 64 columns from 128 t on for row tile t
//   O += P V     (128 x D)       columns [256 + 128 t, +D); P, 16-bit, lies over the first 32 columns of its scores
// with V as an N-major operand.  The softmax warps (4-7 and 8-11, a thread per row) take a half's scores into registers and put its
// weights in their place, as the A operand of the second product, which spares shared memory a write and a read (it is what
// bounds products of 128 x 128 tiles: 128 bytes per cycle) and leaves it to three stages of K and two of V.  Warps 1 and 2 issue the
// products of a row tile each; the scores of half n + 2 follow the value product of half n, so that the softmax finds its next ones ready.
// The reference m of a row is raised only when a score exceeds it by 2^8, behind the last value product.
//
// Warp 0 moves 16-bit pages by TMA (one box per page and 64 dimensions, 128-byte swizzle; boxes of 16 and more rows are whole
// swizzle atoms and stack up to the tile).  Codes take four more warps (12-15) instead: they load a tile's codes into registers
// while the tile before is used, and store them as fp16 (exact) in the swizzled layout.  Queries of bf16 models then become
// fp16 with a power of two per row, which keeps all their bits.  A page's key scale multiplies its scores, and the value
// scale z enters the exponent, 2^(s + log2 z - m), and leaves the sum again: fp16 weights keep their precision where pages
// differ in magnitude.  Both are one fused multiply-add per score, as without scales.
//
// bf16 weights over 16-bit pages are rounded once (2^-8 of a weight, which averages out over keys): in two pieces, as in the
// few-token kernel, the second product would take twice as long.  fp16 weights (of fp16 models and of codes) are rounded once, 2^-11.
//
// Values that are not finite are taken out of tiles that hide keys from some rows: 16-bit pages by warp 3, which looks at such tiles between the
// copies and the products, codes by the issuing warps, on the cue of the warps that convert them.
//
// Bound by the chain scores -> softmax -> weights of a row tile: 2100 cycles per 64 keys and pair of row tiles, of which the special-function unit
// is busy 1024 and the tensor core 1280 (531 to 1024 tokens behind 3700 to 7000 cached ones, e4m3, 32 heads on 8: 280 us, 825 TFLOP/s).
// Tried and not kept, when that took 277 us: weights through shared memory, 311 us; weights in columns of their own, scores handed back before the softmax, 289 us; a part of
// the powers of two by multiply-adds (1 to 3 of 8), 290 to 300 us; halves that the mask hides skipped one by one, 296 us; two sets of softmax warps that take halves in turn, 415 us; converting with two warps instead
// of four, twice as long.  Over 16-bit pages of 64 positions the same took 330 us: twice the bytes through the second-level cache.
// Few rows behind a long past do not fill the machine: the key tiles are then split over CTAs, whose rows are merged by
// a second launch.
//
// Every mbarrier wait is bounded; a wait that runs out is recorded, the CTA's roles leave (each decision made
// uniform over the warp first), copies in flight are given time to land, TMEM is freed and the kernel returns.
#include <type_traits>

#include "paged_prompt.cuh"
#include "tc_ops.cuh"

namespace eb {
namespace {

constexpr int kKeys = 128, kRowTiles = 2, kCtaRows = kRowTiles * kRows, kHalf = 64, kConvertWarps = 4, kLookWarp = 3, kSoftmaxWarp = 4, kConvertWarp = kSoftmaxWarp + 4 * kRowTiles, kScaleRing = 4;
constexpr float kRaise = 8.f;               // the reference of a row is raised when a score exceeds it by 2^8
constexpr float kLiftHalf = 6.f;             // fp16 weights are 2^6 times as large, up to 2^14: fewer fall below the normal range
constexpr float kNone = -3.402823466e38f;

// tcgen05.wait::ld that the registers of two loads pass through: nothing reads them before
__device__ __forceinline__ void tc_ld_wait_for(float (&a)[32], float (&b)[32]) {
  tc_ld_wait();
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    asm volatile("" : "+f"(a[i]), "+f"(a[i + 1]), "+f"(a[i + 2]), "+f"(a[i + 3]), "+f"(a[i + 4]), "+f"(a[i + 5]), "+f"(a[i + 6]), "+f"(a[i + 7]));
    asm volatile("" : "+f"(b[i]), "+f"(b[i + 1]), "+f"(b[i + 2]), "+f"(b[i + 3]), "+f"(b[i + 4]), "+f"(b[i + 5]), "+f"(b[i + 6]), "+f"(b[i + 7]));
  }
}

// bar_wait in line: a function of its own would tie the register counts of the roles together
__device__ __forceinline__ bool wait_inline(uint32_t bar, uint32_t parity, volatile int *abort_flag, int where) {
  if (bar_try(bar, parity)) return true;
  const unsigned long long t0 = gtimer();
  for (unsigned it = 1;; ++it) {
    if (bar_try(bar, parity)) return true;
    if ((it & 63u) == 0) {
      if (*abort_flag) return false;
      if (gtimer() - t0 > kTcWaitNs) {
        *abort_flag = 1;
        if (atomicCAS(&g_tc_status[0], 0, EB_ETIMEDOUT) == 0) {
          g_tc_status[1] = where;
          g_tc_status[2] = blockIdx.x;
          g_tc_status[3] = (int)parity;
        }
        return false;
      }
    }
  }
}

__device__ __forceinline__ void tc_ld16(uint32_t taddr, uint32_t *r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                 "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr));
  tc_ld_wait();
#pragma unroll
  for (int i = 0; i < 16; i += 8)
    asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]));
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z, int w) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(map), "r"(x),
               "r"(y), "r"(z), "r"(w), "r"(bar)
               : "memory");
}

template <int D, bool EIGHT> struct PromptSmem {
  static constexpr uint32_t kQBytes = (D / 64) * kRows * 128, kKBytes = (D / 64) * kKeys * 128;
  static constexpr int kKStages = 3, kVStages = 2;
  static constexpr int kThreads = (kConvertWarp + (EIGHT ? kConvertWarps : 0)) * 32;
  static constexpr size_t kTotal = 1024 + 1024 + (size_t)kRowTiles * kQBytes + (kKStages + kVStages) * (size_t)kKBytes;
};

// Shared memory (1024-aligned): [1 KB: barriers, TMEM slot, abort flag, per 16 keys of the last four tiles: key scale, log2 of
// the value scale and its inverse, and a word of those in no page; of tiles that hide keys from some rows: the keys whose values are not finite][Q][K: 3 stages][V: 2 stages]
template <typename T, bool EIGHT, int D>
__global__ void __launch_bounds__(PromptSmem<D, EIGHT>::kThreads, 1)
paged_prompt_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const PromptParams p) {
  using Smem = PromptSmem<D, EIGHT>;
  using M = typename std::conditional<EIGHT, __half, T>::type;
  constexpr int kSub = D / 64, kKStages = Smem::kKStages, kVStages = Smem::kVStages;
  constexpr uint32_t kQBytes = Smem::kQBytes, kKBytes = Smem::kKBytes, kTmemCols = 512, kPvCol = 2 * kKeys;
  constexpr bool kScaled = EIGHT && std::is_same<T, __nv_bfloat16>::value;        // queries become fp16, a power of two per row
  constexpr float kLift = std::is_same<M, __half>::value ? kLiftHalf : 0.f;
  constexpr int kBf16 = std::is_same<M, __nv_bfloat16>::value ? 1 : 0;
  constexpr uint32_t kIdescS = tc_idesc(kHalf, kBf16), kIdescPV = tc_idesc(D, kBf16) | (1u << 16);     // bit 16: B is N-major

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = s32(smem_raw);
  uint8_t *smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  const uint32_t bar0 = s32(smem);
  // per stage of K and V; per row tile and buffer of scores and weights
  const uint32_t q_full = bar0, q_raw = bar0 + 8, k_full = bar0 + 16, k_empty = bar0 + 40, v_full = bar0 + 64, v_empty = bar0 + 80, s_full = bar0 + 96,
                 p_full = bar0 + 128, pv_full = bar0 + 160, v_ready = bar0 + 192;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + 256);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + 264);
  float *key_scale = reinterpret_cast<float *>(smem + 272), *value_log = key_scale + kScaleRing * 8, *value_inv = value_log + kScaleRing * 8;
  uint32_t *no_page = reinterpret_cast<uint32_t *>(value_inv + kScaleRing * 8);
  // [0]: whether there may be any; [1] to [3]: what says which tiles they are (in registers it would cost the softmax some); from [4] on four words per tile
  volatile uint32_t *bad = no_page + kScaleRing;
  uint8_t *q_ptr = smem + 1024, *k_ptr = q_ptr + kRowTiles * kQBytes, *v_ptr = k_ptr + kKStages * kKBytes;
  const uint32_t q_addr = s32(q_ptr), k_addr = s32(k_ptr), v_addr = s32(v_ptr);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  griddep_wait();
  // of a sequence the latest rows, which see most, of all heads first: its earliest, with few keys, fill up the end
  const int blocks = gridDim.x / p.splits, id = blockIdx.y * gridDim.x + blockIdx.x, hk = id % p.kv_heads, of_head = id / p.kv_heads,
            split = of_head % p.splits, qb = blocks - 1 - of_head / p.splits, b = blockIdx.z;
  const PagedRows r = paged_rows(p.batch, b);
  const int all = r.count * p.group, q0 = qb * kCtaRows, reach = p.batch.table_cols << p.batch.page_shift;
  if (all <= p.few || q0 >= all) return;
  // Halves of key tiles (64 keys) that each row tile walks, [hs, he), none for one that lies behind the sequence's rows; the CTA's own tiles
  // are [jmin, nmax).  Keys outside of [lo, hi) are seen by no row of the CTA.
  int hs[kRowTiles], he[kRowTiles], nmax = 0, jmin = 0x7fffffff, lo = 0x7fffffff, hi = 0;
#pragma unroll
  for (int t = 0; t < kRowTiles; ++t) {
    const int a = q0 + t * kRows, z = min(a + kRows, all) - 1;
    const int first = p.window > 0 ? max(0, r.past + a / p.group - p.window + 1) : 0, end = a < all ? min(r.past + z / p.group + 1, reach) : 0;
    he[t] = (end + kHalf - 1) / kHalf;
    hs[t] = first / kHalf;
    if (he[t] > hs[t]) {
      jmin = min(jmin, hs[t] / 2);
      nmax = max(nmax, (he[t] + 1) / 2);
      lo = min(lo, first);
      hi = max(hi, end);
    }
  }
  if (jmin > nmax) jmin = nmax;
  if (p.splits > 1) {
    jmin += split * p.split_tiles;
    if (split > 0 && jmin >= nmax) return;
    nmax = min(nmax, split == p.splits - 1 ? nmax : jmin + p.split_tiles);
#pragma unroll
    for (int t = 0; t < kRowTiles; ++t) {
      hs[t] = max(hs[t], 2 * jmin);
      he[t] = min(he[t], 2 * nmax);
    }
  }
#pragma unroll
  for (int t = 0; t < kRowTiles; ++t)
    if (he[t] <= hs[t]) he[t] = hs[t] = 0;                // (walks nothing)

  // A weight of 0 does not hide a value that is not finite: later tokens of the call, or keys that a window has left behind, may hold such for rows that do
  // not see them.  Where a tile hides keys from some of the CTA's rows (three tiles at either end at most), such values leave it, and are added at
  // the end to the rows that see them.  (2 % of the time of 16-bit prompts, 5 % of that of e4m3 ones of three to seven tiles.)
  auto hides = [&](int j) { return j >= (int)bad[1] || j * kKeys <= (int)bad[3]; };
  auto bad_of = [&](int j) { return 4 + 4 * (j >= (int)bad[1] ? j - (int)bad[1] : 4 + j - (int)bad[2]); };
  auto is_bad = [&](int j, int row) {
    atomicOr(const_cast<uint32_t *>(bad) + bad_of(j) + (row >> 5), 1u << (row & 31));
    bad[0] = 1;
  };
  // (by a warp, of a tile of values; two may find and write the same)
  constexpr int kChunks = kKeys * kSub * 8;
  auto take_out = [&](uint4 *tile, int j) {
#pragma unroll 1
    for (int e = lane; e < kChunks; e += 32)
      if (any_not_finite<M>(tile[e])) {
        tile[e] = finite_only<M>(tile[e]);
        is_bad(j, (e >> 3) % kKeys);
      }
  };
  if (threadIdx.x < 36) {
    const int first_pos = r.past + q0 / p.group, last_pos = r.past + (min(q0 + kCtaRows, all) - 1) / p.group;
    bad[threadIdx.x] = threadIdx.x == 1 ? (first_pos + 1) / kKeys : threadIdx.x == 2 ? lo / kKeys : threadIdx.x == 3 ? (p.window > 0 ? last_pos - p.window : -1) : 0;
  }

  if (threadIdx.x == 0) {
    if (!EIGHT) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(&tm_k) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&tm_v) : "memory");
    }
    bar_init(q_full, p.q_tma && !kScaled ? 1 : kRowTiles * 4);
    bar_init(q_raw, 1);
    for (int s = 0; s < kKStages; ++s) {
      bar_init(k_full + 8 * s, EIGHT ? kConvertWarps : 1);
      bar_init(k_empty + 8 * s, kRowTiles);
    }
    for (int s = 0; s < kVStages; ++s) {
      bar_init(v_full + 8 * s, EIGHT ? kConvertWarps : 1);
      bar_init(v_empty + 8 * s, kRowTiles);
      bar_init(v_ready + 8 * s, 1);
    }
    for (int s = 0; s < 2 * kRowTiles; ++s) {
      bar_init(s_full + 8 * s, 1);
      bar_init(p_full + 8 * s, 4);
      bar_init(pv_full + 8 * s, 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (p.q_tma) {
      // queries as soon as there is a barrier to land on: [tokens][heads of the group][D] as rows of a tile; those of bf16 models over codes then become
      // fp16 where they lie.  (Rows behind the sequence's last are the next one's, or zeros: they store nothing.)
      const uint32_t bar = kScaled ? q_raw : q_full;
      bar_expect_tx(bar, kRowTiles * kQBytes);
#pragma unroll
      for (int t = 0; t < kRowTiles; ++t)
#pragma unroll
        for (int kb = 0; kb < kSub; ++kb)
          tma_load_4d(q_addr + t * kQBytes + kb * kRows * 128, &tm_q, bar, kb * 64, 0, hk, r.row0 + (q0 + t * kRows) / p.group);
    }
  }
  if (warp == 1) {
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(tmem_slot)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // the pages of a tile, of lane l of warp 0; those of the first tiles are looked up on the way to the barrier
  const int per_tile = kKeys >> p.batch.page_shift, page_size = 1 << p.batch.page_shift;
  auto page_of = [&](int j) {                              // (one outside of the pool reads as zeros)
    const int key = j * kKeys + (lane << p.batch.page_shift);
    return lane < per_tile && j < nmax && key < hi && key + page_size > lo ? paged_page(p.batch, b, key >> p.batch.page_shift) : -1;
  };
  int now = -1, next = -1;
  if (!EIGHT && warp == 0) {
    now = page_of(jmin);
    next = page_of(jmin + 1);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  griddep_launch();                                       // (not before: a following kernel must not take the tensor memory first)
  auto all_wait = [&](uint32_t bar, uint32_t parity, int where) { return __all_sync(0xffffffffu, wait_inline(bar, parity, abort_flag, where)) != 0; };

  // Registers go where 64 scores and their weights are kept: of 128 per thread at launch with the converters' warpgroup 80 + 2 x 168 + 96,
  // of 168 without it 120 + 2 x 192.  (The launch checks that the kernel got them.)
  if (warp < kSoftmaxWarp) {
    if (EIGHT) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 120;");
  }
  if (warp == 0) {
    // ---------------- 16-bit pages: TMA, a lane per page of a tile ----------------
    if (!EIGHT && nmax > jmin) {
      const int outside = p.batch.pages * p.kv_heads;
      auto load = [&](const CUtensorMap *map, uint32_t dst, uint32_t bar, int page) {
        if (lane == 0) bar_expect_tx(bar, kKBytes);
        __syncwarp();
        if (lane < per_tile) {
          const int block = page >= 0 ? page * p.kv_heads + hk : outside;
#pragma unroll
          for (int kb = 0; kb < kSub; ++kb) tma_load_3d(dst + kb * kKeys * 128 + (lane << p.batch.page_shift) * 128, map, bar, kb * 64, 0, block);
        }
      };
      auto load_k = [&](int j, int page) -> bool {
        const int i = j - jmin, st = i % kKStages;
        if (i >= kKStages && !all_wait(k_empty + 8 * st, (i / kKStages - 1) & 1, 1)) return false;
        // groups of 16 keys without a page, where some row could see them
        const int key = j * kKeys + (lane << p.batch.page_shift), groups = page_size >> 4;
        uint32_t mine = lane < per_tile && page < 0 && key < hi && key + page_size > lo ? ((1u << groups) - 1) << (lane * groups) : 0;
        mine = __reduce_or_sync(0xffffffffu, mine);
        if (lane == 0) no_page[i & (kScaleRing - 1)] = mine;
        load(&tm_k, k_addr + st * kKBytes, k_full + 8 * st, page);
        return true;
      };
      bool ok = load_k(jmin, now);
      for (int j = jmin; j < nmax && ok; ++j) {
        const int i = j - jmin, vs = i % kVStages, vu = i / kVStages;
        const int later = page_of(j + 2);
        if (j + 1 < nmax && !load_k(j + 1, next)) break;
        if (i >= kVStages && !all_wait(v_empty + 8 * vs, (vu - 1) & 1, 9)) break;
        load(&tm_v, v_addr + vs * kKBytes, v_full + 8 * vs, now);
        now = next;
        next = later;
      }
    }
  } else if (warp <= kRowTiles) {
    // ---------------- MMA issuers: a warp per row tile ----------------
    // The scores of the first two halves, then for every half n, as soon as P(n) is written: O += P(n) V(n), and behind that S(n + 2), which takes
    // P(n)'s place, so that scores are there a whole half before they are needed.  Both warps hand back every stage, those of tiles that
    // theirs does not walk too, each when it is full (an earlier arrival would count for the stage's use before).
    const int t = warp - 1, first = t == 0 ? hs[0] : hs[1], end = t == 0 ? he[0] : he[1];
    const uint32_t t_s = tmem + t * kKeys, t_pv = t_s + kPvCol;
    auto pass = [&](int j) -> bool {                       // a tile that this row tile does not walk
      const int i = j - jmin, ks = i % kKStages, vs = i % kVStages;
      if (!all_wait(k_full + 8 * ks, (i / kKStages) & 1, 3)) return false;
      if (lane == 0) bar_arrive(k_empty + 8 * ks);
      if (!all_wait((EIGHT ? v_full : v_ready) + 8 * vs, (i / kVStages) & 1, 10)) return false;
      if (lane == 0) bar_arrive(v_empty + 8 * vs);
      return true;
    };
    auto issue_scores = [&](int n) -> bool {
      const int i = (n >> 1) - jmin, st = i % kKStages, buf = (n - first) & 1;
      if (!all_wait(k_full + 8 * st, (i / kKStages) & 1, 3)) return false;
      tc_fence_after();
#pragma unroll
      for (int kb = 0; kb < kSub; ++kb) {
        const uint64_t a = tc_desc(q_addr + t * kQBytes + kb * kRows * 128), bd = tc_desc(k_addr + st * kKBytes + kb * kKeys * 128 + (n & 1) * kHalf * 128);
#pragma unroll
        for (int k = 0; k < 4; ++k) tc_mma_warp(t_s + buf * kHalf, a + 2 * k, bd + 2 * k, kIdescS, (kb > 0 || k > 0) ? 1u : 0u);
      }
      tc_commit_warp(s_full + 8 * (2 * t + buf));
      if ((n & 1) || n + 1 == end) tc_commit_warp(k_empty + 8 * st);
      return true;
    };
    bool ok = true;
    if (end > first) {
      for (int j = jmin; j < first / 2 && ok; ++j) ok = pass(j);
      ok = ok && all_wait(q_full, 0, 2) && issue_scores(first) && (first + 1 == end || issue_scores(first + 1));
      for (int n = first; n < end && ok; ++n) {
        const int at = n - first, buf = at & 1, j = n >> 1, i = j - jmin, vs = i % kVStages;
        if (EIGHT && ((n & 1) == 0 || n == first)) {
          if (!(ok = all_wait(v_full + 8 * vs, (i / kVStages) & 1, 10))) break;
          if (__any_sync(0xffffffffu, bad[0]) && hides(j)) {
            take_out(reinterpret_cast<uint4 *>(v_ptr + vs * kKBytes), j);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
          }
        }
        ok = all_wait(p_full + 8 * (2 * t + buf), (at >> 1) & 1, 5) && (EIGHT || all_wait(v_ready + 8 * vs, (i / kVStages) & 1, 10));
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          // 16 keys per instruction: two 8-row groups (2048 bytes) down the V tile, eight columns of P
          const uint64_t bd = tc_desc_nmajor(v_addr + vs * kKBytes + ((n & 1) * 4 + k) * 2048, kKeys * 128);
          tc_mma_ts_warp(t_pv, t_s + buf * kHalf + k * 8, bd, kIdescPV, (at > 0 || k > 0) ? 1u : 0u);
        }
        tc_commit_warp(pv_full + 8 * (2 * t + buf));
        if ((n & 1) || n + 1 == end) tc_commit_warp(v_empty + 8 * vs);
        // (products on different accumulators are ordered by nothing but their completion)
        if (n + 2 < end) ok = all_wait(pv_full + 8 * (2 * t + buf), (at >> 1) & 1, 4) && issue_scores(n + 2);
      }
    }
    for (int j = max((end + 1) / 2, jmin); j < nmax && ok; ++j) ok = pass(j);
  } else if (!EIGHT && warp == kLookWarp) {
    // ---------------- a look at the 16-bit values of a tile, on their way to the products ----------------
    // (By a warp of its own: the issuing warps, at the same work, took 194 us for the prompts that take 184 so.)
    bool ok = true;
    for (int j = jmin; j < nmax && ok; ++j) {
      const int i = j - jmin, vs = i % kVStages;
      if (!(ok = all_wait(v_full + 8 * vs, (i / kVStages) & 1, 12))) break;
      const bool edge = j * kKeys < lo || (j + 1) * kKeys > hi;
      if (edge || hides(j)) {
        uint4 *tile = reinterpret_cast<uint4 *>(v_ptr + vs * kKBytes);
        constexpr int kBatch = 8;
        if (edge)                                          // value rows that no row sees may hold anything
          for (int e = lane; e < kChunks; e += 32) {
            const int key = j * kKeys + (e >> 3) % kKeys;
            if (key < lo || key >= hi) tile[e] = make_uint4(0, 0, 0, 0);
          }
        bool found = false;
#pragma unroll 1
        for (int e = lane; e < kChunks; e += 32 * kBatch) {
          uint4 x[kBatch];
#pragma unroll
          for (int u = 0; u < kBatch; ++u) x[u] = tile[e + u * 32];
#pragma unroll
          for (int u = 0; u < kBatch; ++u) found |= any_not_finite<M>(x[u]);
        }
        if (__any_sync(0xffffffffu, found)) take_out(tile, j);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
      }
      if (lane == 0) bar_arrive(v_ready + 8 * vs);
    }
  } else if (warp >= kSoftmaxWarp && warp < kConvertWarp) {
    if (EIGHT) asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    // ---------------- softmax warps: 4 per row tile, thread = row ----------------
    const int t = (warp - kSoftmaxWarp) >> 2, quarter = warp & 3, row = quarter * 32 + lane, at = q0 + t * kRows + row;
    const bool there = at < all;
    const int token = at / p.group, head = hk * p.group + at % p.group;
    const int end_half = t == 0 ? he[0] : he[1], first_half = t == 0 ? hs[0] : hs[1];
    const uint32_t t_row = tmem + ((uint32_t)(quarter * 32) << 16) + t * kKeys, t_pv = t_row + kPvCol;
    const uint32_t my_s_full = s_full + 16 * t, my_p_full = p_full + 16 * t, my_pv_full = pv_full + 16 * t;
    float factor = p.scale_log2;                          // exponent of a score
    bool alive = true;
    {
      if (p.q_tma) {
        // (waited for by rows that walk nothing too: their memory is used below, and nothing may be on its way when the CTA leaves)
        if (!all_wait(kScaled ? q_raw : q_full, 0, 6)) alive = false;
      } else {
        // groups that do not divide a tile: the warp's 32 rows, swizzled, D / 8 lanes per row, straight to shared memory.  (With most of it
        // taken, the first-level cache is too small for as many loads to registers: 6 us instead of 2 in front of the first product.)
        constexpr int kLanesPer = D / 8, kRowsPer = 32 / kLanesPer;
        const int sub = lane / kLanesPer, chunk = lane % kLanesPer;
        const uint32_t dst = q_addr + t * kQBytes + (chunk >> 3) * (kRows * 128);
#pragma unroll 4
        for (int i = 0; i < 32 / kRowsPer; ++i) {
          // (token and head of the row, computed by its own lane)
          const int from = i * kRowsPer + sub, to = quarter * 32 + from, tk = __shfl_sync(0xffffffffu, token, from), hd = __shfl_sync(0xffffffffu, head, from);
          const bool ok = q0 + t * kRows + to < all;
          const T *src = reinterpret_cast<const T *>(p.q) + (ok ? (long long)(r.row0 + tk) * p.ldq + (long long)hd * D + chunk * 8 : 0);
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + to * 128 + (((chunk & 7) ^ (to & 7)) << 4)), "l"(src), "r"(ok ? 16 : 0) : "memory");
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
      }
      if constexpr (kScaled) {
        uint8_t *to = q_ptr + t * kQBytes + row * 128;
        const uint8_t *from = to;
        float m = 0.f;
#pragma unroll 4
        for (int i = 0; i < D / 8; ++i) {
          const uint4 w = *reinterpret_cast<const uint4 *>(from + (i >> 3) * (kRows * 128) + (((i & 7) ^ (row & 7)) << 4));
          const float2 f0 = unpack2<T>(w.x), f1 = unpack2<T>(w.y), f2 = unpack2<T>(w.z), f3 = unpack2<T>(w.w);
          m = fmaxf(fmaxf(fmaxf(m, fmaxf(fabsf(f0.x), fabsf(f0.y))), fmaxf(fabsf(f1.x), fabsf(f1.y))),
                    fmaxf(fmaxf(fabsf(f2.x), fabsf(f2.y)), fmaxf(fabsf(f3.x), fabsf(f3.y))));
        }
        // the largest magnitude to [2^14, 2^15): what falls out of fp16's range below is 2^-38 of it
        const int e = min(max(14 - ((__float_as_int(m) >> 23) - 127), -100), 100);
        const float up = __int_as_float((127 + e) << 23);
        factor *= __int_as_float((127 - e) << 23);
#pragma unroll 4
        for (int i = 0; i < D / 8; ++i) {
          const int at16 = (i >> 3) * (kRows * 128) + (((i & 7) ^ (row & 7)) << 4);
          const uint4 w = *reinterpret_cast<const uint4 *>(from + at16);
          const float2 f0 = unpack2<T>(w.x), f1 = unpack2<T>(w.y), f2 = unpack2<T>(w.z), f3 = unpack2<T>(w.w);
          *reinterpret_cast<uint4 *>(to + at16) = make_uint4(pack2<__half>(f0.x * up, f0.y * up), pack2<__half>(f1.x * up, f1.y * up),
                                                             pack2<__half>(f2.x * up, f2.y * up), pack2<__half>(f3.x * up, f3.y * up));
        }
      }
      if (kScaled || !p.q_tma) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) bar_arrive(q_full);
      }
    }
    const int pos = r.past + token;
    const int vis_end = there ? min(pos + 1, reach) : 0, vis_begin = p.window > 0 ? max(0, pos - p.window + 1) : 0;       // this row sees [vis_begin, vis_end)
    float m_ref = kNone, l_run = 0.f;
    for (int n = first_half; n < end_half && alive; ++n) {
      const int at_half = n - first_half, buf = at_half & 1, key0 = n * kHalf, slot = ((n >> 1) - jmin) & (kScaleRing - 1), c0 = (n & 1) * 2;      // (c0: the half's first chunk of 32 keys in its tile)
      const uint32_t t_s = t_row + buf * kHalf;            // scores of the half, and its weights in the first 32 columns
      if (!all_wait(my_s_full + 8 * buf, (at_half >> 1) & 1, 7)) { alive = false; break; }
      tc_fence_after();
      float x0[32], x1[32];
      tc_ld32_issue(t_s, reinterpret_cast<uint32_t *>(x0));
      tc_ld32_issue(t_s + 32, reinterpret_cast<uint32_t *>(x1));
      // groups of 16 keys without a page
      const uint32_t gone = EIGHT ? 0 : no_page[slot] >> (2 * c0) & 15;
      // most halves of a long prompt: every row sees every key
      const bool whole = __all_sync(0xffffffffu, !there || (key0 >= vis_begin && key0 + kHalf <= vis_end)) && !gone;
      tc_ld_wait_for(x0, x1);
      // Which of 32 keys this row sees.  (Rows behind the sequence's last count as seeing all, which leaves it to the others.)
      auto hide = [&](float (&x)[32], int c) {
        const int end = vis_end - (key0 + c * 32), begin = vis_begin - (key0 + c * 32);
        uint32_t bits = end >= 32 ? 0xffffffffu : end <= 0 ? 0u : (1u << end) - 1u;
        if (begin > 0) bits &= begin >= 32 ? 0u : ~((1u << begin) - 1u);
        if (!EIGHT && gone) bits &= ((gone >> (2 * c)) & 1 ? 0u : 0xffffu) | ((gone >> (2 * c)) & 2 ? 0u : 0xffff0000u);
        if (!there) bits = 0xffffffffu;
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = (bits >> e) & 1 ? x[e] : -INFINITY;
      };
      if (!whole) {
        hide(x0, 0);
        hide(x1, 1);
      }
      // factor and summand of a group's exponents (the factor is never 0, which would make a NaN of a hidden score)
      float factors[4], logs[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        factors[g] = EIGHT ? fmaxf(factor * key_scale[slot * 8 + 2 * c0 + g], 1e-37f) : factor;
        logs[g] = EIGHT ? value_log[slot * 8 + 2 * c0 + g] : 0.f;
      }
      auto largest = [&](const float *x, int g) {          // exponent of 16 keys
        float r0 = x[0], r1 = x[1];
#pragma unroll
        for (int e = 2; e < 14; e += 4) {
          r0 = fmaxf(r0, fmaxf(x[e], x[e + 1]));           // (one instruction for three)
          r1 = fmaxf(r1, fmaxf(x[e + 2], x[e + 3]));
        }
        return fmaf(fmaxf(fmaxf(r0, r1), fmaxf(x[14], x[15])), factors[g], logs[g]);
      };
      const float m = fmaxf(fmaxf(largest(x0, 0), largest(x0 + 16, 1)), fmaxf(largest(x1, 2), largest(x1 + 16, 3)));
      // (Rows behind the sequence's last have no vote: they hold another sequence's queries, or anything, which must not change these rows' bits.)
      if (__any_sync(0xffffffffu, there && m > m_ref + kRaise)) {
        // The reference is raised, for all rows of the warp (tensor memory is read and written warp-wide), behind the last value product.
        const float m_new = fmaxf(m_ref, m), alpha = ex2(m_ref - m_new);
        l_run = EIGHT ? sum_at(l_run, m_ref - m_new) : l_run * alpha;
        m_ref = m_new;
        if (at_half > 0) {
          if (!all_wait(my_pv_full + 8 * (buf ^ 1), ((at_half - 1) >> 1) & 1, 8)) { alive = false; break; }
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t y[16];
            tc_ld16(t_pv + c * 16, y);
#pragma unroll
            for (int e = 0; e < 16; ++e) y[e] = __float_as_uint(__uint_as_float(y[e]) * alpha);
            tc_st16(t_pv + c * 16, y);
          }
          tc_st_wait();
        }
      }
      // Weights: exponents, powers, their sum (without the value scale), and the 16-bit operand of the second product, two to a register.
      uint32_t w0[16], w1[16];
      auto weigh = [&](float (&x)[32], int c, uint32_t (&w)[16]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float f = factors[2 * c + h], a = logs[2 * c + h] - (m_ref - kLift);
          float l0 = 0.f, l1 = 0.f;
#pragma unroll
          for (int e = h * 16; e < h * 16 + 16; e += 2) {
            fma2(x[e], x[e + 1], x[e], x[e + 1], f, f, a, a);
            x[e] = ex2(x[e]);
            x[e + 1] = ex2(x[e + 1]);
            add2(l0, l1, l0, l1, x[e], x[e + 1]);
            w[e / 2] = pack2<M>(x[e], x[e + 1]);
          }
          l_run = EIGHT ? fmaf(l0 + l1, value_inv[slot * 8 + 2 * (c0 + c) + h], l_run) : l_run + (l0 + l1);
        }
      };
      if (EIGHT && __builtin_expect(fminf(fminf(logs[0], logs[1]), fminf(logs[2], logs[3])) < m_ref - kFarBelow, 0)) {
        auto far = [&](const float (&x)[32], int c) {
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const int g = 2 * c + e / 16;
            if (logs[g] > kNone && fmaf(x[e], factors[g], logs[g] - (m_ref - kLift)) < kLeastPower) l_run += ex2(fmaf(x[e], factors[g], kLift - m_ref));
          }
        };
        far(x0, 0);
        far(x1, 1);
      }
      weigh(x0, 0, w0);
      weigh(x1, 1, w1);
      tc_st16(t_s, w0);                                    // (over scores of this warp's own rows, which are in registers)
      tc_st16(t_s + 16, w1);
      tc_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive(my_p_full + 8 * buf);      // P is complete for this warp's 32 rows (and these are rescaled)
    }
    const bool walked = end_half > first_half;
    const int last = end_half - 1 - first_half;
    if (walked && alive && !all_wait(my_pv_full + 8 * (last & 1), (last >> 1) & 1, 11)) alive = false;
    if (alive || !walked) {
      tc_fence_after();
      float *part = p.part ? p.part + ((((long long)b * p.kv_heads + hk) * blocks + qb) * p.splits + split) * kCtaRows * (D + 2) + (long long)(t * kRows + row) * (D + 2) : nullptr;
      if (part && there) *reinterpret_cast<float2 *>(part + D) = make_float2(m_ref, l_run);
      const float inv = part ? 1.f : l_run == 0.f ? 0.f : 1.f / l_run;
      // 16-bit rows go through the memory of Q, which the last product is done with: written by their threads, 16 bytes of 32 rows
      // at a time, they took 6100 cycles
      uint8_t *stage = q_ptr + t * kQBytes;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        float x[32];
        if (walked) {
          tc_ld32(t_pv + c * 32, x);                 // warp-wide: rows behind the sequence's last are read too, and store nothing
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] = 0.f;
        }
        if (part) {
          if (there)
#pragma unroll
            for (int e = 0; e < 32; e += 2) *reinterpret_cast<float2 *>(part + c * 32 + e) = make_float2(x[e], x[e + 1]);
        } else {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const float *y = x + g * 8;
            *reinterpret_cast<uint4 *>(stage + (c >> 1) * (kRows * 128) + row * 128 + ((((c & 1) * 4 + g) ^ (row & 7)) << 4)) =
                make_uint4(pack2<T>(y[0] * inv, y[1] * inv), pack2<T>(y[2] * inv, y[3] * inv), pack2<T>(y[4] * inv, y[5] * inv), pack2<T>(y[6] * inv, y[7] * inv));
          }
        }
      }
      if (walked && bad[0]) {
        const int page_mask = (1 << p.batch.page_shift) - 1;
#pragma unroll 1
        for (int j = first_half / 2; j < (end_half + 1) / 2; ++j) {
          if (!hides(j)) continue;
#pragma unroll 1
          for (int key = max(j * kKeys, vis_begin); key < min((j + 1) * kKeys, vis_end); ++key) {
            if (!(bad[bad_of(j) + ((key % kKeys) >> 5)] >> (key & 31) & 1)) continue;
            const int page = paged_page(p.batch, b, key >> p.batch.page_shift);
            const long long from = (((long long)page * p.kv_heads + hk) << p.batch.page_shift) * D + (key & page_mask) * D;
#pragma unroll 1
            for (int d = 0; d < D; ++d) {
              float v;
              if constexpr (EIGHT) v = unpack2<__half>(e4m3x2_to_half2(reinterpret_cast<const uint8_t *>(p.v_pages)[from + d])).x;
              else v = to_f32<T>(reinterpret_cast<const T *>(p.v_pages)[from + d]);
              if (isfinite(v)) continue;
              T *y = reinterpret_cast<T *>(stage + (d >> 6) * (kRows * 128) + row * 128 + ((((d >> 3) & 7) ^ (row & 7)) << 4) + (d & 7) * 2);
              if (part) part[d] += v;
              else *y = from_f32<T>(to_f32<T>(*y) + v);
            }
          }
        }
      }
      if (!part) {
        __syncwarp();
        constexpr int kLanesPer = D / 8, kRowsPer = 32 / kLanesPer;
        const int sub = lane / kLanesPer, chunk = lane % kLanesPer;
        T *out = reinterpret_cast<T *>(p.o) + chunk * 8;
#pragma unroll 4
        for (int i = 0; i < 32 / kRowsPer; ++i) {
          const int from = i * kRowsPer + sub, of = quarter * 32 + from, tk = __shfl_sync(0xffffffffu, token, from), hd = __shfl_sync(0xffffffffu, head, from);
          if (q0 + t * kRows + of < all)
            *reinterpret_cast<uint4 *>(out + (long long)(r.row0 + tk) * p.ldo + (long long)hd * D) =
                *reinterpret_cast<const uint4 *>(stage + (chunk >> 3) * (kRows * 128) + of * 128 + (((chunk & 7) ^ (of & 7)) << 4));
        }
      }
    }
  } else if (EIGHT && warp >= kConvertWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    // ---------------- e4m3 codes: registers one tile ahead, fp16 into shared memory ----------------
    // Warp w has keys 32 w .. + 31 of a tile: a load takes kRowsPer rows, kLanesPer lanes of 16 codes each.
    constexpr int kOwn = kKeys / kConvertWarps, kLanesPer = D / 16, kRowsPer = 32 / kLanesPer, kLoads = kOwn / kRowsPer, kGroups = kOwn / 16;
    const int w = warp - kConvertWarp, sub = lane / kLanesPer, chunk = lane % kLanesPer;
    const long long block_bytes = (long long)D << p.batch.page_shift;
    const int in_page = (1 << p.batch.page_shift) - 1;
    // lane l keeps the page of the warp's group l mod 2 of 16 keys
    auto page_of = [&](int j) {
      const int key = j * kKeys + w * kOwn + (lane & (kGroups - 1)) * 16;
      return j < nmax && key < hi && key + 16 > lo ? paged_page(p.batch, b, key >> p.batch.page_shift) : -1;
    };
    uint4 kbuf[kLoads], vbuf[kLoads];
    auto fetch = [&](const void *pool, uint4 (&buf)[kLoads], int j, int group_pages) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int row = i * kRowsPer + sub, key = j * kKeys + w * kOwn + row, page = __shfl_sync(0xffffffffu, group_pages, row >> 4);
        buf[i] = make_uint4(0, 0, 0, 0);
        if (page >= 0 && key >= lo && key < hi)
          buf[i] = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint8_t *>(pool) + ((long long)page * p.kv_heads + hk) * block_bytes + (key & in_page) * D + chunk * 16);
      }
    };
    // 16 codes = two 16-byte chunks of fp16; the lanes of the second 64 dimensions store theirs the other way around, or pairs of
    // lanes would meet in a bank
    auto store = [&](uint8_t *tile, const uint4 (&buf)[kLoads]) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int row = w * kOwn + i * kRowsPer + sub;
        const uint4 lo8 = make_uint4(e4m3x2_to_half2(buf[i].x), e4m3x2_to_half2(buf[i].x >> 16), e4m3x2_to_half2(buf[i].y), e4m3x2_to_half2(buf[i].y >> 16));
        const uint4 hi8 = make_uint4(e4m3x2_to_half2(buf[i].z), e4m3x2_to_half2(buf[i].z >> 16), e4m3x2_to_half2(buf[i].w), e4m3x2_to_half2(buf[i].w >> 16));
        const bool swap = chunk >= 4;
        uint8_t *dst = tile + (chunk >> 2) * (kKeys * 128) + row * 128;
        const int c0 = (chunk & 3) * 2;
        *reinterpret_cast<uint4 *>(dst + (((c0 + (swap ? 1 : 0)) ^ (row & 7)) << 4)) = swap ? hi8 : lo8;
        *reinterpret_cast<uint4 *>(dst + (((c0 + (swap ? 0 : 1)) ^ (row & 7)) << 4)) = swap ? lo8 : hi8;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
    };
    auto scales = [&](int j, int page) {
      if (lane < kGroups) {
        const int at = ((j - jmin) & (kScaleRing - 1)) * 8 + w * kGroups + lane;
        const long long block = (long long)page * p.kv_heads + hk;
        const float z = page >= 0 ? fmaxf(p.v_scale[block], kLeastScale) : 0.f;
        key_scale[at] = page >= 0 ? p.k_scale[block] : 1.f;
        value_log[at] = page >= 0 ? __log2f(z) : -INFINITY;
        value_inv[at] = page >= 0 ? 1.f / z : 0.f;
      }
      __syncwarp();
    };
    if (nmax > jmin) {
      int k_pages = page_of(jmin), v_pages = k_pages, next = page_of(jmin + 1);
      fetch(p.k_pages, kbuf, jmin, k_pages);
      fetch(p.v_pages, vbuf, jmin, v_pages);
      // K runs a tile ahead of V: its stage is released earlier
      auto put_k = [&](int j) -> bool {
        const int i = j - jmin, st = i % kKStages;
        if (i >= kKStages && !all_wait(k_empty + 8 * st, (i / kKStages - 1) & 1, 1)) return false;
        scales(j, k_pages);
        store(k_ptr + st * kKBytes, kbuf);
        if (lane == 0) bar_arrive(k_full + 8 * st);
        k_pages = next;
        next = page_of(j + 2);
        fetch(p.k_pages, kbuf, j + 1, k_pages);
        return true;
      };
      bool ok = put_k(jmin);
      for (int j = jmin; j < nmax && ok; ++j) {
        const int i = j - jmin, vs = i % kVStages, vu = i / kVStages;
        const int following = k_pages;                     // (of tile j + 1)
        if (j + 1 < nmax && !put_k(j + 1)) break;
        if (i >= kVStages && !all_wait(v_empty + 8 * vs, (vu - 1) & 1, 9)) break;
        if (hides(j)) {
          bool found = false;
#pragma unroll
          for (int e = 0; e < kLoads; ++e) found |= any_not_finite<uint8_t>(vbuf[e]);
          if (found) bad[0] = 1;                           // (the issuing warps' cue)
        }
        store(v_ptr + vs * kKBytes, vbuf);
        if (lane == 0) bar_arrive(v_full + 8 * vs);
        v_pages = following;
        fetch(p.v_pages, vbuf, j + 1, v_pages);
      }
    }
  }

  // ---------------- teardown ----------------
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    const unsigned long long t0 = gtimer();
    while (gtimer() - t0 < 2000000ull) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

template <typename T, bool EIGHT, int D> int launch_prompt(const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv, const PromptParams &p, dim3 grid, cudaStream_t st) {
  using Smem = PromptSmem<D, EIGHT>;
  static_assert(Smem::kTotal <= 227 * 1024, "shared memory");
  auto kern = paged_prompt_kernel<T, EIGHT, D>;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Smem::kTotal) != cudaSuccess) {
      cudaGetLastError();
      return fail(EB_ECUDA, "paged_attention: cannot reserve %zu bytes of shared memory", Smem::kTotal);
    }
    cudaFuncAttributes attr{};
    if (cudaFuncGetAttributes(&attr, kern) != cudaSuccess || attr.numRegs != (EIGHT ? 128 : 168)) {
      cudaGetLastError();
      return fail(EB_EUNSUPPORTED, "paged_attention: the kernel was built with %d registers, its roles share out %d", attr.numRegs, EIGHT ? 128 : 168);
    }
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  launch_pdl(kern, grid, dim3(Smem::kThreads), Smem::kTotal, st, mq, mk, mv, p);
  return check_launch("paged_attention");
}

}  // namespace

int paged_tc_status(int *out4, bool clear) { return tc_status(out4, clear); }

PromptPlan prompt_plan(int batch, int kv_heads, int rows_per_head, long long keys) {
  PromptPlan s;
  s.blocks = (rows_per_head + kCtaRows - 1) / kCtaRows;
  const long long ctas = (long long)batch * kv_heads * s.blocks;
  const int tiles = (int)((keys + 2 * kKeys - 2) / kKeys);                 // (the first tile may begin in front of the first key)
  int splits = (int)(sm_count() / ctas);                                   // what one wave has room for, of at least eight tiles each
  if (splits > tiles / 8) splits = tiles / 8;
  if (splits < 1) splits = 1;
  s.split_tiles = (tiles + splits - 1) / splits;
  s.splits = (tiles + s.split_tiles - 1) / s.split_tiles;
  if (s.splits < 1) s.splits = 1;
  return s;
}

int paged_prompt(PromptParams p, const PromptPlan &s, int head_dim, int dtype, cudaStream_t st) {
  const bool eight = p.k_scale != nullptr;
  CUtensorMap mq{}, mk{}, mv{};
  p.q_tma = kRows % p.group == 0;
  if (p.q_tma) {
    EncodeFn fn = tc_encode_fn();
    if (!fn) return fail(EB_ECUDA, "tensor map: cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[4] = {(cuuint64_t)head_dim, (cuuint64_t)p.group, (cuuint64_t)p.kv_heads, (cuuint64_t)p.batch.rows};
    const cuuint64_t strides[3] = {(cuuint64_t)head_dim * 2, (cuuint64_t)p.group * head_dim * 2, (cuuint64_t)p.ldq * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)p.group, 1, (cuuint32_t)(kRows / p.group)}, ones[4] = {1, 1, 1, 1};
    const CUresult r = fn(&mq, dtype == EB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void *>(p.q), dims, strides, box, ones,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(EB_ECUDA, "tensor map: cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
  }
  if (!eight) {
    const long long blocks = (long long)p.batch.pages * p.kv_heads, page = 1ll << p.batch.page_shift;
    if (blocks >= (1ll << 31)) return fail(EB_EUNSUPPORTED, "paged_attention: %lld blocks exceed the tensor map", blocks);
    if (int rc = tc_map3(&mk, p.k_pages, dtype, head_dim, page, blocks, head_dim, page * head_dim, (int)page)) return rc;
    if (int rc = tc_map3(&mv, p.v_pages, dtype, head_dim, page, blocks, head_dim, page * head_dim, (int)page)) return rc;
  }
  p.splits = s.splits;
  p.split_tiles = s.split_tiles;
  const dim3 grid(s.blocks * s.splits, p.kv_heads, p.batch.batch);
#define EB_PROMPT(T, E) (head_dim == 64 ? launch_prompt<T, E, 64>(mq, mk, mv, p, grid, st) : launch_prompt<T, E, 128>(mq, mk, mv, p, grid, st))
  if (dtype == EB_F16) return eight ? EB_PROMPT(__half, true) : EB_PROMPT(__half, false);
  return eight ? EB_PROMPT(__nv_bfloat16, true) : EB_PROMPT(__nv_bfloat16, false);
#undef EB_PROMPT
}

}  // namespace eb
