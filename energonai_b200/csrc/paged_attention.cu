// Attention of few new tokens per sequence over a paged cache (generation steps, draft tokens): one pass over the keys and
// values, 16-bit or e4m3 codes with a scale for each page and head.  Bound by memory: a cached byte is asked for
// once per key / value head and tile of 8 or 16 query rows (token, head of the group); up to one tile that is once for all heads that share it, 17 to 24
// rows are three tiles, of which the second-level cache serves two.
//
// Both products are mma.sync tiles with the cached rows on the long side: S^T = K Q^T (16 keys x 8 query rows) and
// O^T += V^T P^T (16 dimensions x 8 query rows), so that 8 query rows (token, head of the group) fill a tile.  A warp takes
// 16 keys at a time, which lie in one page, through a small ring of tiles of its own in shared memory (asynchronous copies of 16 bytes, no
// barrier between warps, 16 warps per multiprocessor).  The contraction of S runs over dimensions in any order and that of O
// over keys in any order, so each lane reads 16 bytes where they lie, as the fragments of the products need them, and the queries
// are laid out to match; the chunks are swizzled so that these reads meet in no bank.  P^T comes from S^T by an 8 x 8
// transpose within the warp.  Tried and slower, for 64 sequences of 2048 to 4095 keys in e4m3, 8 heads of 128 (76 us then, 81 now): keys and values straight to
// registers, one tile ahead (88 us); bulk copies into unswizzled rings, twice as deep with 12 warps (93 us).
//
// e4m3 codes become fp16 (exact), whatever the model's type: queries of bf16 models go to fp16 with a power of two per
// row, which keeps all their bits.  A page's key scale multiplies its scores; the value scale z is added to the exponent,
// 2^(s + log2 z - m), so that fp16 weights keep their precision where pages differ in magnitude, and taken out of the sum again.
//
// The reference m of a row is raised only when a score exceeds it by 2^8 (one vote per tile instead of a reduction); fp16
// weights are 2^6 times as large, up to 2^14, which leaves fewer of them below fp16's normal range.
// Weights of bf16 caches are split into two bf16 pieces, which costs tensor time that is there and keeps
// the result within its own rounding; fp16 weights (of fp16 caches and of codes) are rounded once, 2^-11.
//
// Keys are split over CTAs by a fixed number of keys per CTA (short sequences then take fewer CTAs), the warps of a
// CTA take every fourth tile; partial rows are merged in order, across CTAs by a second launch.
#include <type_traits>

#include "attention_mma.cuh"
#include "paged_prompt.cuh"

namespace eb {
namespace {

constexpr int kStepWarps = 4;
constexpr float kLog2eStep = 1.4426950408889634f;
constexpr float kGrow = 8.f, kLiftHalf = 6.f;

struct StepParams {
  PagedBatch batch;
  const void *q;
  void *o;
  long long ldq, ldo;
  const void *k_pages, *v_pages;
  const float *k_scale, *v_scale;
  int kv_heads, group, window, few;      // few: sequences with more rows (tokens x group) than this are left to the prompt kernel
  int row_tiles, tile_rows, chunk;       // tiles of query rows, rows of a tile (of the largest one), keys per CTA
  float scale_log2;
  float *part;                           // [batch][kv_heads][row tiles][splits][rows][D + 2], or null: one split
  int splits;
};

__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
template <typename T> __device__ __forceinline__ void mma_tile(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Keys that the query rows of a tile see: [lo, hi), and the rows' own limits.
struct StepTile {
  int rows, past, lo, hi;
};
__device__ __forceinline__ StepTile step_tile(const StepParams &p, const PagedRows &r, int rt, int tile_rows) {
  StepTile t;
  const int all = r.count * p.group;
  t.rows = min(tile_rows, all - rt * tile_rows);
  t.past = r.past;
  const int first = r.past + rt * tile_rows / p.group, last = r.past + (rt * tile_rows + t.rows - 1) / p.group;
  t.hi = min(last + 1, p.batch.table_cols << p.batch.page_shift);
  t.lo = p.window > 0 ? max(0, first - p.window + 1) : 0;
  return t;
}
// whether one of the 16 keys from key0 on is seen by some only of the rows at the positions from `first` to `last`
__device__ __forceinline__ bool step_hides(int first, int last, int key0, int window) { return key0 + 15 > first || (window > 0 && key0 <= last - window); }

// The values that are not finite of a warp's tiles (from key0 on, every kStepWarps-th), each added to the partial rows that see it; V: the values' type, or
// uint8_t for codes.
template <typename V> __device__ __noinline__ void add_not_finite(const PagedBatch batch, const uint8_t *values, long long page_bytes, int b, int key0, int hi, const StepTile t, int row0,
                                                                  int group, int window, int dim, float *rows) {
  constexpr bool kCodes = std::is_same<V, uint8_t>::value;
  __syncwarp();
  for (; key0 < hi; key0 += kStepWarps * 16) {
    const int id = paged_page(batch, b, key0 >> batch.page_shift);
    if (id < 0 || !step_hides(t.past + row0 / group, t.past + (row0 + t.rows - 1) / group, key0, window)) continue;
    for (int key = max(key0, t.lo); key < min(key0 + 16, hi); ++key) {
      const V *y = reinterpret_cast<const V *>(values + id * page_bytes) + (key & ((1 << batch.page_shift) - 1)) * dim;
      for (int d = threadIdx.x & 31; d < dim; d += 32) {
        float v;
        if constexpr (kCodes) v = unpack2<__half>(e4m3x2_to_half2(y[d])).x;
        else v = to_f32<V>(y[d]);
        if (isfinite(v)) continue;
        for (int row = 0; row < t.rows; ++row) {
          const int pos = t.past + (row0 + row) / group;
          if (key <= pos && (window == 0 || key > pos - window)) rows[row * (dim + 2) + d] += v;
        }
      }
    }
  }
}

// T: type of queries and output; EIGHT: e4m3 pages; NT: tiles of 8 query rows; SPREAD: a tile's rows may be at several positions
template <bool EIGHT, int D, int NT> struct StepShape {
  static constexpr int kCtas = D == 64 ? (NT == 1 ? 4 : 3) : NT == 1 ? (EIGHT ? 4 : 3) : 2;      // resident per multiprocessor
};
template <typename T, bool EIGHT, int D, int NT, int STAGES, bool SPREAD>
__global__ void __launch_bounds__(kStepWarps * 32, StepShape<EIGHT, D, NT>::kCtas) paged_step_kernel(const StepParams p) {
  using M = typename std::conditional<EIGHT, __half, T>::type;           // operand type of the products
  constexpr bool kSplitP = std::is_same<M, __nv_bfloat16>::value;
  constexpr float kLift = kSplitP ? 0.f : kLiftHalf;
  constexpr int kRowsT = 8 * NT, kTiles = D / 16;
  constexpr int kKeyRegs = EIGHT ? D / 16 : D / 8;                       // registers per lane and key row
  constexpr int kValRegs = EIGHT ? D / 32 : D / 16;                      // ... and value row
  extern __shared__ __align__(128) uint8_t smem[];
  float (*red)[kRowsT][D + 2] = reinterpret_cast<float (*)[kRowsT][D + 2]>(smem);      // behind the key loop: [warps][rows][D + 2]
  griddep_wait();
  griddep_launch();
  const int split = blockIdx.x, hk = blockIdx.y / p.row_tiles, rt = blockIdx.y % p.row_tiles, b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const PagedRows r = paged_rows(p.batch, b);
  if (p.batch.clear) {
    paged_clear_ends(p.batch, reinterpret_cast<T *>(p.o), p.ldo, p.kv_heads * p.group * D);
    if (split == 0 && rt == 0) paged_clear(r, reinterpret_cast<T *>(p.o), p.ldo, hk * p.group * D, p.group * D, threadIdx.x, kStepWarps * 32);
  }
  if (r.count * p.group > p.few || rt * kRowsT >= r.count * p.group) return;
  const StepTile t = step_tile(p, r, rt, kRowsT);
  const int lo = (t.lo & ~15) + split * p.chunk, hi = split == p.splits - 1 ? t.hi : min(t.hi, lo + p.chunk);
  if (split > 0 && lo >= hi) return;

  constexpr int kRowBytes = EIGHT ? D : 2 * D, kChunks = kRowBytes / 16, kHalf = 16 * kRowBytes, kTile = 2 * kHalf;
  const long long block_bytes = (long long)kRowBytes << p.batch.page_shift;
  const uint8_t *kp = reinterpret_cast<const uint8_t *>(p.k_pages), *vp = reinterpret_cast<const uint8_t *>(p.v_pages);
  const int blocks = hi > lo ? (hi - lo + 15) / 16 : 0, mine = blocks > warp ? (blocks - warp + kStepWarps - 1) / kStepWarps : 0;
  // lane l holds the page of this warp's tile 32 n + l (and its scales), and of the next 32
  struct Ids {
    int id;
    float ks, vs;
  };
  auto fetch_ids = [&](int i0) {
    Ids x{-1, 1.f, 1.f};
    if (i0 + lane < mine) x.id = paged_page(p.batch, b, (lo + (warp + (i0 + lane) * kStepWarps) * 16) >> p.batch.page_shift);
    if (EIGHT && x.id >= 0) {
      x.ks = p.k_scale[(long long)x.id * p.kv_heads + hk];
      x.vs = fmaxf(p.v_scale[(long long)x.id * p.kv_heads + hk], kLeastScale);
    }
    return x;
  };
  Ids ids = fetch_ids(0), ids_next = fetch_ids(32);
  // The warp's ring of tiles.  Chunks of 16 bytes are swizzled so that neither the keys' reads (rows g, chunks c + 4 j) nor the values'
  // (rows 2 c + h, chunks g) meet in a bank.
  uint8_t *ring = smem + warp * STAGES * kTile;
  const uint32_t ring_at = smem_u32(ring);
  auto swizzle = [](int row) { return kChunks >= 8 ? ((row >> 1) & 3) << 1 ^ (row & 1) << 2 : (row >> 1) & 3; };
  // tile i of this warp, whose page is held by lane i mod 32 of `from` (a page that is none: nothing is requested)
  auto request = [&](int i, int id) {
    if (i < mine && id >= 0) {
      const int key = lo + (warp + i * kStepWarps) * 16;
      const long long at = ((long long)id * p.kv_heads + hk) * block_bytes + (key & ((1 << p.batch.page_shift) - 1)) * kRowBytes + lane * 16;
      const uint32_t to = ring_at + (i % STAGES) * kTile;
#pragma unroll
      for (int n = 0; n < kHalf / 512; ++n) {
        const int row = (n * 32 + lane) / kChunks, chunk = (n * 32 + lane) % kChunks;
        const uint32_t off = row * kRowBytes + (chunk ^ swizzle(row)) * 16;
        cp_async16(to + off, kp + at + n * 512, true);
        cp_async16(to + kHalf + off, vp + at + n * 512, true);
      }
    }
    cp_async_commit();
  };
  auto id_of = [&](int i, int base) {                      // page of tile i, with the windows that begin at tile `base`
    const int x = __shfl_sync(0xffffffffu, ids.id, i & 31), y = __shfl_sync(0xffffffffu, ids_next.id, i & 31);
    return i - base < 32 ? x : y;
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) request(i, id_of(i, 0));

  // ---- queries: fragments of the second operand, k index permuted like the keys ----
  uint32_t qf[NT][kTiles][2];
  float factor[NT][2];                                                   // exponent of a score, for the two query rows of this lane
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int row = rt * kRowsT + n * 8 + g, tok = row / p.group, head = hk * p.group + row % p.group;
    const bool there = n * 8 + g < t.rows;
    const T *q = reinterpret_cast<const T *>(p.q) + (long long)(r.row0 + tok) * p.ldq + (long long)head * D;
    float row_factor = p.scale_log2;
    // chunk j of 16 bytes of codes (16 dimensions) or of 16-bit values (8), taken by lane c as chunk c + 4 j
    constexpr int kPer = EIGHT ? 16 : 8, kChunks = D / kPer / 4;
    uint4 raw[kTiles / 2];
#pragma unroll
    for (int j = 0; j < kChunks; ++j)
#pragma unroll
      for (int i = 0; i < kPer / 8; ++i)
        raw[j * (kPer / 8) + i] = there ? *reinterpret_cast<const uint4 *>(q + (c + 4 * j) * kPer + i * 8) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < kTiles / 2; ++i) {
      qf[n][2 * i][0] = raw[i].x;
      qf[n][2 * i][1] = raw[i].y;
      qf[n][2 * i + 1][0] = raw[i].z;
      qf[n][2 * i + 1][1] = raw[i].w;
    }
    if constexpr (EIGHT && std::is_same<T, __nv_bfloat16>::value) {
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 f = unpack2<__nv_bfloat16>(qf[n][i][e]);
          m = fmaxf(m, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
      // the largest magnitude to [2^14, 2^15): what falls out of fp16's range below is 2^-38 of it
      const int e = min(max(14 - ((__float_as_int(m) >> 23) - 127), -100), 100);
      const float up = __int_as_float((127 + e) << 23);
      row_factor *= __int_as_float((127 - e) << 23);
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float2 f = unpack2<__nv_bfloat16>(qf[n][i][k]);
          qf[n][i][k] = pack2<__half>(f.x * up, f.y * up);
        }
    }
    factor[n][0] = __shfl_sync(0xffffffffu, row_factor, 8 * c);          // (row 2c is held by lanes 8c .. 8c + 3)
    factor[n][1] = __shfl_sync(0xffffffffu, row_factor, 8 * c + 4);
  }
  int row_pos[NT][2];                                                    // position of the two query rows
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) row_pos[n][e] = t.past + (rt * kRowsT + n * 8 + 2 * c + e) / p.group;
  const int first_pos = t.past + rt * kRowsT / p.group, last_pos = t.past + (rt * kRowsT + t.rows - 1) / p.group;
  using V = typename std::conditional<EIGHT, uint8_t, T>::type;
  bool taken = false;                                                    // values that are not finite were taken out of a tile

  float acc[NT][kTiles][4], m_ref[NT][2], l_run[NT][2], far_below = -3.402823466e38f;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m_ref[n][0] = m_ref[n][1] = -3.402823466e38f;
    l_run[n][0] = l_run[n][1] = 0.f;
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][i][e] = 0.f;
  }

  for (int i = 0; i < mine; ++i) {
    const int key0 = lo + (warp + i * kStepWarps) * 16;
    if (i > 0 && (i & 31) == 0) {
      ids = ids_next;
      ids_next = fetch_ids(i + 32);
    }
    const int id = __shfl_sync(0xffffffffu, ids.id, i & 31);
    const float ks = EIGHT ? __shfl_sync(0xffffffffu, ids.ks, i & 31) : 1.f, vs = EIGHT ? __shfl_sync(0xffffffffu, ids.vs, i & 31) : 1.f;
    cp_async_wait<STAGES - 2>();
    __syncwarp();                                          // (tile i is there, and all lanes have read tile i - 1, whose memory the next request takes)
    request(i + STAGES - 1, id_of(i + STAGES - 1, i & ~31));
    if (id < 0) continue;                                  // (a page that is none: nothing to see)
    const uint8_t *tile = ring + (i % STAGES) * kTile;
    // A weight of 0 does not hide a value that is not finite: tokens further on in the call, or keys that a window left behind, may hold such for rows
    // that do not see them.  They leave the tile here, and are added behind the loop to the rows that do.  (In front of the scores, so that the
    // values' loads need not wait for what is stored here.)
    if (SPREAD && step_hides(first_pos, last_pos, key0, p.window)) {
      bool found = false;
#pragma unroll 1
      for (int n = 0; n < kHalf / 512; ++n) {
        const int key = key0 + (n * 32 + lane) / kChunks;
        if (key < hi && key >= t.lo) found |= any_not_finite<V>(*reinterpret_cast<const uint4 *>(tile + kHalf + (n * 32 + lane) * 16));
      }
      if (__builtin_expect(__any_sync(0xffffffffu, found), 0)) {
        taken = true;
#pragma unroll 1
        for (int n = 0; n < kHalf / 512; ++n) {
          uint4 *x = reinterpret_cast<uint4 *>(ring + (i % STAGES) * kTile + kHalf + (n * 32 + lane) * 16);
          *x = finite_only<V>(*x);
        }
        __syncwarp();
      }
    }
    // ---- scores ----
    float s[NT][4], s2[NT][4];                             // (two chains of dependent products)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = s2[n][e] = 0.f;
#pragma unroll
    for (int j = 0; j < kKeyRegs / 4; ++j) {
      const uint4 x = *reinterpret_cast<const uint4 *>(tile + g * kRowBytes + ((c + 4 * j) ^ swizzle(g)) * 16), y = *reinterpret_cast<const uint4 *>(tile + (g + 8) * kRowBytes + ((c + 4 * j) ^ swizzle(g)) * 16);
      const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
      if constexpr (EIGHT) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t a0 = e4m3x2_to_half2(xs[w]), a1 = e4m3x2_to_half2(ys[w]), a2 = e4m3x2_to_half2(xs[w] >> 16), a3 = e4m3x2_to_half2(ys[w] >> 16);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_tile<M>((w & 1) ? s2[n] : s[n], a0, a1, a2, a3, qf[n][4 * j + w][0], qf[n][4 * j + w][1]);
        }
      } else {
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_tile<M>((w & 1) ? s2[n] : s[n], xs[2 * w], ys[2 * w], xs[2 * w + 1], ys[2 * w + 1], qf[n][2 * j + w][0], qf[n][2 * j + w][1]);
      }
    }
    const float v_log = EIGHT ? __log2f(vs) : 0.f, v_inv = EIGHT ? 1.f / vs : 1.f;
    const bool whole = key0 + 16 <= min(hi, first_pos + 1) && key0 >= t.lo && (p.window == 0 || key0 > last_pos - p.window);
    bool grows = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = s[n][e] + s2[n][e];
        float v = EIGHT ? fmaf(x, factor[n][e & 1] * ks, v_log) : x * factor[n][e & 1];
        if (!whole) {
          const int key = key0 + g + (e >> 1) * 8, pos = row_pos[n][e & 1];
          if (key >= hi || key > pos || (p.window > 0 && key <= pos - p.window)) v = -INFINITY;
        }
        s[n][e] = v;
        grows |= v > m_ref[n][e & 1] + kGrow;
      }
    if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float m = fmaxf(m_ref[n][e], fmaxf(s[n][e], s[n][e + 2]));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
          const float alpha = pow2(m_ref[n][e] - m);
          l_run[n][e] = EIGHT ? sum_at(l_run[n][e], m_ref[n][e] - m) : l_run[n][e] * alpha;
          m_ref[n][e] = m;
          if (EIGHT) far_below = fmaxf(far_below, m - kFarBelow);
#pragma unroll
          for (int k = 0; k < kTiles; ++k) {
            acc[n][k][e] *= alpha;
            acc[n][k][e + 2] *= alpha;
          }
        }
    }
    if (EIGHT && __builtin_expect(v_log < far_below, 0)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = s[n][e] - (m_ref[n][e & 1] - kLift);
          if (x < kLeastPower) l_run[n][e & 1] += pow2(x - v_log);
        }
    }
    uint32_t pf[NT][2], pl[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float w0 = pow2(s[n][2 * h] - (m_ref[n][0] - kLift)), w1 = pow2(s[n][2 * h + 1] - (m_ref[n][1] - kLift));
        const uint32_t w = pack2<M>(w0, w1);
        const float2 rounded = unpack2<M>(w);
        pf[n][h] = transposed(w);
        if constexpr (kSplitP) pl[n][h] = transposed(pack2<M>(w0 - rounded.x, w1 - rounded.y));
        // fp16 weights of 16-bit pages are summed as they are rounded, which takes a tenth off the error.  Not those of codes: weights of a page
        // whose values are far smaller than another's fall below fp16, where they add nothing to the values, but they count in the sum.
        constexpr bool kAsRounded = !EIGHT && !kSplitP;
        l_run[n][0] = fmaf(kAsRounded ? rounded.x : w0, v_inv, l_run[n][0]);
        l_run[n][1] = fmaf(kAsRounded ? rounded.y : w1, v_inv, l_run[n][1]);
      }
    // ---- O^T += V^T P^T: value rows 2c, 2c + 1, 2c + 8, 2c + 9, dimensions by g ----
    const bool edge = key0 + 16 > hi || key0 < t.lo;
    constexpr int kPart = kValRegs < 4 ? kValRegs : 4;   // registers of a row at a time
#pragma unroll
    for (int j = 0; j < kValRegs / kPart; ++j) {
      uint32_t vr[4][kPart];
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int row = 2 * c + (h & 1) + (h >> 1) * 8;
        const uint8_t *y = tile + kHalf + row * kRowBytes + (kPart == 2 ? ((g >> 1) ^ swizzle(row)) * 16 + (g & 1) * 8 : ((8 * j + g) ^ swizzle(row)) * 16);
        if constexpr (kPart == 2) {
          const uint2 w = *reinterpret_cast<const uint2 *>(y);
          vr[h][0] = w.x;
          vr[h][1] = w.y;
        } else {
          const uint4 w = *reinterpret_cast<const uint4 *>(y);
          vr[h][0] = w.x;
          vr[h][1] = w.y;
          vr[h][2] = w.z;
          vr[h][3] = w.w;
        }
        // value rows that no query row of the tile sees may hold anything
        if (edge && (key0 + row >= hi || key0 + row < t.lo)) {
#pragma unroll
          for (int e = 0; e < kPart; ++e) vr[h][e] = 0;
        }
      }
#pragma unroll
      for (int q = 0; q < (EIGHT ? 2 * kPart : kPart); ++q) {
        const int k = j * (EIGHT ? 2 * kPart : kPart) + q;
        uint32_t a0, a1, a2, a3;
        if constexpr (EIGHT) {
          // bytes 2 (q % 2) and the next of word q / 2: two dimensions of four keys
          const uint32_t sel = (q & 1) ? 0x7362 : 0x5140;
          const uint32_t x = __byte_perm(vr[0][q / 2], vr[1][q / 2], sel), y = __byte_perm(vr[2][q / 2], vr[3][q / 2], sel);
          a0 = e4m3x2_to_half2(x);
          a1 = e4m3x2_to_half2(x >> 16);
          a2 = e4m3x2_to_half2(y);
          a3 = e4m3x2_to_half2(y >> 16);
        } else {
          a0 = __byte_perm(vr[0][q], vr[1][q], 0x5410);
          a1 = __byte_perm(vr[0][q], vr[1][q], 0x7632);
          a2 = __byte_perm(vr[2][q], vr[3][q], 0x5410);
          a3 = __byte_perm(vr[2][q], vr[3][q], 0x7632);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_tile<M>(acc[n][k], a0, a1, a2, a3, pf[n][0], pf[n][1]);
          if constexpr (kSplitP) mma_tile<M>(acc[n][k], a0, a1, a2, a3, pl[n][0], pl[n][1]);
        }
      }
    }
  }
  __syncthreads();                                         // (the rings' memory holds the partial rows from here on)

  // ---- the warps' partial rows ----
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float l = l_run[n][e];
      l += __shfl_xor_sync(0xffffffffu, l, 4);
      l += __shfl_xor_sync(0xffffffffu, l, 8);
      l += __shfl_xor_sync(0xffffffffu, l, 16);
      float *row = red[warp][n * 8 + 2 * c + e];
#pragma unroll
      for (int k = 0; k < kTiles; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // tile k of e4m3 rows: dimensions (D / 8) g + 2 k + h; of 16-bit rows: 8 g + 2 (k % 4) + h of half k / 4
          const int d = EIGHT ? D / 8 * g + 2 * k + h : k / 4 * 64 + 8 * g + 2 * (k % 4) + h;
          row[d] = acc[n][k][e + 2 * h];
        }
      if (g == 0) {
        row[D] = m_ref[n][e];
        row[D + 1] = l;
      }
    }
  if (SPREAD && __builtin_expect(taken, 0))
    add_not_finite<V>(p.batch, vp + hk * block_bytes, p.kv_heads * block_bytes, b, lo + warp * 16, hi, t, rt * kRowsT, p.group, p.window, D, &red[warp][0][0]);
  __syncthreads();
  // two columns of a row, of this CTA's warps
  struct Sum {
    float m, l, x, y;
  };
  auto of_warps = [&](int row, int d) {
    Sum r{red[0][row][D], 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 1; w < kStepWarps; ++w) r.m = fmaxf(r.m, red[w][row][D]);
#pragma unroll
    for (int w = 0; w < kStepWarps; ++w) {
      const float a = pow2(red[w][row][D] - r.m);
      r.l = EIGHT ? r.l + sum_at(red[w][row][D + 1], red[w][row][D] - r.m) : fmaf(red[w][row][D + 1], a, r.l);
      r.x = fmaf(red[w][row][d], a, r.x);
      r.y = fmaf(red[w][row][d + 1], a, r.y);
    }
    return r;
  };
  auto write = [&](int row, int d, const Sum &v) {
    const int all = rt * kRowsT + row;
    T *out = reinterpret_cast<T *>(p.o) + (long long)(r.row0 + all / p.group) * p.ldo + (long long)(hk * p.group + all % p.group) * D + d;
    const float inv = v.l == 0.f ? 0.f : 1.f / v.l;
    *reinterpret_cast<uint32_t *>(out) = pack2<T>(v.x * inv, v.y * inv);
  };
  for (int i = threadIdx.x; i < t.rows * (D / 2); i += kStepWarps * 32) {
    const int row = i / (D / 2), d = 2 * (i % (D / 2));
    const Sum v = of_warps(row, d);
    if (p.part) {
      float *out = p.part + ((((long long)b * p.kv_heads + hk) * p.row_tiles + rt) * p.splits + split) * kRowsT * (D + 2) + row * (D + 2);
      *reinterpret_cast<float2 *>(out + d) = make_float2(v.x, v.y);
      if (d == 0) *reinterpret_cast<float2 *>(out + D) = make_float2(v.m, v.l);
    } else {
      write(row, d, v);
    }
  }
}

// A row of the output from its splits (D values, maximum, sum; `stride` floats apart) by the four warps of a CTA: each adds up
// every fourth split, in order, then the warps' sums are added in order.
constexpr int kMergeWarps = 4;
template <typename T, int D> __device__ __forceinline__ void merge_row(const float *in, int stride, int splits, T *out) {
  constexpr int kPer = D / 32;
  __shared__ float sums[kMergeWarps][D + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float m = -3.402823466e38f, l = 0.f, x[kPer];
  for (int s = lane; s < splits; s += 32) m = fmaxf(m, in[(long long)s * stride + D]);
  m = warp_max(m);
#pragma unroll
  for (int e = 0; e < kPer; ++e) x[e] = 0.f;
#pragma unroll 8
  for (int s = warp; s < splits; s += kMergeWarps) {
    const float *one = in + (long long)s * stride;
    const float2 ml = *reinterpret_cast<const float2 *>(one + D);
    const float a = pow2(ml.x - m);
    l += sum_at(ml.y, ml.x - m);
#pragma unroll
    for (int e = 0; e < kPer; e += 2) {
      const float2 v = *reinterpret_cast<const float2 *>(one + lane * kPer + e);
      x[e] = fmaf(v.x, a, x[e]);
      x[e + 1] = fmaf(v.y, a, x[e + 1]);
    }
  }
#pragma unroll
  for (int e = 0; e < kPer; ++e) sums[warp][lane * kPer + e] = x[e];
  if (lane == 0) sums[warp][D] = l;
  __syncthreads();
  if (threadIdx.x < D / 2) {
    float y0 = 0.f, y1 = 0.f, all = 0.f;
#pragma unroll
    for (int w = 0; w < kMergeWarps; ++w) {
      y0 += sums[w][2 * threadIdx.x];
      y1 += sums[w][2 * threadIdx.x + 1];
      all += sums[w][D];
    }
    const float inv = all == 0.f ? 0.f : 1.f / all;
    *reinterpret_cast<uint32_t *>(out + 2 * threadIdx.x) = pack2<T>(y0 * inv, y1 * inv);
  }
}

template <typename T, int D, int NT> __global__ void __launch_bounds__(128) paged_merge_kernel(const StepParams p) {
  constexpr int kRowsT = 8 * NT;
  griddep_wait();
  griddep_launch();
  const int hk = blockIdx.y / p.row_tiles, rt = blockIdx.y % p.row_tiles, b = blockIdx.z, row = blockIdx.x;
  const PagedRows r = paged_rows(p.batch, b);
  if (r.count * p.group > p.few || rt * kRowsT >= r.count * p.group) return;
  const StepTile t = step_tile(p, r, rt, kRowsT);
  if (row >= t.rows) return;
  const int splits = min(p.splits, max(1, (t.hi - (t.lo & ~15) + p.chunk - 1) / p.chunk)), all = rt * kRowsT + row;
  const float *in = p.part + (((long long)b * p.kv_heads + hk) * p.row_tiles + rt) * p.splits * kRowsT * (D + 2) + row * (D + 2);
  merge_row<T, D>(in, kRowsT * (D + 2), splits,
                  reinterpret_cast<T *>(p.o) + (long long)(r.row0 + all / p.group) * p.ldo + (long long)(hk * p.group + all % p.group) * D);
}

// The same for the prompt kernel's blocks of 256 rows.
template <typename T, int D> __global__ void __launch_bounds__(128) paged_prompt_merge_kernel(const PromptParams p, int blocks) {
  constexpr int kBlock = 256;
  griddep_wait();
  griddep_launch();
  const int hk = blockIdx.y, b = blockIdx.z, all = blockIdx.x, qb = all / kBlock;
  const PagedRows r = paged_rows(p.batch, b);
  const int count = r.count * p.group;
  if (count <= p.few || all >= count) return;
  // key tiles of the block's rows, as the prompt kernel counts them
  const int first = p.window > 0 ? max(0, r.past + qb * kBlock / p.group - p.window + 1) : 0,
            end = min(r.past + (min((qb + 1) * kBlock, count) - 1) / p.group + 1, p.batch.table_cols << p.batch.page_shift);
  const int splits = min(p.splits, max(1, ((end + 127) / 128 - first / 128 + p.split_tiles - 1) / p.split_tiles));
  const float *in = p.part + (((long long)b * p.kv_heads + hk) * blocks + qb) * p.splits * kBlock * (D + 2) + (long long)(all % kBlock) * (D + 2);
  merge_row<T, D>(in, kBlock * (D + 2), splits,
                  reinterpret_cast<T *>(p.o) + (long long)(r.row0 + all / p.group) * p.ldo + (long long)(hk * p.group + all % p.group) * D);
}

template <typename T, bool EIGHT, int D, int NT, bool SPREAD> int launch_step(const StepParams &p, cudaStream_t st) {
  constexpr int kTile = 16 * 2 * (EIGHT ? D : 2 * D), kRed = kStepWarps * 8 * NT * (D + 2) * 4;
  // (64 sequences of 2048 to 4095 keys in e4m3, heads of 128: 76 us with two tiles, 77 with three, 86 with four, which cost resident CTAs;
  // 32 of 1500, 16-bit heads of 64: 26, 23 and 23)
  constexpr int kStages = D == 64 ? 3 : 2, kSmem = kStepWarps * kStages * kTile > kRed ? kStepWarps * kStages * kTile : kRed;
  auto kern = paged_step_kernel<T, EIGHT, D, NT, kStages, SPREAD>;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (kSmem > 48 * 1024 && (dev < 0 || dev >= 64 || !configured[dev])) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess) {
      cudaGetLastError();
      return fail(EB_ECUDA, "paged_attention: cannot reserve %d bytes of shared memory", kSmem);
    }
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  launch_pdl(kern, dim3(p.splits, p.kv_heads * p.row_tiles, p.batch.batch), dim3(kStepWarps * 32), kSmem, st, p);
  if (p.part) launch_pdl(paged_merge_kernel<T, D, NT>, dim3(p.tile_rows, p.kv_heads * p.row_tiles, p.batch.batch), dim3(128), 0, st, p);
  return check_launch("paged_attention");
}

constexpr int kMostKeys = 8192, kLeastKeys = 256;
// What the partial rows of a call may take: as many sequences as a call brings may be long, and the tables may address more than any of them is.
// Fewer splits cost a long sequence among many more than the memory is worth (tables of 131072 positions, 32 heads on 8, 62 short sequences, one of
// 100,000 keys and a prompt chunk: 276 MB unbounded and with 256 MB 362 us, with 128 MB 462, with 64 MB 706, without splits 1262; 40 heads of 128
// sequences beside a chunk: 2762 MB 1411 us, with 256 MB, which leaves no splits, 1690).
constexpr size_t kMostPartial = (size_t)256 << 20;
// How the step form cuts a call: query rows per tile, tiles, keys per CTA, splits.
struct StepPlan {
  int tiles8, row_tiles, chunk, splits;
};
StepPlan step_plan(int batch, int kv_heads, int rows_per_head, long long keys, int head_dim, bool eight, bool beside) {
  StepPlan s;
  // Tiles of 16 rows read the keys half as often (128 heads on 8, 64 sequences of 2048 to 4095 keys: 108 us, with tiles of 8 125), but not where the
  // last one would be half empty (20 rows, 24 sequences, window 1024: 25 us, with three tiles of 8 21).
  s.tiles8 = rows_per_head > 8 && !(rows_per_head > 16 && rows_per_head <= 24) ? 2 : 1;
  s.row_tiles = (rows_per_head + 8 * s.tiles8 - 1) / (8 * s.tiles8);
  const long long units = (long long)batch * kv_heads * s.row_tiles, sms = sm_count();
  // CTAs that are resident at a time, as the launch bounds have it.  From half of them on there are no splits, fewer are split to fill
  // them once.  No CTA gets more than kMostKeys keys (a long sequence among short ones would keep the call waiting) nor fewer
  // than kLeastKeys.  Beside prompts, whose launch follows this one, there are splits only for the former: the plan does not know how many of
  // the sequences bring few rows.
  const long long slots = sms * (head_dim == 64 ? (s.tiles8 == 1 ? 4 : 3) : s.tiles8 == 1 ? (eight ? 4 : 3) : 2);
  const long long want = beside || 2 * units >= slots ? 1 : slots / units;
  keys += 15;                                               // (the first tile may begin in front of the first key)
  long long chunk = (keys + want - 1) / want;
  if (chunk > kMostKeys) chunk = kMostKeys;
  if (chunk < kLeastKeys) chunk = kLeastKeys;
  if (chunk < (keys + 511) / 512) chunk = (keys + 511) / 512;
  const long long most = (long long)(kMostPartial / ((size_t)batch * kv_heads * s.row_tiles * 8 * s.tiles8 * (head_dim + 2) * sizeof(float)));
  if (chunk * most < keys) chunk = most > 0 ? (keys + most - 1) / most : keys;
  chunk = (chunk + 63) / 64 * 64;
  s.splits = (int)((keys + chunk - 1) / chunk);
  s.chunk = (int)chunk;
  return s;
}
long long step_keys(long long most_length, int window, int most_new) {
  const long long seen = (long long)window + most_new;
  return window > 0 && seen < most_length ? seen : most_length;
}
size_t step_scratch(const StepPlan &s, int batch, int kv_heads, int head_dim) {
  return s.splits > 1 ? (size_t)batch * kv_heads * s.row_tiles * s.splits * 8 * s.tiles8 * (head_dim + 2) * sizeof(float) : 0;
}

// Sequences that bring at most so many rows (tokens x heads of a group) take the step kernel, the others the prompt kernel.
constexpr int kFewRows = 64;

struct PagedPlan {
  bool prompt;
  int step_rows;
  StepPlan step;
  PromptPlan tiles;
  size_t step_bytes, prompt_bytes;
};
PagedPlan paged_plan(int batch, int kv_heads, int group, int head_dim, bool eight, int most_new, int most_length, int window) {
  PagedPlan s{};
  const long long keys = step_keys(most_length, window, most_new);
  const int rows = most_new * group;
  s.prompt = rows > kFewRows;
  s.step_rows = s.prompt ? kFewRows : rows;
  s.step = step_plan(batch, kv_heads, s.step_rows, s.prompt ? step_keys(most_length, window, kFewRows) : keys, head_dim, eight, s.prompt);
  s.step_bytes = step_scratch(s.step, batch, kv_heads, head_dim);
  if (s.prompt) {
    // a block's keys with a window: its own rows' and the window in front
    s.tiles = prompt_plan(batch, kv_heads, rows, step_keys(most_length, window, 256 / group + 1));
    s.prompt_bytes = s.tiles.splits > 1 ? (size_t)batch * kv_heads * s.tiles.blocks * s.tiles.splits * 256 * (head_dim + 2) * sizeof(float) : 0;
  }
  return s;
}

template <typename T, int D> void launch_prompt_merge(const PromptParams &p, const PromptPlan &s, cudaStream_t st) {
  launch_pdl(paged_prompt_merge_kernel<T, D>, dim3(s.blocks * 256, p.kv_heads, p.batch.batch), dim3(128), 0, st, p, s.blocks);
}

}  // namespace
}  // namespace eb

using namespace eb;

extern "C" size_t eb_paged_attention_scratch_bytes(int batch, int heads, int kv_heads, int head_dim, int eight_bit, int most_new, int most_length, int window) {
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 || most_new <= 0 || most_length <= 0 || window < 0 || heads % kv_heads) return 0;
  if ((long long)most_new * (heads / kv_heads) >= (1 << 30)) return 0;
  const PagedPlan s = paged_plan(batch, kv_heads, heads / kv_heads, head_dim, eight_bit != 0, most_new, most_length, window);
  return s.step_bytes + s.prompt_bytes;
}

extern "C" int eb_paged_attention(const eb_paged *cache, const void *q, long long ldq, void *out, long long ldo, int rows, int heads, int window, float scale,
                                  void *scratch, size_t scratch_bytes, void *stream) {
  EB_REQUIRE(cache, "paged_attention: null pointer");
  const int batch = cache->batch, kv_heads = cache->kv_heads, head_dim = cache->head_dim, page_size = cache->page_size, dtype = cache->dtype,
            table_cols = cache->table_cols;
  int most_new = cache->most_new, most_length = cache->most_length;
  const void *k_pages = cache->k_pages, *v_pages = cache->v_pages;
  const float *k_scale = cache->k_scale, *v_scale = cache->v_scale;
  if (rows == 0 || batch == 0 || most_new == 0) return EB_OK;
  StepParams p{};
  if (int rc = paged_check("paged_attention", p.batch, *cache, rows)) return rc;
  EB_REQUIRE(dtype == EB_F16 || dtype == EB_BF16, "paged_attention: fp16 or bf16 only (dtype %d)", dtype);
  EB_REQUIRE(head_dim == 64 || head_dim == 128, "paged_attention: head_dim %d not supported (64 or 128)", head_dim);
  EB_REQUIRE(heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && (long long)heads * head_dim < (1 << 28), "paged_attention: %d heads do not share %d key / value heads", heads, kv_heads);
  EB_REQUIRE(q && out && k_pages && v_pages, "paged_attention: null pointer");
  EB_REQUIRE(!k_scale == !v_scale, "paged_attention: 8-bit pages have scales for keys and for values");
  EB_REQUIRE(most_new > 0 && most_length > 0 && window >= 0, "paged_attention: bad limits (most_new %d, most_length %d, window %d)", most_new, most_length, window);
  EB_REQUIRE(scale > 0.f, "paged_attention: the scale must be positive");
  EB_REQUIRE(ldq >= (long long)heads * head_dim && ldo >= (long long)heads * head_dim && ldq % 8 == 0 && ldo % 8 == 0,
             "paged_attention: row strides must be multiples of 8 elements that hold a row");
  EB_REQUIRE(aligned16(q) && aligned16(out) && aligned16(k_pages) && aligned16(v_pages), "paged_attention: pointers must be 16-byte aligned");
  if (most_new > rows) most_new = rows;
  const long long reach = (long long)table_cols * page_size;
  if (most_length > reach) most_length = (int)reach;
  const int group = heads / kv_heads;
  EB_REQUIRE((long long)most_new * group < (1 << 30), "paged_attention: too many rows");
  const PagedPlan plan = paged_plan(batch, kv_heads, group, head_dim, k_scale != nullptr, most_new, most_length, window);
  const StepPlan &s = plan.step;
  EB_REQUIRE((long long)kv_heads * s.row_tiles <= 65535, "paged_attention: %d heads exceed the grid", kv_heads);
  const size_t need = plan.step_bytes + plan.prompt_bytes;
  EB_REQUIRE(need == 0 || (scratch && aligned16(scratch) && scratch_bytes >= need), "paged_attention: %zu bytes of scratch needed, %zu given", need, scratch_bytes);
  p.q = q; p.o = out; p.ldq = ldq; p.ldo = ldo; p.k_pages = k_pages; p.v_pages = v_pages; p.k_scale = k_scale; p.v_scale = v_scale;
  p.kv_heads = kv_heads; p.group = group; p.window = window; p.few = kFewRows; p.row_tiles = s.row_tiles; p.tile_rows = plan.step_rows < 8 * s.tiles8 ? plan.step_rows : 8 * s.tiles8; p.chunk = s.chunk; p.splits = s.splits;
  p.scale_log2 = scale * kLog2eStep; p.part = plan.step_bytes ? reinterpret_cast<float *>(scratch) : nullptr;
  cudaStream_t st = as_stream(stream);
  int rc;
  // Single tokens take a kernel of their own: what rows at several positions need costs it 9 % (64 sequences of 2048 to 4095 keys in e4m3)
#define EB_STEP(T, E, D)                                                                                      \
  (most_new == 1 ? (s.tiles8 == 1 ? launch_step<T, E, D, 1, false>(p, st) : launch_step<T, E, D, 2, false>(p, st)) \
                 : (s.tiles8 == 1 ? launch_step<T, E, D, 1, true>(p, st) : launch_step<T, E, D, 2, true>(p, st)))
#define EB_STEP_D(T, E) (head_dim == 64 ? EB_STEP(T, E, 64) : EB_STEP(T, E, 128))
  if (dtype == EB_F16) rc = k_scale ? EB_STEP_D(__half, true) : EB_STEP_D(__half, false);
  else rc = k_scale ? EB_STEP_D(__nv_bfloat16, true) : EB_STEP_D(__nv_bfloat16, false);
#undef EB_STEP_D
#undef EB_STEP
  if (rc != EB_OK || !plan.prompt) return rc;
  PromptParams t{};
  t.batch = p.batch; t.q = q; t.o = out; t.ldq = ldq; t.ldo = ldo; t.k_pages = k_pages; t.v_pages = v_pages; t.k_scale = k_scale; t.v_scale = v_scale;
  t.kv_heads = kv_heads; t.group = group; t.window = window; t.few = kFewRows; t.scale_log2 = p.scale_log2;
  t.part = plan.prompt_bytes ? reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(scratch) + plan.step_bytes) : nullptr;
  t.splits = plan.tiles.splits; t.split_tiles = plan.tiles.split_tiles;
  if ((rc = paged_prompt(t, plan.tiles, head_dim, dtype, st)) != EB_OK || !t.part) return rc;
  if (dtype == EB_F16) head_dim == 64 ? launch_prompt_merge<__half, 64>(t, plan.tiles, st) : launch_prompt_merge<__half, 128>(t, plan.tiles, st);
  else head_dim == 64 ? launch_prompt_merge<__nv_bfloat16, 64>(t, plan.tiles, st) : launch_prompt_merge<__nv_bfloat16, 128>(t, plan.tiles, st);
  return check_launch("paged_attention");
}
