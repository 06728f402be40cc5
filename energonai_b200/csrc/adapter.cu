// Low-rank adapters of many requests: delta = s (x A^T) B^T, with the A [rank][width], B [columns][rank] and s of each
// sequence's adapter, for the rows of a packed batch.  In bf16 the projection beside it adds delta to its fp32 sums as a
// residual, so that the result is rounded once (and delta, the smaller part, before).  In fp16, whose range delta may leave where the sum does not,
// it is the other way around: the second launch takes the projection's fp32 sums and writes the result (4107 rows, 4096 -> 6144, rank 64: 232 us instead
// of 208 with a residual, and 0.6 of its error; 48 rows, 5120 -> 5120, rank 16: 35 us either way).  The first launch stays in front of the product, so that
// the GPU has it while the host prepares that.
//
// Two launches.  The first has x A^T: bound by reading x and the adapters that occur.  With up to 16 rows per sequence a CTA takes them and
// a part of the columns, its warps take slices of that part, and a lane loads 16 bytes of its row straight
// into the fragments of mma.sync (the contraction runs over columns in any order); the warps' sums meet in shared memory.  Longer sequences
// go 64 rows at a time through shared memory, or every 16 rows would read the adapter again.  Where the columns are split over CTAs,
// partial sums go to scratch, summed in order by the second launch.  That one has the
// product with B^T: bound by writing delta.  The low-rank row stays fp32 between the two and enters the product as two
// 16-bit pieces: it costs tensor time that is there, and no rounding.
#include <type_traits>

#include "attention_mma.cuh"

namespace eb {
namespace {

constexpr int kAdapterWarps = 4, kRowTile = 16;

struct AdapterParams {
  const void *x, *a, *b;
  const float *scales;
  const int *index, *starts;
  const float *base;                     // [rows][columns]: what delta is added to (or null)
  void *delta;
  float *low;                            // [splits][rows][rank]
  long long ldx, ldd, ldbase;
  int rows, width, columns, rank, count, batch, most_new, splits, per_split, chunk;   // per_split: columns of x per CTA; chunk: columns of delta per CTA
};

template <typename T> __device__ __forceinline__ void mma_low(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// two numbers as two 16-bit pieces each (an infinity is its first piece, and nothing is left of it)
template <typename T> __device__ __forceinline__ void two_pieces(float x, float y, uint32_t &hi, uint32_t &lo) {
  hi = pack2<T>(x, y);
  const float2 f = unpack2<T>(hi);
  lo = pack2<T>(x == f.x ? 0.f : x - f.x, y == f.y ? 0.f : y - f.y);
}

// fp16 pieces: the power of two that brings the largest magnitude m of a low-rank row to [2^14, 2^15), so that the row keeps its
// 22 bits whatever its size (from 2^-100 on); the products are divided by it in fp32.  bf16 has fp32's range, but for what rounds up
// beyond its largest number.
template <typename T> __device__ __forceinline__ int lift_of(float m) {
  const int e = (__float_as_int(m) >> 23) - 127;
  return std::is_same<T, __half>::value ? min(max(14 - e, -113), 100) : e > 126 ? -1 : 0;
}
__device__ __forceinline__ float pow2_of(int e) { return __int_as_float((127 + e) << 23); }
__device__ __forceinline__ float largest_of(const float4 &v) { return fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))); }

// Rows and adapter of sequence b, which serves `live` of them, the announced ones.
struct AdapterRows {
  int row0, count, live, adapter;
};
__device__ __forceinline__ AdapterRows adapter_rows(const AdapterParams &p, int b) {
  AdapterRows r;
  r.row0 = min(max(p.starts[b], 0), p.rows);
  r.count = min(p.starts[b + 1], p.rows) - r.row0;
  r.adapter = p.index[b];
  if (r.adapter >= p.count) r.adapter = -1;
  r.live = r.adapter < 0 ? 0 : min(r.count, p.most_new);
  return r;
}

// low[split][row][r] = sum over the split's columns of x[row] A[r].  NR: tiles of 8 ranks
template <typename T, int NR> __global__ void __launch_bounds__(kAdapterWarps * 32) adapter_low_kernel(const AdapterParams p) {
  __shared__ float red[kAdapterWarps][kRowTile][NR * 8 + 2];
  griddep_wait();
  griddep_launch();
  const int split = blockIdx.y, b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const AdapterRows r = adapter_rows(p, b);
  const int t0 = blockIdx.x * kRowTile;
  if (t0 >= r.live) return;
  const int rows = min(kRowTile, r.live - t0), row0 = r.row0 + t0;
  const T *x = reinterpret_cast<const T *>(p.x), *a = reinterpret_cast<const T *>(p.a) + (long long)r.adapter * p.rank * p.width;
  const T *x0 = x + (long long)(row0 + min(g, rows - 1)) * p.ldx, *x1 = x + (long long)(row0 + min(g + 8, rows - 1)) * p.ldx;
  const bool in0 = g < rows, in1 = g + 8 < rows;
  const int begin = split * p.per_split, end = min(p.width, begin + p.per_split);
  float acc[NR][4];
#pragma unroll
  for (int n = 0; n < NR; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
  // 32 columns at a time, those of lane c from 8c on; the warps take turns.  Two turns are loaded ahead of their products.
  constexpr int kAhead = NR <= 4 ? 4 : 2;
  const uint4 none = make_uint4(0, 0, 0, 0);
  for (int k0 = begin + warp * 32; k0 < end; k0 += kAdapterWarps * 32 * kAhead) {
    uint4 xa[kAhead][2], w[kAhead][NR];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int col = k0 + u * kAdapterWarps * 32 + c * 8;
      const bool ok = col < end;
      xa[u][0] = ok && in0 ? *reinterpret_cast<const uint4 *>(x0 + col) : none;
      xa[u][1] = ok && in1 ? *reinterpret_cast<const uint4 *>(x1 + col) : none;
#pragma unroll
      for (int n = 0; n < NR; ++n) w[u][n] = ok && n * 8 < p.rank ? __ldg(reinterpret_cast<const uint4 *>(a + (long long)(n * 8 + g) * p.width + col)) : none;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        mma_low<T>(acc[n], xa[u][0].x, xa[u][1].x, xa[u][0].y, xa[u][1].y, w[u][n].x, w[u][n].y);
        mma_low<T>(acc[n], xa[u][0].z, xa[u][1].z, xa[u][0].w, xa[u][1].w, w[u][n].z, w[u][n].w);
      }
  }
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    *reinterpret_cast<float2 *>(&red[warp][g][n * 8 + 2 * c]) = make_float2(acc[n][0], acc[n][1]);
    *reinterpret_cast<float2 *>(&red[warp][g + 8][n * 8 + 2 * c]) = make_float2(acc[n][2], acc[n][3]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * p.rank; i += kAdapterWarps * 32) {
    const int row = i / p.rank, k = i % p.rank;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kAdapterWarps; ++w) sum += red[w][row][k];
    p.low[((long long)split * p.rows + row0 + row) * p.rank + k] = sum;
  }
}

// The same for many rows: 64 rows of a sequence, a split's columns in steps of 64 through shared memory (x and A, each read once per
// CTA), four steps in flight.  RT: tiles of 16 ranks.
constexpr int kLowRows = 64, kLowStep = 64, kLowStages = 4;
template <int RT> struct LowSmem {
  static constexpr int kX = kLowRows * kLowStep * 2, kA = RT * 16 * kLowStep * 2, kStage = kX + kA, kTotal = kLowStages * kStage;
};
template <typename T, int RT> __global__ void __launch_bounds__(kAdapterWarps * 32) adapter_low_many_kernel(const AdapterParams p) {
  using S = LowSmem<RT>;
  extern __shared__ __align__(128) uint8_t low_smem[];
  griddep_wait();
  griddep_launch();
  const int split = blockIdx.y, b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const AdapterRows r = adapter_rows(p, b);
  const int t0 = blockIdx.x * kLowRows;
  if (t0 >= r.live) return;
  const int rows = min(kLowRows, r.live - t0), row0 = r.row0 + t0;
  const T *x = reinterpret_cast<const T *>(p.x) + (long long)row0 * p.ldx, *a = reinterpret_cast<const T *>(p.a) + (long long)r.adapter * p.rank * p.width;
  const int begin = split * p.per_split, end = min(p.width, begin + p.per_split), steps = (end - begin + kLowStep - 1) / kLowStep;
  const uint32_t base = smem_u32(low_smem);
  // 8 lanes per row of 64 columns; chunks XOR-swizzled with the row
  auto fetch = [&](int i) {
    if (i < steps) {
      const uint32_t xs = base + (i % kLowStages) * S::kStage, as = xs + S::kX;
      const int k0 = begin + i * kLowStep, chunk = threadIdx.x & 7, col = k0 + chunk * 8;
      const bool in = col < end;
#pragma unroll
      for (int n = 0; n < kLowRows / 16; ++n) {
        const int row = n * 16 + (threadIdx.x >> 3);
        const bool ok = in && row < rows;
        cp_async16(xs + tile_off<kLowStep>(row, chunk), ok ? x + (long long)row * p.ldx + col : x, ok);
      }
#pragma unroll
      for (int n = 0; n < RT; ++n) {
        const int row = n * 16 + (threadIdx.x >> 3);
        const bool ok = in && row < p.rank;
        cp_async16(as + tile_off<kLowStep>(row, chunk), ok ? a + (long long)row * p.width + col : a, ok);
      }
    }
    cp_async_commit();
  };
  float acc[2 * RT][4];
#pragma unroll
  for (int n = 0; n < 2 * RT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
  for (int i = 0; i < kLowStages - 1; ++i) fetch(i);
  for (int i = 0; i < steps; ++i) {
    cp_async_wait<kLowStages - 2>();
    __syncthreads();
    fetch(i + kLowStages - 1);                             // (into the stage that all warps are done with)
    const uint32_t xs = base + (i % kLowStages) * S::kStage, as = xs + S::kX;
    const int mrow = warp * 16 + (lane & 15), half = lane >> 4;
#pragma unroll
    for (int k = 0; k < kLowStep / 16; ++k) {
      uint32_t xa[4], w[RT][4];                            // ranks 16 n .. + 7 and + 8 .. + 15, columns of the step's halves
      ldmatrix_x4(xa, xs + tile_off<kLowStep>(mrow, 2 * k + half));
#pragma unroll
      for (int n = 0; n < RT; ++n) ldmatrix_x4(w[n], as + tile_off<kLowStep>(n * 16 + (lane & 7) + (lane >> 4) * 8, 2 * k + ((lane >> 3) & 1)));
#pragma unroll
      for (int n = 0; n < RT; ++n) {
        mma_low<T>(acc[2 * n], xa[0], xa[1], xa[2], xa[3], w[n][0], w[n][1]);
        mma_low<T>(acc[2 * n + 1], xa[0], xa[1], xa[2], xa[3], w[n][2], w[n][3]);
      }
    }
  }
  float *low = p.low + ((long long)split * p.rows + row0) * p.rank;
#pragma unroll
  for (int n = 0; n < 2 * RT; ++n) {
    const int k = n * 8 + 2 * c, r0 = warp * 16 + g;
    if (k >= p.rank) continue;
    if (r0 < rows) *reinterpret_cast<float2 *>(low + (long long)r0 * p.rank + k) = make_float2(acc[n][0], acc[n][1]);
    if (r0 + 8 < rows) *reinterpret_cast<float2 *>(low + (long long)(r0 + 8) * p.rank + k) = make_float2(acc[n][2], acc[n][3]);
  }
}

// Eight columns that delta is added to; and the sum of them and of row g (from = 0) or g + 8 (2), rounded once.  They are requested a step ahead
// (4107 rows, 6144 columns, rank 64: both launches 57 us, a turn ahead 73, in front of the products 81).
template <bool ADD> struct BaseRow {
  float4 lo, hi;
  __device__ __forceinline__ void load(const float *at, bool there) {
    if (ADD && there) {
      lo = *reinterpret_cast<const float4 *>(at);
      hi = *reinterpret_cast<const float4 *>(at + 4);
    }
  }
  template <typename T> __device__ __forceinline__ uint4 alone() const {
    return ADD ? make_uint4(pack2<T>(lo.x, lo.y), pack2<T>(lo.z, lo.w), pack2<T>(hi.x, hi.y), pack2<T>(hi.z, hi.w)) : make_uint4(0, 0, 0, 0);
  }
  template <typename T> __device__ __forceinline__ uint4 with(const float (&acc)[4][4], int from, float down) const {
    auto sum = [&](int t, float x, float y) {
      return ADD ? pack2<T>(fmaf(acc[t][from], down, x), fmaf(acc[t][from + 1], down, y)) : pack2<T>(acc[t][from] * down, acc[t][from + 1] * down);
    };
    return make_uint4(sum(0, lo.x, lo.y), sum(1, lo.z, lo.w), sum(2, hi.x, hi.y), sum(3, hi.z, hi.w));
  }
};

// The rows in front of the first sequence and behind the last, by the whole grid: a padded batch may have many.
template <typename T, bool ADD> __device__ __forceinline__ void adapter_ends(const AdapterParams &p) {
  const int front = min(max(p.starts[0], 0), p.rows), behind = min(max(p.starts[p.batch], 0), p.rows);
  if (__builtin_expect(front == 0 && behind == p.rows, 1)) return;
  const int per = p.columns / 8;
  const long long cta = ((long long)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x, thread = cta * blockDim.x + threadIdx.x,
                  threads = (long long)gridDim.x * gridDim.y * gridDim.z * blockDim.x;
#pragma unroll 1
  for (long long i = thread; i < (long long)(front + p.rows - behind) * per; i += threads) {
    const long long at = i / per, row = at < front ? at : at - front + behind, col = i % per * 8;
    BaseRow<ADD> y;
    y.load(ADD ? p.base + row * p.ldbase + col : nullptr, true);
    *reinterpret_cast<uint4 *>(reinterpret_cast<T *>(p.delta) + row * p.ldd + col) = y.template alone<T>();
  }
}

// delta[row][n] = s sum_r low[row][r] B[n][r] (ADD: + base[row][n]), 16 rows of a sequence, the warps take turns over the columns.  KR: steps
// of 16 ranks.
template <typename T, int KR, bool ADD> __global__ void __launch_bounds__(kAdapterWarps * 32) adapter_delta_kernel(const AdapterParams p) {
  griddep_wait();
  griddep_launch();
  const int b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  adapter_ends<T, ADD>(p);
  const AdapterRows r = adapter_rows(p, b);
  const int begin = blockIdx.y * p.chunk, end = min(p.columns, begin + p.chunk), first = begin + warp * 32, step = kAdapterWarps * 32;
  T *delta = reinterpret_cast<T *>(p.delta);
  // (a sequence may bring more rows than the grid has tiles for)
  for (int t0 = blockIdx.x * kRowTile; t0 < r.count; t0 += gridDim.x * kRowTile) {
    const int rows = min(kRowTile, r.count - t0), live = min(rows, r.live - t0), row0 = r.row0 + t0;
    T *out0 = delta + (long long)(row0 + g) * p.ldd + c * 8, *out1 = out0 + 8 * p.ldd;
    const float *base0 = ADD ? p.base + (long long)(row0 + g) * p.ldbase + c * 8 : nullptr, *base1 = ADD ? base0 + 8 * p.ldbase : nullptr;
    BaseRow<ADD> y0, y1;
    if (live < rows) {                                     // (rows that were not announced have no low-rank row)
      for (int n0 = first; n0 < end; n0 += step) {
        const bool in0 = n0 + c * 8 < end && g >= live && g < rows, in1 = n0 + c * 8 < end && g + 8 >= live && g + 8 < rows;
        y0.load(base0 + n0, in0);
        y1.load(base1 + n0, in1);
        if (in0) *reinterpret_cast<uint4 *>(out0 + n0) = y0.template alone<T>();
        if (in1) *reinterpret_cast<uint4 *>(out1 + n0) = y1.template alone<T>();
      }
      if (live <= 0) continue;
    }
    const T *bm = reinterpret_cast<const T *>(p.b) + (long long)r.adapter * p.columns * p.rank + c * 4;
    // column i of tile t is n0 + 8 (i / 2) + 2 t + i % 2: lane c ends up with 8 columns that follow one another
    uint2 w[4][KR];
    auto fetch = [&](int n0) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int n = n0 + g / 2 * 8 + 2 * t + g % 2;
#pragma unroll
        for (int k = 0; k < KR; ++k)
          w[t][k] = n < end && k * 16 + c * 4 < p.rank ? __ldg(reinterpret_cast<const uint2 *>(bm + (long long)n * p.rank + k * 16)) : make_uint2(0, 0);
      }
    };
    fetch(first);
    const float s = p.scales[r.adapter];
    // low-rank rows g and g + 8, ranks 16 k + 4 c .. + 3: two pieces each
    uint32_t hi[KR][4], lo[KR][4];
    float down[2];
    {
      float4 v[KR][2] = {};
#pragma unroll 4
      for (int q = 0; q < p.splits; ++q)                   // (a split's loads together)
#pragma unroll
        for (int k = 0; k < KR; ++k)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (k * 16 + c * 4 < p.rank && g + 8 * h < live) {
              const float4 one = *reinterpret_cast<const float4 *>(p.low + ((long long)q * p.rows + row0 + g + 8 * h) * p.rank + k * 16 + c * 4);
              v[k][h] = make_float4(v[k][h].x + one.x, v[k][h].y + one.y, v[k][h].z + one.z, v[k][h].w + one.w);
            }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float m = 0.f;
#pragma unroll
        for (int k = 0; k < KR; ++k) {
          v[k][h] = make_float4(v[k][h].x * s, v[k][h].y * s, v[k][h].z * s, v[k][h].w * s);
          m = fmaxf(m, largest_of(v[k][h]));
        }
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const int e = lift_of<T>(m);
        const float up = pow2_of(e);
        down[h] = pow2_of(-e);
#pragma unroll
        for (int k = 0; k < KR; ++k) {
          two_pieces<T>(v[k][h].x * up, v[k][h].y * up, hi[k][h], lo[k][h]);
          two_pieces<T>(v[k][h].z * up, v[k][h].w * up, hi[k][h + 2], lo[k][h + 2]);
        }
      }
    }
    auto base_of = [&](int n) {
      y0.load(base0 + n, n + c * 8 < end && g < live);
      y1.load(base1 + n, n + c * 8 < end && g + 8 < live);
    };
    base_of(first);
    for (int n0 = first; n0 < end; n0 += step) {
      const BaseRow<ADD> now0 = y0, now1 = y1;
      base_of(n0 + step);
      float acc[4][4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
#pragma unroll
        for (int k = 0; k < KR; ++k) {
          mma_low<T>(acc[t], lo[k][0], lo[k][1], lo[k][2], lo[k][3], w[t][k].x, w[t][k].y);
          mma_low<T>(acc[t], hi[k][0], hi[k][1], hi[k][2], hi[k][3], w[t][k].x, w[t][k].y);
        }
      }
      fetch(n0 + step);                                    // (the next columns, while these are stored)
      if (n0 + c * 8 < end) {
        if (g < live) *reinterpret_cast<uint4 *>(out0 + n0) = now0.template with<T>(acc, 0, down[0]);
        if (g + 8 < live) *reinterpret_cast<uint4 *>(out1 + n0) = now1.template with<T>(acc, 2, down[1]);
      }
    }
  }
}

// The same for 64 rows of a sequence, 16 per warp; B comes through shared memory, 128 columns at a time, two steps ahead.  (Loaded to
// registers by every warp, 8 bytes of eight rows at a time, it kept the first-level cache busy for 48 us where this takes 20:
// 6144 columns, rank 64, 4000 rows.)  The rows of 32 columns lie in the order in which the tiles use them, so that a tile's
// eight rows follow one another; their chunks of 16 bytes are XOR-swizzled.
constexpr int kDeltaCols = 128, kDeltaStages = 3;
template <typename T, int KR, bool ADD> __global__ void __launch_bounds__(kAdapterWarps * 32) adapter_delta_many_kernel(const AdapterParams p) {
  constexpr int kChunks = 2 * KR, kRowBytes = 32 * KR, kStage = kDeltaCols * kRowBytes;
  extern __shared__ __align__(128) uint8_t delta_smem[];
  griddep_wait();
  griddep_launch();
  const int b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  adapter_ends<T, ADD>(p);
  const AdapterRows r = adapter_rows(p, b);
  const int begin = blockIdx.y * p.chunk, end = min(p.columns, begin + p.chunk), steps = (end - begin + kDeltaCols - 1) / kDeltaCols;
  const uint32_t base = smem_u32(delta_smem);
  T *delta = reinterpret_cast<T *>(p.delta);
  // chunk of row i of a tile's eight
  auto swizzled = [](int i, int chunk) { return KR == 1 ? chunk ^ (i >> 2) : KR == 2 ? chunk ^ (i >> 1) : chunk ^ i; };
  for (int t0 = blockIdx.x * kLowRows; t0 < r.count; t0 += gridDim.x * kLowRows) {
    const int row0 = r.row0 + t0 + warp * kRowTile;          // (of this warp, which may have none: <= 0)
    const int rows = min(kRowTile, r.count - t0 - warp * kRowTile), live = min(rows, r.live - t0 - warp * kRowTile);
    T *out0 = delta + (long long)(row0 + g) * p.ldd + c * 8, *out1 = out0 + 8 * p.ldd;
    const float *base0 = ADD ? p.base + (long long)(row0 + g) * p.ldbase + c * 8 : nullptr, *base1 = ADD ? base0 + 8 * p.ldbase : nullptr;
    BaseRow<ADD> y0[kDeltaCols / 32], y1[kDeltaCols / 32];   // (of a step; each is requested again, for the next step, when it was used)
    if (live < rows)                                       // (rows that were not announced have no low-rank row)
      for (int n0 = begin; n0 < end; n0 += 32) {
        const bool in0 = n0 + c * 8 < end && g >= live && g < rows, in1 = n0 + c * 8 < end && g + 8 >= live && g + 8 < rows;
        y0[0].load(base0 + n0, in0);
        y1[0].load(base1 + n0, in1);
        if (in0) *reinterpret_cast<uint4 *>(out0 + n0) = y0[0].template alone<T>();
        if (in1) *reinterpret_cast<uint4 *>(out1 + n0) = y1[0].template alone<T>();
      }
    if (t0 >= r.live) continue;
    const T *bm = reinterpret_cast<const T *>(p.b) + (long long)r.adapter * p.columns * p.rank;
    auto fetch = [&](int i) {
      if (i < steps) {
        const uint32_t at = base + (i % kDeltaStages) * kStage;
#pragma unroll 4
        for (int e = threadIdx.x; e < kDeltaCols * kChunks; e += kAdapterWarps * 32) {
          const int col = e / kChunks, chunk = e % kChunks, n = begin + i * kDeltaCols + col, in = col & 31;
          const int tile = (in & 7) >> 1, row = (in >> 3) * 2 + (in & 1);
          const bool ok = n < end && chunk * 8 < p.rank;
          cp_async16(at + ((col & ~31) + tile * 8 + row) * kRowBytes + swizzled(row, chunk) * 16, ok ? bm + (long long)n * p.rank + chunk * 8 : bm, ok);
        }
      }
      cp_async_commit();
    };
    __syncthreads();                                       // (the stages of the rows before are done with)
    for (int i = 0; i < kDeltaStages - 1; ++i) fetch(i);
    const float s = p.scales[r.adapter];
    // The low-rank rows, summed over the splits in order, 4 ranks of a row at a time, then as two pieces each through shared memory to the
    // fragments.  A split's loads go together, kPer of a thread, so that the CTA waits for splits and not for rows of splits.
    constexpr int kPieces = kLowRows * kRowBytes;
    const uint32_t at_hi = base + kDeltaStages * kStage, at_lo = at_hi + kPieces;
    uint8_t *pieces = delta_smem + kDeltaStages * kStage;
    float *downs = reinterpret_cast<float *>(pieces + 2 * kPieces);
    const int all = min(kLowRows, r.live - t0), quads = p.rank / 4;
    constexpr int kPer = 8 < 2 * KR ? 8 : 2 * KR;
    for (int e0 = threadIdx.x; e0 < kLowRows * KR * 4; e0 += kPer * kAdapterWarps * 32) {
      float4 v[kPer];
#pragma unroll
      for (int u = 0; u < kPer; ++u) v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
      for (int q = 0; q < p.splits; ++q) {
        const float4 *from = reinterpret_cast<const float4 *>(p.low + ((long long)q * p.rows + r.row0 + t0) * p.rank);
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
          const int e = e0 + u * kAdapterWarps * 32, row = e / (KR * 4), quad = e % (KR * 4);
          if (row < all && quad < quads) {
            const float4 one = from[row * quads + quad];
            v[u] = make_float4(v[u].x + one.x, v[u].y + one.y, v[u].z + one.z, v[u].w + one.w);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kPer; ++u) {
        const int e = e0 + u * kAdapterWarps * 32, row = e / (KR * 4), quad = e % (KR * 4);
        v[u] = make_float4(v[u].x * s, v[u].y * s, v[u].z * s, v[u].w * s);
        float m = largest_of(v[u]);                        // (a row's quads are in lanes that follow one another)
#pragma unroll
        for (int o = 1; o < KR * 4; o *= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const int lift = lift_of<T>(m);
        const float up = pow2_of(lift);
        if (quad == 0) downs[row] = pow2_of(-lift);
        uint2 hi2, lo2;
        two_pieces<T>(v[u].x * up, v[u].y * up, hi2.x, lo2.x);
        two_pieces<T>(v[u].z * up, v[u].w * up, hi2.y, lo2.y);
        const int to = row * kRowBytes + swizzled(row & 7, quad >> 1) * 16 + (quad & 1) * 8;
        *reinterpret_cast<uint2 *>(pieces + to) = hi2;
        *reinterpret_cast<uint2 *>(pieces + kPieces + to) = lo2;
      }
    }
    __syncthreads();
    uint32_t hi[KR][4], lo[KR][4];
#pragma unroll
    for (int k = 0; k < KR; ++k) {
      const int row = warp * kRowTile + (lane & 15), to = row * kRowBytes + swizzled(row & 7, 2 * k + (lane >> 4)) * 16;
      ldmatrix_x4(hi[k], at_hi + to);
      ldmatrix_x4(lo[k], at_lo + to);
    }
    auto base_of = [&](int u, int n) {
      y0[u].load(base0 + n, n + c * 8 < end && g < live);
      y1[u].load(base1 + n, n + c * 8 < end && g + 8 < live);
    };
#pragma unroll
    for (int u = 0; u < kDeltaCols / 32; ++u) base_of(u, begin + u * 32);
    const float down[2] = {downs[warp * kRowTile + g], downs[warp * kRowTile + g + 8]};
    for (int i = 0; i < steps; ++i) {
      cp_async_wait<kDeltaStages - 2>();
      __syncthreads();
      fetch(i + kDeltaStages - 1);
      const uint32_t at = base + (i % kDeltaStages) * kStage;
#pragma unroll(ADD ? kDeltaCols / 32 : 1)
      for (int n0 = 0; n0 < kDeltaCols; n0 += 32) {
        const int n = begin + i * kDeltaCols + n0, u = ADD ? n0 / 32 : 0;
        float acc[4][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
        constexpr int kTogether = KR < 4 ? KR : 4;           // steps whose operands are loaded before the first product
#pragma unroll
        for (int k0 = 0; k0 < KR; k0 += kTogether) {
          uint32_t w[kTogether][2][4];                     // tiles t and t + 1, ranks 16 k .. + 7 and + 8 .. + 15 each
#pragma unroll
          for (int k = 0; k < kTogether; ++k)
#pragma unroll
            for (int t = 0; t < 2; ++t)
              ldmatrix_x4(w[k][t], at + (n0 + (2 * t + (lane >> 4)) * 8 + (lane & 7)) * kRowBytes + swizzled(lane & 7, 2 * (k0 + k) + ((lane >> 3) & 1)) * 16);
          // (four products that do not wait for one another, then the next four on the same sums)
#pragma unroll
          for (int k = 0; k < kTogether; ++k) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
              mma_low<T>(acc[t], lo[k0 + k][0], lo[k0 + k][1], lo[k0 + k][2], lo[k0 + k][3], w[k][t / 2][2 * (t & 1)], w[k][t / 2][2 * (t & 1) + 1]);
#pragma unroll
            for (int t = 0; t < 4; ++t)
              mma_low<T>(acc[t], hi[k0 + k][0], hi[k0 + k][1], hi[k0 + k][2], hi[k0 + k][3], w[k][t / 2][2 * (t & 1)], w[k][t / 2][2 * (t & 1) + 1]);
          }
        }
        if (n + c * 8 < end) {
          if (g < live) *reinterpret_cast<uint4 *>(out0 + n) = y0[u].template with<T>(acc, 0, down[0]);
          if (g + 8 < live) *reinterpret_cast<uint4 *>(out1 + n) = y1[u].template with<T>(acc, 2, down[1]);
        }
        base_of(u, n + kDeltaCols);
      }
    }
  }
}

struct AdapterPlan {
  bool many;
  int tiles, splits, per_split;
};
AdapterPlan adapter_plan(int batch, int most_new, int width) {
  AdapterPlan s;
  s.many = most_new > kRowTile;
  const int rows = s.many ? kLowRows : kRowTile, turn = s.many ? kLowStep : kAdapterWarps * 32;
  s.tiles = (most_new + rows - 1) / rows;
  const long long ctas = (long long)s.tiles * batch;
  const int turns = (width + turn - 1) / turn, least = s.many ? 8 : 4;                  // turns of the CTA over its columns, at least
  int want = (int)((4ll * sm_count() + ctas - 1) / ctas);
  if (want > turns / least) want = turns / least > 0 ? turns / least : 1;
  const int per = (turns + want - 1) / want;
  s.splits = (turns + per - 1) / per;
  s.per_split = per * turn;
  return s;
}

template <typename T, int NR> int launch_low(const AdapterParams &p, const AdapterPlan &s, cudaStream_t st) {
  const dim3 grid(s.tiles, s.splits, p.batch), block(kAdapterWarps * 32);
  if (!s.many) {
    launch_pdl(adapter_low_kernel<T, NR>, grid, block, 0, st, p);
    return EB_OK;
  }
  constexpr int RT = (NR + 1) / 2, kSmem = LowSmem<RT>::kTotal;
  auto kern = adapter_low_many_kernel<T, RT>;
  if (kSmem > 48 * 1024 && cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess) {
    cudaGetLastError();
    return fail(EB_ECUDA, "adapter_delta: cannot reserve %d bytes of shared memory", kSmem);
  }
  launch_pdl(kern, grid, block, kSmem, st, p);
  return EB_OK;
}
template <typename T, int KR, bool ADD> int launch_delta(AdapterParams p, const AdapterPlan &s, cudaStream_t st) {
  // columns per CTA: enough CTAs for four on every multiprocessor, no fewer columns than a turn of the warps
  const long long ctas = (long long)s.tiles * p.batch;
  const int turns = (p.columns + kDeltaCols - 1) / kDeltaCols;
  const long long want = (4ll * sm_count() + ctas - 1) / ctas;
  const int parts = (int)(want < turns ? want : turns);
  p.chunk = (turns + parts - 1) / parts * kDeltaCols;
  static_assert(kDeltaCols == kAdapterWarps * 32, "a turn of either form");
  const dim3 grid(s.tiles, (p.columns + p.chunk - 1) / p.chunk, p.batch), block(kAdapterWarps * 32);
  if (!s.many) {
    launch_pdl(adapter_delta_kernel<T, KR, ADD>, grid, block, 0, st, p);
    return EB_OK;
  }
  constexpr int kSmem = (kDeltaStages * kDeltaCols + 2 * kLowRows) * 32 * KR + kLowRows * (int)sizeof(float);
  auto kern = adapter_delta_many_kernel<T, KR, ADD>;
  if (kSmem > 48 * 1024 && cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess) {
    cudaGetLastError();
    return fail(EB_ECUDA, "adapter_delta: cannot reserve %d bytes of shared memory", kSmem);
  }
  launch_pdl(kern, grid, block, kSmem, st, p);
  return EB_OK;
}
template <typename T> int launch_first(const AdapterParams &p, const AdapterPlan &s, cudaStream_t st) {
  return p.rank <= 8 ? launch_low<T, 1>(p, s, st) : p.rank <= 16 ? launch_low<T, 2>(p, s, st) : p.rank <= 32 ? launch_low<T, 4>(p, s, st)
                 : p.rank <= 64 ? launch_low<T, 8>(p, s, st) : launch_low<T, 16>(p, s, st);
}
template <typename T, bool ADD> int launch_second(const AdapterParams &p, const AdapterPlan &s, cudaStream_t st) {
  return p.rank <= 16 ? launch_delta<T, 1, ADD>(p, s, st) : p.rank <= 32 ? launch_delta<T, 2, ADD>(p, s, st)
     : p.rank <= 64 ? launch_delta<T, 4, ADD>(p, s, st) : launch_delta<T, 8, ADD>(p, s, st);
}

}  // namespace
}  // namespace eb

using namespace eb;

extern "C" size_t eb_adapter_scratch_bytes(int rows, int width, int rank, int batch, int most_new) {
  if (rows <= 0 || width <= 0 || rank <= 0 || batch <= 0 || most_new <= 0) return 0;
  return (size_t)adapter_plan(batch, most_new < rows ? most_new : rows, width).splits * rows * rank * sizeof(float);
}

// What all entry points check, and the parameters that they share.
static int adapter_params(const char *what, AdapterParams &p, AdapterPlan &s, const int32_t *index, const int32_t *starts, int rows, int width, int rank,
                          int adapters, int batch, int most_new, int dtype, void *scratch, size_t scratch_bytes) {
  EB_REQUIRE(dtype == EB_F16 || dtype == EB_BF16, "%s: fp16 or bf16 only (dtype %d)", what, dtype);
  EB_REQUIRE(index && starts, "%s: null pointer", what);
  EB_REQUIRE(rows > 0 && width > 0 && adapters > 0 && batch > 0 && batch < 65534 && most_new > 0, "%s: bad sizes", what);
  EB_REQUIRE(rank >= 8 && rank <= 128 && rank % 8 == 0, "%s: rank %d not supported (multiples of 8 up to 128; fill up with zeros)", what, rank);
  const size_t need = eb_adapter_scratch_bytes(rows, width, rank, batch, most_new);
  EB_REQUIRE(scratch && aligned16(scratch) && scratch_bytes >= need, "%s: %zu bytes of scratch needed, %zu given", what, need, scratch_bytes);
  if (most_new > rows) most_new = rows;
  s = adapter_plan(batch, most_new, width);
  p.index = index; p.starts = starts; p.low = reinterpret_cast<float *>(scratch); p.rows = rows; p.width = width; p.rank = rank; p.count = adapters; p.batch = batch;
  p.most_new = most_new; p.splits = s.splits; p.per_split = s.per_split;
  return EB_OK;
}
static int adapter_first(const char *what, AdapterParams &p, const void *x, long long ldx, const void *a) {
  EB_REQUIRE(x && a, "%s: null pointer", what);
  EB_REQUIRE(p.width % 8 == 0 && ldx % 8 == 0 && ldx >= p.width, "%s: widths and strides must be multiples of 8 elements that hold a row", what);
  EB_REQUIRE(aligned16(x) && aligned16(a), "%s: pointers must be 16-byte aligned", what);
  p.x = x; p.ldx = ldx; p.a = a;
  return EB_OK;
}
static int adapter_second(const char *what, AdapterParams &p, const void *b, const float *scales, const float *base, long long ldbase, void *out, long long ldo,
                          int columns) {
  EB_REQUIRE(b && scales && out, "%s: null pointer", what);
  EB_REQUIRE(columns > 0, "%s: bad sizes", what);
  EB_REQUIRE(columns % 8 == 0 && ldo % 8 == 0 && ldo >= columns && (!base || (ldbase % 8 == 0 && ldbase >= columns)),
             "%s: widths and strides must be multiples of 8 elements that hold a row", what);
  EB_REQUIRE(aligned16(b) && aligned16(out) && aligned16(base), "%s: pointers must be 16-byte aligned", what);
  p.b = b; p.scales = scales; p.base = base; p.ldbase = ldbase; p.delta = out; p.ldd = ldo; p.columns = columns;
  return EB_OK;
}

extern "C" int eb_adapter_delta(const void *x, long long ldx, const void *a, const void *b, const float *scales, const int32_t *index,
                                const int32_t *starts, void *delta, long long ldd, int rows, int width, int columns, int rank, int adapters, int batch,
                                int most_new, int dtype, void *scratch, size_t scratch_bytes, void *stream) {
  if (rows == 0 || columns == 0) return EB_OK;
  AdapterParams p{};
  AdapterPlan s{};
  int rc;
  if ((rc = adapter_params("adapter_delta", p, s, index, starts, rows, width, rank, adapters, batch, most_new, dtype, scratch, scratch_bytes))) return rc;
  if ((rc = adapter_first("adapter_delta", p, x, ldx, a)) || (rc = adapter_second("adapter_delta", p, b, scales, nullptr, 0, delta, ldd, columns))) return rc;
  cudaStream_t st = as_stream(stream);
  if ((rc = dtype == EB_F16 ? launch_first<__half>(p, s, st) : launch_first<__nv_bfloat16>(p, s, st))) return rc;
  if ((rc = dtype == EB_F16 ? launch_second<__half, false>(p, s, st) : launch_second<__nv_bfloat16, false>(p, s, st))) return rc;
  return check_launch("adapter_delta");
}

extern "C" int eb_adapter_low(const void *x, long long ldx, const void *a, const int32_t *index, const int32_t *starts, int rows, int width, int rank,
                              int adapters, int batch, int most_new, int dtype, void *scratch, size_t scratch_bytes, void *stream) {
  if (rows == 0) return EB_OK;
  AdapterParams p{};
  AdapterPlan s{};
  int rc;
  if ((rc = adapter_params("adapter_low", p, s, index, starts, rows, width, rank, adapters, batch, most_new, dtype, scratch, scratch_bytes))) return rc;
  if ((rc = adapter_first("adapter_low", p, x, ldx, a))) return rc;
  EB_REQUIRE(dtype == EB_F16, "adapter_low: fp16 only (dtype %d)", dtype);
  if ((rc = launch_first<__half>(p, s, as_stream(stream)))) return rc;
  return check_launch("adapter_low");
}

extern "C" int eb_adapter_add(const void *b, const float *scales, const int32_t *index, const int32_t *starts, const float *base, long long ldbase, void *out,
                              long long ldo, int rows, int width, int columns, int rank, int adapters, int batch, int most_new, int dtype,
                              void *scratch, size_t scratch_bytes, void *stream) {
  if (rows == 0 || columns == 0) return EB_OK;
  AdapterParams p{};
  AdapterPlan s{};
  int rc;
  EB_REQUIRE(base, "adapter_add: null pointer");
  if ((rc = adapter_params("adapter_add", p, s, index, starts, rows, width, rank, adapters, batch, most_new, dtype, scratch, scratch_bytes))) return rc;
  if ((rc = adapter_second("adapter_add", p, b, scales, base, ldbase, out, ldo, columns))) return rc;
  EB_REQUIRE(dtype == EB_F16, "adapter_add: fp16 only (dtype %d)", dtype);
  if ((rc = launch_second<__half, true>(p, s, as_stream(stream)))) return rc;
  return check_launch("adapter_add");
}
