// Low-rank adapters of many requests: delta = s (x A^T) B^T, with the A [rank][width], B [columns][rank] and s of each
// sequence's adapter, for the rows of a packed batch.  The projection beside it adds delta to its fp32 sums as a
// residual, so that the result is rounded once (and delta, the smaller part, before).
//
// Two launches.  The first has x A^T: bound by reading x and the adapters that occur; a CTA takes 16 rows of one
// sequence and a part of the columns, its warps take slices of that part, a lane loads 16 bytes of its row straight
// into the fragments of mma.sync (the contraction runs over columns in any order), partial sums go to shared memory and,
// where the columns are split over CTAs, to scratch, summed in order by the second launch.  That one has the
// product with B^T: bound by writing delta.  The low-rank row stays fp32 between the two and enters the product as two
// 16-bit pieces: it costs tensor time that is there, and no rounding.
#include <type_traits>

#include "common.cuh"

namespace eb {
namespace {

constexpr int kAdapterWarps = 4, kRowTile = 16;

struct AdapterParams {
  const void *x, *a, *b;
  const float *scales;
  const int *index, *starts;
  void *delta;
  float *low;                            // [splits][rows][rank]
  long long ldx, ldd;
  int rows, width, columns, rank, count, batch, splits, per_split, chunk;   // per_split: columns of x per CTA; chunk: columns of delta per CTA
};

template <typename T> __device__ __forceinline__ void mma_low(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Rows and adapter of sequence b; b = batch: the rows behind the last sequence, without one.
struct AdapterRows {
  int row0, count, adapter;
};
__device__ __forceinline__ AdapterRows adapter_rows(const AdapterParams &p, int b) {
  AdapterRows r;
  r.row0 = min(max(p.starts[b], 0), p.rows);
  r.count = (b < p.batch ? min(p.starts[b + 1], p.rows) : p.rows) - r.row0;
  r.adapter = b < p.batch ? p.index[b] : -1;
  if (r.adapter >= p.count) r.adapter = -1;
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
  if (r.adapter < 0 || t0 >= r.count) return;
  const int rows = min(kRowTile, r.count - t0), row0 = r.row0 + t0;
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

// delta[row][n] = s sum_r low[row][r] B[n][r].  KR: steps of 16 ranks.  MANY: the warps take 16 rows each of 64, else they
// take turns over the columns of 16 rows.
template <typename T, int KR, bool MANY> __global__ void __launch_bounds__(kAdapterWarps * 32) adapter_delta_kernel(const AdapterParams p) {
  griddep_wait();
  griddep_launch();
  const int b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const AdapterRows r = adapter_rows(p, b);
  constexpr int kRowsCta = MANY ? kAdapterWarps * kRowTile : kRowTile;
  const int begin = blockIdx.y * p.chunk, end = min(p.columns, begin + p.chunk);
  T *delta = reinterpret_cast<T *>(p.delta);
  // (the rows behind the last sequence may be more than the grid has tiles for)
  for (int t0 = blockIdx.x * kRowsCta + (MANY ? warp * kRowTile : 0); t0 < r.count; t0 += gridDim.x * kRowsCta) {
    const int rows = min(kRowTile, r.count - t0), row0 = r.row0 + t0;
    T *out0 = delta + (long long)(row0 + g) * p.ldd + c * 8, *out1 = out0 + 8 * p.ldd;
    const int first = begin + (MANY ? 0 : warp * 32), step = MANY ? 32 : kAdapterWarps * 32;
    if (r.adapter < 0) {
      for (int n0 = first; n0 < end; n0 += step)
        if (n0 + c * 8 < end) {
          if (g < rows) *reinterpret_cast<uint4 *>(out0 + n0) = make_uint4(0, 0, 0, 0);
          if (g + 8 < rows) *reinterpret_cast<uint4 *>(out1 + n0) = make_uint4(0, 0, 0, 0);
        }
      continue;
    }
    const float s = p.scales[r.adapter];
    // low-rank rows g and g + 8, ranks 16 k + 4 c .. + 3: two pieces each
    uint32_t hi[KR][4], lo[KR][4];
#pragma unroll
    for (int k = 0; k < KR; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (k * 16 + c * 4 < p.rank && g + 8 * h < rows)
          for (int q = 0; q < p.splits; ++q) {
            const float4 one = *reinterpret_cast<const float4 *>(p.low + ((long long)q * p.rows + row0 + g + 8 * h) * p.rank + k * 16 + c * 4);
            v.x += one.x;
            v.y += one.y;
            v.z += one.z;
            v.w += one.w;
          }
        v.x *= s;
        v.y *= s;
        v.z *= s;
        v.w *= s;
        hi[k][h] = pack2<T>(v.x, v.y);
        hi[k][h + 2] = pack2<T>(v.z, v.w);
        const float2 f0 = unpack2<T>(hi[k][h]), f1 = unpack2<T>(hi[k][h + 2]);
        lo[k][h] = pack2<T>(v.x - f0.x, v.y - f0.y);
        lo[k][h + 2] = pack2<T>(v.z - f1.x, v.w - f1.y);
      }
    const T *bm = reinterpret_cast<const T *>(p.b) + (long long)r.adapter * p.columns * p.rank + c * 4;
    for (int n0 = first; n0 < end; n0 += step) {
      // column i of tile t is n0 + 8 (i / 2) + 2 t + i % 2: lane c ends up with 8 columns that follow one another
      float acc[4][4];
      uint2 w[4][KR];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int n = n0 + g / 2 * 8 + 2 * t + g % 2;
#pragma unroll
        for (int k = 0; k < KR; ++k)
          w[t][k] = n < end && k * 16 + c * 4 < p.rank ? __ldg(reinterpret_cast<const uint2 *>(bm + (long long)n * p.rank + k * 16)) : make_uint2(0, 0);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
#pragma unroll
        for (int k = 0; k < KR; ++k) {
          mma_low<T>(acc[t], lo[k][0], lo[k][1], lo[k][2], lo[k][3], w[t][k].x, w[t][k].y);
          mma_low<T>(acc[t], hi[k][0], hi[k][1], hi[k][2], hi[k][3], w[t][k].x, w[t][k].y);
        }
      }
      if (n0 + c * 8 < end) {
        if (g < rows)
          *reinterpret_cast<uint4 *>(out0 + n0) = make_uint4(pack2<T>(acc[0][0], acc[0][1]), pack2<T>(acc[1][0], acc[1][1]), pack2<T>(acc[2][0], acc[2][1]), pack2<T>(acc[3][0], acc[3][1]));
        if (g + 8 < rows)
          *reinterpret_cast<uint4 *>(out1 + n0) = make_uint4(pack2<T>(acc[0][2], acc[0][3]), pack2<T>(acc[1][2], acc[1][3]), pack2<T>(acc[2][2], acc[2][3]), pack2<T>(acc[3][2], acc[3][3]));
      }
    }
  }
}

struct AdapterPlan {
  int tiles, splits, per_split;
};
AdapterPlan adapter_plan(int batch, int most_new, int width) {
  AdapterPlan s;
  s.tiles = (most_new + kRowTile - 1) / kRowTile;
  const long long ctas = (long long)s.tiles * batch;
  const int turns = (width + kAdapterWarps * 32 - 1) / (kAdapterWarps * 32);          // of the warps over all columns
  int want = (int)((2ll * sm_count() + ctas - 1) / ctas);
  if (want > turns / 4) want = turns / 4 > 0 ? turns / 4 : 1;
  const int per = (turns + want - 1) / want;
  s.splits = (turns + per - 1) / per;
  s.per_split = per * kAdapterWarps * 32;
  return s;
}

template <typename T, int NR> void launch_low(const AdapterParams &p, const AdapterPlan &s, cudaStream_t st) {
  launch_pdl(adapter_low_kernel<T, NR>, dim3(s.tiles, s.splits, p.batch), dim3(kAdapterWarps * 32), 0, st, p);
}
template <typename T, int KR> void launch_delta(AdapterParams p, int most_new, cudaStream_t st) {
  const bool many = most_new > kRowTile;
  const int rows = many ? kAdapterWarps * kRowTile : kRowTile, tiles = (most_new + rows - 1) / rows;
  // columns per CTA: enough CTAs for four on every multiprocessor, no fewer columns than a turn of the warps
  const long long ctas = (long long)tiles * p.batch;
  const int turn = many ? 32 : kAdapterWarps * 32, turns = (p.columns + turn - 1) / turn;
  const long long want = (4ll * sm_count() + ctas - 1) / ctas;
  const int parts = (int)(want < turns ? want : turns);
  p.chunk = (turns + parts - 1) / parts * turn;
  const dim3 grid(tiles, (p.columns + p.chunk - 1) / p.chunk, p.batch + 1);
  if (many) launch_pdl(adapter_delta_kernel<T, KR, true>, grid, dim3(kAdapterWarps * 32), 0, st, p);
  else launch_pdl(adapter_delta_kernel<T, KR, false>, grid, dim3(kAdapterWarps * 32), 0, st, p);
}
template <typename T> int launch_adapter(const AdapterParams &p, const AdapterPlan &s, int most_new, cudaStream_t st) {
  if (p.rank <= 8) launch_low<T, 1>(p, s, st);
  else if (p.rank <= 16) launch_low<T, 2>(p, s, st);
  else if (p.rank <= 32) launch_low<T, 4>(p, s, st);
  else if (p.rank <= 64) launch_low<T, 8>(p, s, st);
  else launch_low<T, 16>(p, s, st);
  if (p.rank <= 16) launch_delta<T, 1>(p, most_new, st);
  else if (p.rank <= 32) launch_delta<T, 2>(p, most_new, st);
  else if (p.rank <= 64) launch_delta<T, 4>(p, most_new, st);
  else launch_delta<T, 8>(p, most_new, st);
  return check_launch("adapter_delta");
}

}  // namespace
}  // namespace eb

using namespace eb;

extern "C" size_t eb_adapter_scratch_bytes(int rows, int width, int rank, int batch, int most_new) {
  if (rows <= 0 || width <= 0 || rank <= 0 || batch <= 0 || most_new <= 0) return 0;
  return (size_t)adapter_plan(batch, most_new < rows ? most_new : rows, width).splits * rows * rank * sizeof(float);
}

extern "C" int eb_adapter_delta(const void *x, long long ldx, const void *a, const void *b, const float *scales, const int32_t *index,
                                const int32_t *starts, void *delta, long long ldd, int rows, int width, int columns, int rank, int adapters, int batch,
                                int most_new, int dtype, void *scratch, size_t scratch_bytes, void *stream) {
  if (rows == 0 || columns == 0) return EB_OK;
  EB_REQUIRE(dtype == EB_F16 || dtype == EB_BF16, "adapter_delta: fp16 or bf16 only (dtype %d)", dtype);
  EB_REQUIRE(x && a && b && scales && index && starts && delta, "adapter_delta: null pointer");
  EB_REQUIRE(rows > 0 && width > 0 && columns > 0 && adapters > 0 && batch > 0 && batch < 65535 && most_new > 0, "adapter_delta: bad sizes");
  EB_REQUIRE(rank >= 8 && rank <= 128 && rank % 8 == 0, "adapter_delta: rank %d not supported (multiples of 8 up to 128; fill up with zeros)", rank);
  EB_REQUIRE(width % 8 == 0 && columns % 8 == 0 && ldx % 8 == 0 && ldd % 8 == 0 && ldx >= width && ldd >= columns,
             "adapter_delta: widths and strides must be multiples of 8 elements that hold a row");
  EB_REQUIRE(aligned16(x) && aligned16(a) && aligned16(b) && aligned16(delta), "adapter_delta: pointers must be 16-byte aligned");
  const size_t need = eb_adapter_scratch_bytes(rows, width, rank, batch, most_new);
  EB_REQUIRE(scratch && aligned16(scratch) && scratch_bytes >= need, "adapter_delta: %zu bytes of scratch needed, %zu given", need, scratch_bytes);
  if (most_new > rows) most_new = rows;
  const AdapterPlan s = adapter_plan(batch, most_new, width);
  AdapterParams p{};
  p.x = x; p.a = a; p.b = b; p.scales = scales; p.index = index; p.starts = starts; p.delta = delta; p.low = reinterpret_cast<float *>(scratch);
  p.ldx = ldx; p.ldd = ldd; p.rows = rows; p.width = width; p.columns = columns; p.rank = rank; p.count = adapters; p.batch = batch;
  p.splits = s.splits; p.per_split = s.per_split;
  return dtype == EB_F16 ? launch_adapter<__half>(p, s, most_new, as_stream(stream)) : launch_adapter<__nv_bfloat16>(p, s, most_new, as_stream(stream));
}
