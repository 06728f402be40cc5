// New tokens of a packed batch into a paged cache: queries and keys are turned by rotary positions (neighbouring pairs of
// the leading dimensions, angle = position * frequency in 64 bits), keys and values go to their pages, in the model's
// type or as e4m3 codes with one scale for each page and head.
//
// The scale is a power of two, the smallest with which the largest magnitude is at most 448 (e4m3's largest value): a
// floating type loses nothing by that, and when a later token raises a page's scale, the codes that the page holds
// already are divided by a power of two, which is exact but for e4m3's subnormal range.
//
// Bound by memory (each row is read and written once) or, with few tokens, by latency.  A CTA serves the rows of one
// page of one sequence and a range of heads: sines and cosines are computed once into shared memory for all of them.  A
// warp takes one head's keys, values or queries at a time, a row in D / 8 lanes of 16 bytes.  The largest magnitude of
// a page's rows has to be known before the first code, so 8-bit keys and values are read twice, the second time from the
// caches (first- and, in part, second-level: nine prompts of up to 1500 tokens read 226 MB through it and 125 MB from memory): keeping
// them would cost registers that loads in flight need.
#include <type_traits>

#include "paged.cuh"

namespace eb {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kMinScaleExp = -100;

struct AppendParams {
  PagedBatch batch;
  const void *q, *k, *v;
  void *q_out;                         // null: the queries stay as they are
  long long ldq, ldk, ldv, ldo;
  void *k_pages, *v_pages;             // [pages][kv_heads][page_size][D]
  float *k_scale, *v_scale;            // [pages][kv_heads] (8 bits)
  const float *freq;                   // [pairs]
  int heads, kv_heads, pairs, parts;   // parts: CTAs that share the heads
};

// Sine and cosine of an angle of any size: less its quarter turns in 64 bits (two parts of pi / 2: the rest is good to 2^-40 for
// angles up to 2^30), what is left, at most pi / 4, by the series of both to the terms below 2^-28, in 32 bits.
__device__ __forceinline__ void turn_of(double angle, float &s, float &c) {
  const double quarters = rint(angle * 0.63661977236758134308);
  const float r = (float)fma(quarters, -6.123233995736766e-17, fma(quarters, -1.5707963267948966, angle)), z = r * r;
  const float sine = fmaf(r * z, fmaf(z, fmaf(z, fmaf(z, 1.f / 362880.f, -1.f / 5040.f), 1.f / 120.f), -1.f / 6.f), r);
  const float cosine = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.f / 3628800.f, 1.f / 40320.f), -1.f / 720.f), 1.f / 24.f), -0.5f), 1.f);
  const int q = (int)((long long)quarters & 3);
  s = q & 1 ? cosine : sine;
  c = q & 1 ? sine : cosine;
  if (q & 2) s = -s;
  if (q == 1 || q == 2) c = -c;
}

// 2^k, the smallest power of two with m <= 448 * 2^k
__device__ __forceinline__ float scale_for(float m) {
  const int bits = __float_as_int(m), e = (bits >> 23) - 126;
  const int k = max(e - 9 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0), kMinScaleExp);
  return __int_as_float((k + 127) << 23);
}

template <typename T, bool EIGHT, int D> __global__ void __launch_bounds__(kAppendThreads, 3) paged_append_kernel(const AppendParams p) {
  extern __shared__ float4 turn_smem[];                  // [rows of the page][D / 2 pairs of cosine and sine]
  constexpr int kLanes = D / 8, kStep = 32 / kLanes;     // lanes per row, rows per warp and load
  griddep_wait();
  griddep_launch();
  const int b = blockIdx.z, part = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int page_size = 1 << p.batch.page_shift;
  const PagedRows r = paged_rows(p.batch, b);
  if (p.batch.clear && p.q_out) {
    paged_clear_ends(p.batch, reinterpret_cast<T *>(p.q_out), p.ldo, p.heads * D);
    if (blockIdx.x == 0) paged_clear(r, reinterpret_cast<T *>(p.q_out), p.ldo, 0, p.heads * D, part * kAppendThreads + threadIdx.x, p.parts * kAppendThreads);
  }
  const int at = (r.past >> p.batch.page_shift) + blockIdx.x, begin = max(at << p.batch.page_shift, r.past), end = min((at + 1) << p.batch.page_shift, r.past + r.count);
  if (begin >= end) return;
  const int n = end - begin, slot0 = begin & (page_size - 1), row0 = r.row0 + begin - r.past;
  const int page = paged_page(p.batch, b, at);

  // (Rows of a sequence behind the announced most_new are left out, as shared memory holds no more of a page.)
  // Cosine and sine of pair j of row i, where lane j / 4 of the row reads its four pairs as two 16-byte words without a bank conflict.
  float2 *turn = reinterpret_cast<float2 *>(turn_smem);
  for (int i = threadIdx.x; i < n * p.pairs; i += kAppendThreads) {
    const int row = i / p.pairs, j = i - row * p.pairs;
    float s, c;
    turn_of((double)(begin + row) * (double)p.freq[j], s, c);
    turn[row * (D / 2) + ((j & 2) / 2 * kLanes + j / 4) * 2 + (j & 1)] = make_float2(c, s);
  }
  __syncthreads();

  const int sub = lane / kLanes, part_of_row = lane % kLanes, col = part_of_row * 8;
  const bool turns_all = col / 2 + 4 <= p.pairs;
  // 8 columns of row i, turned
  auto turned = [&](const uint4 &raw, int i, float (&f)[8]) {
    Vec16<T> x;
    x.raw = raw;
    x.unpack(f);
    if (col / 2 >= p.pairs) return;
    const float4 *t = turn_smem + i * (D / 4) + part_of_row;
    const float4 t0 = t[0], t1 = t[kLanes];
    const float cs[4] = {t0.x, t0.z, t1.x, t1.z}, sn[4] = {t0.y, t0.w, t1.y, t1.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float u = f[2 * e], w = f[2 * e + 1];
      if (turns_all || col / 2 + e < p.pairs) {
        f[2 * e] = u * cs[e] - w * sn[e];
        f[2 * e + 1] = w * cs[e] + u * sn[e];
      }
    }
  };
  using Four = std::integral_constant<int, 4>;
  using Few = std::integral_constant<int, 2>;            // (8-bit rows have more to keep meanwhile)
  // fn(i, raw) for the rows i of this lane, so many loads in flight
  auto each_row = [&](auto unroll, const T *x, long long ld, auto fn) {
    constexpr int kUnroll = decltype(unroll)::value;
    const T *at = x + (long long)(row0 + sub) * ld + col;
    for (int i0 = sub; i0 < n; i0 += kStep * kUnroll, at += kStep * kUnroll * ld) {
      uint4 raw[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (i0 + u * kStep < n) raw[u] = *reinterpret_cast<const uint4 *>(at + u * kStep * ld);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (i0 + u * kStep < n) fn(i0 + u * kStep, raw[u]);
    }
  };

  const int cached = page >= 0 ? 2 * p.kv_heads : 0, items = cached + (p.q_out ? p.heads : 0);
  for (int item = part * (kAppendThreads / 32) + warp; item < items; item += p.parts * (kAppendThreads / 32)) {
    if (item >= cached) {
      const int h = item - cached;
      T *out = reinterpret_cast<T *>(p.q_out) + h * D + col;
      each_row(Four{}, reinterpret_cast<const T *>(p.q) + h * D, p.ldq, [&](int i, const uint4 &raw) {
        float f[8];
        turned(raw, i, f);
        Vec16<T> y;
        y.pack(f);
        y.store(out + (long long)(row0 + i) * p.ldo);
      });
      continue;
    }
    const bool is_k = item < p.kv_heads;
    const int h = is_k ? item : item - p.kv_heads;
    const T *x = reinterpret_cast<const T *>(is_k ? p.k : p.v) + h * D;
    const long long ld = is_k ? p.ldk : p.ldv, block = (long long)page * p.kv_heads + h;
    auto value = [&](const uint4 &raw, int i, float (&f)[8]) {
      if (is_k) {
        turned(raw, i, f);
      } else {
        Vec16<T> y;
        y.raw = raw;
        y.unpack(f);
      }
    };
    if constexpr (!EIGHT) {
      T *out = reinterpret_cast<T *>(is_k ? p.k_pages : p.v_pages) + (block * page_size + slot0) * D + col;
      each_row(Four{}, x, ld, [&](int i, const uint4 &raw) {
        if (is_k && p.pairs > 0) {
          float f[8];
          turned(raw, i, f);
          Vec16<T> y;
          y.pack(f);
          y.store(out + i * D);
        } else {
          *reinterpret_cast<uint4 *>(out + i * D) = raw;
        }
      });
    } else {
      uint8_t *codes = reinterpret_cast<uint8_t *>(is_k ? p.k_pages : p.v_pages) + block * page_size * D + col;
      float *scale = (is_k ? p.k_scale : p.v_scale) + block;
      const float before = *scale;
      float m = 0.f;
      each_row(Few{}, x, ld, [&](int i, const uint4 &raw) {
        float f[8];
        value(raw, i, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(f[e]));         // (of a NaN and a number: the number)
      });
      m = warp_max(m);
      const bool infinite = m > 3.402823466e38f;
      if (infinite) {                                                  // the largest of the finite ones
        m = 0.f;
        each_row(Few{}, x, ld, [&](int i, const uint4 &raw) {
          float f[8];
          value(raw, i, f);
#pragma unroll
          for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(f[e]) <= 3.402823466e38f ? fabsf(f[e]) : 0.f);
        });
        m = warp_max(m);
      }
      const float need = scale_for(m), after = slot0 > 0 ? fmaxf(before, need) : need;
      if (slot0 > 0 && after != before) {
        const float by = before / after;
        for (int i = sub; i < slot0; i += kStep) {
          uint2 w = *reinterpret_cast<const uint2 *>(codes + i * D);
          uint32_t *half = reinterpret_cast<uint32_t *>(&w);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 lo = unpack2<__half>(e4m3x2_to_half2(half[e])), hi = unpack2<__half>(e4m3x2_to_half2(half[e] >> 16));
            half[e] = floats_to_e4m3x2(lo.x * by, lo.y * by) | floats_to_e4m3x2(hi.x * by, hi.y * by) << 16;
          }
          *reinterpret_cast<uint2 *>(codes + i * D) = w;
        }
      }
      if (lane == 0 && (slot0 == 0 || after != before)) *scale = after;
      const float inv = 1.f / after;                                   // (a power of two: exact)
      each_row(Few{}, x, ld, [&](int i, const uint4 &raw) {
        float f[8];
        value(raw, i, f);
        if (infinite) {
          // (x - x is 0, or NaN where x is not finite: the conversion would make infinity its largest value)
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = fmaf(f[e], inv, f[e] - f[e]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] *= inv;
        }
        uint2 w;
        w.x = floats_to_e4m3x2(f[0], f[1]) | floats_to_e4m3x2(f[2], f[3]) << 16;
        w.y = floats_to_e4m3x2(f[4], f[5]) | floats_to_e4m3x2(f[6], f[7]) << 16;
        *reinterpret_cast<uint2 *>(codes + (slot0 + i) * D) = w;
      });
    }
  }
}

template <typename T, bool EIGHT, int D> int launch_append(const AppendParams &p, dim3 grid, int smem, cudaStream_t st) {
  auto kern = paged_append_kernel<T, EIGHT, D>;
  if (smem > 48 * 1024 && cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
    cudaGetLastError();
    return fail(EB_ECUDA, "paged_append: cannot reserve %d bytes of shared memory", smem);
  }
  launch_pdl(kern, grid, dim3(kAppendThreads), smem, st, p);
  return check_launch("paged_append");
}

}  // namespace
}  // namespace eb

using namespace eb;

extern "C" int eb_paged_append(const eb_paged *cache, const void *q, long long ldq, const void *k, long long ldk, const void *v, long long ldv, void *q_out,
                               long long ldo, int rows, int heads, const float *freq, int pairs, void *stream) {
  EB_REQUIRE(cache, "paged_append: null pointer");
  const int batch = cache->batch, kv_heads = cache->kv_heads, head_dim = cache->head_dim, page_size = cache->page_size, dtype = cache->dtype;
  int most_new = cache->most_new;
  void *k_pages = cache->k_pages, *v_pages = cache->v_pages;
  float *k_scale = cache->k_scale, *v_scale = cache->v_scale;
  if (rows == 0 || batch == 0 || most_new == 0) return EB_OK;
  AppendParams p{};
  if (int rc = paged_check("paged_append", p.batch, *cache, rows)) return rc;
  EB_REQUIRE(dtype == EB_F16 || dtype == EB_BF16, "paged_append: fp16 or bf16 only (dtype %d)", dtype);
  EB_REQUIRE(head_dim == 64 || head_dim == 128, "paged_append: head_dim %d not supported (64 or 128)", head_dim);
  EB_REQUIRE(heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && (long long)heads * head_dim < (1 << 28), "paged_append: %d heads do not share %d key / value heads", heads, kv_heads);
  EB_REQUIRE(k && v && k_pages && v_pages && (!q_out || q), "paged_append: null pointer");
  EB_REQUIRE(!k_scale == !v_scale, "paged_append: 8-bit pages have scales for keys and for values");
  EB_REQUIRE(pairs >= 0 && 2 * pairs <= head_dim && (pairs == 0 || freq), "paged_append: %d pairs in heads of %d", pairs, head_dim);
  EB_REQUIRE(most_new > 0, "paged_append: at most %d new rows per sequence", most_new);
  EB_REQUIRE(ldk >= (long long)kv_heads * head_dim && ldv >= (long long)kv_heads * head_dim && (!q_out || (ldq >= (long long)heads * head_dim && ldo >= (long long)heads * head_dim)),
             "paged_append: row strides smaller than the rows they hold");
  EB_REQUIRE(ldk % 8 == 0 && ldv % 8 == 0 && (!q_out || (ldq % 8 == 0 && ldo % 8 == 0)), "paged_append: strides must be multiples of 8 elements");
  EB_REQUIRE(aligned16(k) && aligned16(v) && aligned16(k_pages) && aligned16(v_pages) && (!q_out || (aligned16(q) && aligned16(q_out))),
             "paged_append: pointers must be 16-byte aligned");
  p.q = q; p.k = k; p.v = v; p.q_out = q_out; p.ldq = ldq; p.ldk = ldk; p.ldv = ldv; p.ldo = ldo;
  p.k_pages = k_pages; p.v_pages = v_pages; p.k_scale = k_scale; p.v_scale = v_scale; p.freq = freq;
  p.heads = heads; p.kv_heads = kv_heads; p.pairs = pairs;
  if (most_new > rows) most_new = rows;
  const int touched = (most_new - 1 + page_size - 1) / page_size + 1, held = most_new < page_size ? most_new : page_size;
  // up to eight CTAs for every multiprocessor, as the sequences may bring much less than they are announced with (75 us with two,
  // 61 with eight: nine prompts of up to 1500 tokens); each computes the angles of its rows
  const int items = 2 * kv_heads + (q_out ? heads : 0), most = (items + kAppendThreads / 32 - 1) / (kAppendThreads / 32);
  const long long units = (long long)touched * batch;
  const long long want = (8ll * sm_count() + units - 1) / units;
  p.parts = (int)(want < most ? want : most);
  const dim3 grid(touched, p.parts, batch);
  const int smem = pairs > 0 ? held * head_dim / 2 * (int)sizeof(float2) : 0;
  cudaStream_t st = as_stream(stream);
#define EB_APPEND(T, E) (head_dim == 64 ? launch_append<T, E, 64>(p, grid, smem, st) : launch_append<T, E, 128>(p, grid, smem, st))
  if (dtype == EB_F16) return k_scale ? EB_APPEND(__half, true) : EB_APPEND(__half, false);
  return k_scale ? EB_APPEND(__nv_bfloat16, true) : EB_APPEND(__nv_bfloat16, false);
#undef EB_APPEND
}
