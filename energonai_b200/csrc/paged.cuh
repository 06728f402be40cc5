// What the kernels over paged caches share: the layout of a packed batch, conversions between e4m3 codes and
// fp16 / fp32, and the limits that every page number passes before it becomes an address.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace eb {

// Rows starts[b] .. starts[b + 1] of a packed batch are the last tokens of sequence b, which has lengths[b] positions
// with them; position p lies in slot p mod page_size of page tables[b * table_ld + p / page_size].  Nothing that the
// device arrays hold leads outside the tensors: rows are bounded by `rows`, pages by `pages`, table columns by
// `table_cols`; what lies outside is left out.
struct PagedBatch {
  const int *tables, *starts, *lengths;
  long long table_ld;
  int batch, rows, table_cols, pages, page_shift;
  int most_new, clear;                 // rows of a sequence that are served at most; whether rows that none serves get zeros
};

namespace {

// Value scales below 2^-100, 0 among them, count as 2^-100: 1 / scale and log2(scale) enter the softmax.
constexpr float kLeastScale = 7.888609052210118e-31f;
// The weights of a page are summed without its value scale z, 2^(s + log2 z - m) / z.  Where log2 z is so far below the reference m that
// the power may fall out of fp32's range (pages of next to nothing beside huge ones), those that do are summed as 2^(s - m).  For the
// same reason a sum is taken over to another reference in two halves of its exponent.
constexpr float kFarBelow = 90.f, kLeastPower = -126.f;
__device__ __forceinline__ float pow2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float sum_at(float l, float by) {         // l 2^by
  const float half = pow2(0.5f * by);
  return l * half * half;
}

struct PagedRows {
  int row0, count, past, length, end;  // first row, rows (the announced ones), positions in front of them, positions in all, end of the sequence's rows
};
__device__ __forceinline__ PagedRows paged_rows(const PagedBatch &p, int b) {
  PagedRows r;
  r.row0 = max(p.starts[b], 0);
  r.end = min(p.starts[b + 1], p.rows);
  r.count = min(r.end - r.row0, p.most_new);
  r.length = p.lengths[b];
  r.past = r.length - (p.starts[b + 1] - p.starts[b]);
  if (r.past < 0 || r.count < 0) r.count = 0;          // (no such sequence)
  return r;
}
// Zeros to rows `from` to `to` of `out` (columns `col` to `col + cols`, a multiple of 8), by `threads` threads, this one number `thread`.
template <typename T> __device__ __forceinline__ void paged_zeros(T *out, long long ld, int from, int to, int col, int cols, long long thread, long long threads) {
  const int per = cols / 8;
#pragma unroll 1
  for (long long i = thread; i < (long long)(to - from) * per; i += threads)
    *reinterpret_cast<uint4 *>(out + (from + i / per) * ld + col + i % per * 8) = make_uint4(0, 0, 0, 0);
}
// The rows that no sequence serves: those of a sequence behind its announced ones (all, of one that is none) ...
template <typename T> __device__ __forceinline__ void paged_clear(const PagedRows &r, T *out, long long ld, int col, int cols, int thread, int threads) {
  if (__builtin_expect(r.row0 + r.count < r.end, 0)) paged_zeros(out, ld, r.row0 + r.count, r.end, col, cols, thread, threads);
}
// ... and those in front of the first sequence and behind the last, by the whole grid (a padded batch may have many).
template <typename T> __device__ __forceinline__ void paged_clear_ends(const PagedBatch &p, T *out, long long ld, int cols) {
  const int front = min(max(p.starts[0], 0), p.rows), behind = min(max(p.starts[p.batch], 0), p.rows);
  if (__builtin_expect(front == 0 && behind == p.rows, 1)) return;
  const long long cta = ((long long)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x, thread = cta * blockDim.x + threadIdx.x,
                  threads = (long long)gridDim.x * gridDim.y * gridDim.z * blockDim.x;
  paged_zeros(out, ld, 0, front, 0, cols, thread, threads);
  paged_zeros(out, ld, behind, p.rows, 0, cols, thread, threads);
}
__device__ __forceinline__ int paged_page(const PagedBatch &p, int b, int at) {   // page of table entry `at`, or -1
  if (at < 0 || at >= p.table_cols) return -1;
  const int id = p.tables[(long long)b * p.table_ld + at];
  return id >= 0 && id < p.pages ? id : -1;
}

// e4m3 has a subset of fp16's values; both conversions are exact or round to nearest even.
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t codes) {             // (the lower 16 bits)
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)codes));
  return r;
}
__device__ __forceinline__ uint32_t floats_to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// Whether one of the values in 16 bytes is not finite (T: the 16-bit type, or uint8_t for e4m3 codes).
template <typename T> __device__ __forceinline__ bool any_not_finite(const uint4 &x) {
  // (the exponent's ones, or a NaN code's, and one more carry into the sign's place)
  constexpr uint32_t kOnes = std::is_same<T, __half>::value ? 0x7c007c00u : std::is_same<T, __nv_bfloat16>::value ? 0x7f807f80u : 0x7f7f7f7fu;
  constexpr uint32_t kOne = kOnes & ~(kOnes << 1), kSigns = std::is_same<T, uint8_t>::value ? 0x80808080u : 0x80008000u;
  return ((((x.x & kOnes) + kOne) | ((x.y & kOnes) + kOne) | ((x.z & kOnes) + kOne) | ((x.w & kOnes) + kOne)) & kSigns) != 0;
}
// The same bytes with zeros in the place of such values.
template <typename T> __device__ __forceinline__ uint4 finite_only(const uint4 &x) {
  constexpr uint32_t kOnes = std::is_same<T, __half>::value ? 0x7c007c00u : std::is_same<T, __nv_bfloat16>::value ? 0x7f807f80u : 0x7f7f7f7fu;
  auto kept = [](uint32_t w) { return w & ~(std::is_same<T, uint8_t>::value ? __vcmpeq4(w & kOnes, kOnes) : __vcmpeq2(w & kOnes, kOnes)); };
  return make_uint4(kept(x.x), kept(x.y), kept(x.z), kept(x.w));
}

// Host side of the checks that all entry points make of a packed batch.
inline int paged_check(const char *what, PagedBatch &p, const eb_paged &c, int rows) {
  const int32_t *tables = c.tables, *starts = c.starts, *lengths = c.lengths;
  const long long table_ld = c.table_ld;
  const int batch = c.batch, table_cols = c.table_cols, pages = c.pages, page_size = c.page_size;
  EB_REQUIRE(tables && starts && lengths, "%s: null pointer", what);
  EB_REQUIRE(batch > 0 && batch <= 65535 && rows > 0 && table_cols > 0 && table_ld >= table_cols && pages > 0, "%s: bad sizes", what);
  EB_REQUIRE(page_size == 16 || page_size == 32 || page_size == 64 || page_size == 128, "%s: pages of %d positions not supported (16, 32, 64 or 128)", what,
             page_size);
  EB_REQUIRE((long long)table_cols * page_size < (1ll << 30), "%s: a table addresses at most 2^30 positions", what);
  EB_REQUIRE((c.flags & ~EB_PAGED_CLEAR) == 0, "%s: unknown flag bits 0x%x", what, c.flags);
  p.tables = tables; p.table_ld = table_ld; p.starts = starts; p.lengths = lengths; p.batch = batch; p.rows = rows; p.table_cols = table_cols;
  p.pages = pages; p.most_new = c.most_new < rows ? c.most_new : rows; p.clear = c.flags & EB_PAGED_CLEAR;
  p.page_shift = page_size == 16 ? 4 : page_size == 32 ? 5 : page_size == 64 ? 6 : 7;
  return EB_OK;
}

}  // namespace
}  // namespace eb
