// What the kernels over packed sequences and a paged key/value cache share: the bounds of a
// sequence, the place of a cached token, e4m3 codes with power-of-two scales, and the host-side
// checks of fb200_attention_params / fb200_kv_cache.
//
// Lengths and page numbers live on the device, so a kernel cannot trust them: every offset is cut to
// the extents the host gave, a page number outside the cache becomes page 0, and the status word
// records either.  No value of cu_q, kv_len or the block table makes an access out of range.
#pragma once

#include <cuda_fp8.h>

#include <type_traits>

#include "common.cuh"

namespace fb200 {

enum ServingFault : int {
  kFaultBadPage = 321,     // a page number outside the cache
  kFaultBadLength = 322,   // an offset or a length outside the extents, or more query rows than max_q
};

constexpr int64_t kMostTokens = int64_t(1) << 30;   // of a packed tensor or a cached sequence: sums of a few stay in 32 bits

__host__ __device__ inline int64_t clamp_i64(int64_t x, int64_t lo, int64_t hi) {
  return x < lo ? lo : x > hi ? hi : x;
}

// Rows [begin, begin + len) of sequence s, cut to [0, rows).
__host__ __device__ inline void sequence_span(const int32_t* cu, int64_t s, int64_t rows, int& begin, int& len) {
  const int64_t b = clamp_i64(cu[s], 0, rows), e = clamp_i64(cu[s + 1], b, rows);
  begin = static_cast<int>(b);
  len = static_cast<int>(e - b);
}

// Whether sequence_span takes the bounds of sequence s as they are.
__host__ __device__ inline bool span_fits(const int32_t* cu, int64_t s, int64_t rows) {
  return cu[s] >= 0 && cu[s] <= cu[s + 1] && cu[s + 1] <= rows;
}

// The sequence that owns packed row `row`, or -1.  cu does not decrease; whatever it holds, the search
// ends and the answer is checked.
__host__ __device__ inline int sequence_of_row(const int32_t* cu, int n_seqs, int row) {
  int lo = 0, hi = n_seqs;   // the last s with cu[s] <= row lies in [lo, hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= row) lo = mid; else hi = mid;
  }
  return n_seqs > 0 && cu[lo] <= row && row < cu[lo + 1] ? lo : -1;
}

__device__ __forceinline__ void record_fault(int* status, int code) {
  *reinterpret_cast<volatile int*>(status) = code;
}

// The cache as the kernels see it; strides in elements of the cache's type.
struct PagedCache {
  uint8_t* k;
  uint8_t* v;
  uint8_t* k_scale;
  uint8_t* v_scale;
  int64_t page_stride, token_stride, head_stride;
  int64_t scale_page_stride, scale_token_stride, scale_head_stride;
  const int32_t* table;
  int64_t table_stride;   // pages a sequence's table row holds
  int pages, page_shift;
};

// Page number of page `index` of sequence s; index is below table_stride.
__device__ __forceinline__ int page_number(const PagedCache& c, int64_t s, int64_t index, int* status) {
  int id = c.table[s * c.table_stride + index];
  if (static_cast<uint32_t>(id) >= static_cast<uint32_t>(c.pages)) {
    record_fault(status, kFaultBadPage);
    id = 0;
  }
  return id;
}

// Cached tokens of a sequence, cut to what its table row can hold.
__host__ __device__ inline int most_cached(int64_t table_stride, int page_shift) {
  const int64_t most = table_stride << page_shift;
  return static_cast<int>(most < kMostTokens ? most : kMostTokens);
}
__host__ __device__ inline int cached_length(int32_t kv_len, int64_t table_stride, int page_shift) {
  return static_cast<int>(clamp_i64(kv_len, 0, most_cached(table_stride, page_shift)));
}

__device__ __forceinline__ int64_t token_offset(const PagedCache& c, int page, int token, int head) {
  return page * c.page_stride + (token & ((1 << c.page_shift) - 1)) * c.token_stride + head * c.head_stride;
}
__device__ __forceinline__ int64_t scale_offset(const PagedCache& c, int page, int token, int head) {
  return page * c.scale_page_stride + (token & ((1 << c.page_shift) - 1)) * c.scale_token_stride +
         head * c.scale_head_stride;
}

// ---- e4m3 with a power-of-two scale --------------------------------------------------------------
// Scale byte of a row with the largest magnitude amax: the smallest e >= -126 with
// amax <= 448 * 2^e, as e + 127.  448 = 1.75 * 2^8, so with amax = 1.f * 2^(E - 127) the exponent is
// E - 127 - 8, one more if 1.f > 1.75.  Not finite: 255.
__host__ __device__ inline uint32_t scale_byte_of(uint32_t amax_bits) {
  const uint32_t exponent = amax_bits >> 23, mantissa = amax_bits & 0x7FFFFFu;
  if (exponent == 255u) return 255u;
  const int b = static_cast<int>(exponent) - 8 + (mantissa > 0x600000u ? 1 : 0);
  return b < 1 ? 1u : static_cast<uint32_t>(b);
}
// 2^(b - 127); 255 is a NaN, b = 0 (never written) reads as 0.
__device__ __forceinline__ float scale_of_byte(uint32_t b) { return __uint_as_float(b == 255u ? 0x7FC00000u : b << 23); }

// The largest number of a row may round up to 256 * 2^e, which at the very top of T's range is past its largest
// finite number (65504 becomes 65536 in float16, 248 * 2^120 and more 2^128 in bfloat16).  What comes out of an
// e4m3 cache stops at that number, so that finite numbers stay finite; NaN stays NaN.  Two numbers, `lo` first.
template <typename T> __device__ __forceinline__ uint32_t pack_finite(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value) asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ float2 e4m3x2_to_f32(uint32_t pair) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(pair), __NV_E4M3);
  return __half22float2(__half2(h));
}

// The low (high) two codes of a word as a pair of float16, exactly: one instruction at about one per cycle
// and scheduler (measured).
__device__ __forceinline__ uint32_t codes_low(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 x, y;\n\tmov.b32 {x, y}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, x;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t codes_high(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 x, y;\n\tmov.b32 {x, y}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, y;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
// What the codes of a cache are multiplied with is float16 as well.  A bfloat16 query row is brought there by
// the power of two that puts its largest magnitude into [2^14, 2^15): products with a power of two are exact,
// and what falls below float16's smallest step (2^-24) is 2^-38 of that magnitude.  No power above 2^120 is
// taken, whose inverse fp32 holds well: every bfloat16 is a multiple of 2^-133, so what it is multiplied with
// 2^120 is one of 2^-13, and rows too small to reach 2^14 lose nothing.  Returns the inverse as a factor for
// the scores.
__device__ __forceinline__ float query_lift(float amax, float& factor) {
  const int e = static_cast<int>(__float_as_uint(amax) >> 23);   // biased; 0: subnormal or nothing, 255: not finite
  const int up = e == 255 ? 0 : min(141 - e, 120);               // 2^(14 + 127 - e), from 2^-113 on
  factor = __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
  return __uint_as_float(static_cast<uint32_t>(127 - up) << 23);
}
// float16 holds nothing below 2^-24, and a row over a long cache can have most of its weight in keys far below the
// largest.  So float16 probabilities are taken times 2^7: with the 2^8 by which the running maximum may lag they
// stay below 65504, and a weight is lost from 2^-32 of the row's largest down.  bfloat16 has the range of fp32.
template <typename M> constexpr float kProbLift = std::is_same<M, __half>::value ? 7.0f : 0.0f;

// A probability times its value's scale 2^e has to fit float16 too, so rows are normalised by the largest
// 2^(score + e) instead of 2^score.  e below a floor counts as the floor (rows of zeros have e = -126), and so
// does that of a row that is not finite, which makes NaN of the result through its scale.  The row sum is then
// down to 2^(7 - e) of its largest term: above e = 107 (values past 10^34) terms 2^-26 of it start to be lost.
constexpr int kScaleFloor = -60;
__device__ __forceinline__ float scale_exponent(uint32_t b) {
  const int e = b == 255u ? kScaleFloor : static_cast<int>(b) - 127;
  return static_cast<float>(e < kScaleFloor ? kScaleFloor : e);
}

// ---- host-side checks ----------------------------------------------------------------------------
int check_attention_params(const char* what, const fb200_attention_params* p);
int check_kv_cache(const char* what, const fb200_kv_cache* c, int dtype);
int make_paged_cache(const fb200_kv_cache* c, const int32_t* table, int64_t table_stride, PagedCache* out);

}  // namespace fb200
