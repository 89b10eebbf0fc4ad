// Paged key/value cache: storing new tokens (16-bit, or e4m3 codes with a power-of-two scale per
// token and head) and reading whole sequences back.  The reference has no cache.
//
// Write, per token-head row x of head_dim numbers:
//   e = min { e >= -126 : max|x| <= 448 * 2^e },  code = e4m3(x * 2^-e) to nearest even,  byte = e + 127.
// A power of two keeps every product exact, so the codes do not depend on how the division is done,
// and code * 2^e is exact in bfloat16 when it is read.  A relative step of 2^-4 is all e4m3 has either
// way; the scale only has to keep small numbers out of its denormals.
// Read: code * 2^e, rounded once.
// Both are bound by HBM: (2 + 1) bytes a number either way, 1/head_dim more for the scales.
#include "kv_cache.cuh"

#include <climits>

namespace fb200 {

int device_status_word(int** dev_ptr);

int check_kv_cache(const char* what, const fb200_kv_cache* c, int dtype) {
  if (c == nullptr) return set_error(FB200_INVALID_ARGUMENT, "%s: null cache", what);
  if (dtype != FB200_BF16 && dtype != FB200_F16) {
    return set_error(FB200_UNIMPLEMENTED, "%s: needs bfloat16 or float16 (got dtype %d)", what, dtype);
  }
  if (c->dtype != dtype && c->dtype != FB200_U8) {
    return set_error(FB200_UNIMPLEMENTED, "%s: the cache holds dtype %d; it needs dtype %d or U8 (e4m3 codes)", what,
                     c->dtype, dtype);
  }
  if (c->pages < 0 || c->pages > INT_MAX || c->kv_heads < 1 || c->kv_heads > 65535) {
    return set_error(FB200_INVALID_ARGUMENT, "%s: cache of %lld pages and %lld heads", what, (long long)c->pages,
                     (long long)c->kv_heads);
  }
  if (c->head_dim < 16 || c->head_dim > 128 || c->head_dim % 16) {
    return set_error(FB200_UNIMPLEMENTED, "%s: head_dim must be a multiple of 16 up to 128 (got %lld)", what,
                     (long long)c->head_dim);
  }
  if (c->page_size < 8 || c->page_size > (1 << 20) || (c->page_size & (c->page_size - 1))) {
    return set_error(FB200_UNIMPLEMENTED, "%s: page_size must be a power of two from 8 up (got %lld)", what,
                     (long long)c->page_size);
  }
  const int64_t unit = c->dtype == FB200_U8 ? 16 : 8;
  if (c->page_stride % unit || c->token_stride % unit || c->head_stride % unit || c->page_stride < c->head_dim ||
      c->token_stride < c->head_dim || c->head_stride < c->head_dim) {
    return set_error(FB200_INVALID_ARGUMENT, "%s: cache strides must be multiples of %lld elements and at least head_dim",
                     what, (long long)unit);
  }
  if (c->pages > 0 && (c->k == nullptr || c->v == nullptr)) {
    return set_error(FB200_INVALID_ARGUMENT, "%s: null cache memory", what);
  }
  if (!aligned16(c->k) || !aligned16(c->v)) {
    return set_error(FB200_INVALID_ARGUMENT, "%s: cache memory must be 16-byte aligned", what);
  }
  if (c->dtype == FB200_U8) {
    if (c->pages > 0 && (c->k_scale == nullptr || c->v_scale == nullptr)) {
      return set_error(FB200_INVALID_ARGUMENT, "%s: an e4m3 cache needs k_scale and v_scale", what);
    }
    if (c->scale_page_stride < 1 || c->scale_token_stride < 1 || c->scale_head_stride < 1) {
      return set_error(FB200_INVALID_ARGUMENT, "%s: scale strides must be positive", what);
    }
  }
  return FB200_OK;
}

int make_paged_cache(const fb200_kv_cache* c, const int32_t* table, int64_t table_stride, PagedCache* out) {
  int shift = 0;
  while ((int64_t(1) << shift) < c->page_size) ++shift;
  *out = PagedCache{static_cast<uint8_t*>(c->k), static_cast<uint8_t*>(c->v), c->k_scale, c->v_scale,
                    c->page_stride, c->token_stride, c->head_stride, c->scale_page_stride, c->scale_token_stride,
                    c->scale_head_stride, table, table_stride, static_cast<int>(c->pages), shift};
  return FB200_OK;
}

// Rows of dense k or v beside the cache.
struct DenseRows {
  uint8_t* k;
  uint8_t* v;
  int64_t k_token, k_head, v_token, v_head;   // in elements of two bytes
};

// One row's eight numbers of this lane into the cache.  The lanes of a row (LANES of them) hold all of
// it; lanes at or past `lanes` hold nothing and only take part in the maximum.
template <typename T, bool E4M3, int LANES>
__device__ __forceinline__ void store_row(const uint4& raw, int lane, int lanes, uint8_t* codes, uint8_t* scale) {
  if constexpr (!E4M3) {
    if (lane < lanes) *reinterpret_cast<uint4*>(codes + lane * 16) = raw;
  } else {
    const T* x = reinterpret_cast<const T*>(&raw);
    float f[8], amax = 0.0f;
    bool finite = true;   // fmaxf drops a NaN, so it is looked for by itself
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f[i] = to_f32(x[i]);
      amax = fmaxf(amax, fabsf(f[i]));
      finite = finite && fabsf(f[i]) < INFINITY;
    }
    uint32_t top = finite ? __float_as_uint(amax) : 0x7F800000u;   // non-negative: ordered as integers
#pragma unroll
    for (int d = LANES / 2; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d, LANES));
    const uint32_t byte = scale_byte_of(top);
    // 2^-e = 2^(127 - byte): exponent field 254 - byte, from 0 (byte 254, never met: amax < 2^128) up
    const float inv = byte == 255u ? 0.0f : __uint_as_float((254u - byte) << 23);
    uint32_t out[2] = {0u, 0u};
    if (byte != 255u) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t pair = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * i] * inv, f[2 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
        out[i >> 1] |= pair << ((i & 1) * 16);
      }
    }
    if (lane < lanes) *reinterpret_cast<uint2*>(codes + lane * 8) = make_uint2(out[0], out[1]);
    if (lane == 0) *scale = static_cast<uint8_t>(byte);
  }
}

template <typename T, bool E4M3, int LANES>
__global__ void __launch_bounds__(256) kv_cache_write_kernel(PagedCache cache, DenseRows in, const int32_t* __restrict__ cu_q,
                                                             const int32_t* __restrict__ kv_len, int n_seqs, int rows,
                                                             int heads, int lanes, int* status) {
  const int64_t unit = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / LANES;
  const int lane = threadIdx.x & (LANES - 1);
  const bool there = unit < static_cast<int64_t>(rows) * heads;
  const int row = there ? static_cast<int>(unit / heads) : 0, head = there ? static_cast<int>(unit - static_cast<int64_t>(row) * heads) : 0;
  // the loads do not wait for the lookups of where the row goes
  uint4 k = make_uint4(0, 0, 0, 0), v = k;
  if (there && lane < lanes) {
    k = __ldg(reinterpret_cast<const uint4*>(in.k + 2 * (row * in.k_token + head * in.k_head)) + lane);
    v = __ldg(reinterpret_cast<const uint4*>(in.v + 2 * (row * in.v_token + head * in.v_head)) + lane);
  }
  const int seq = there ? sequence_of_row(cu_q, n_seqs, row) : -1;
  int page = -1, token = 0;
  if (seq >= 0) {
    const int64_t pos = static_cast<int64_t>(kv_len[seq]) - cu_q[seq + 1] + row;
    if (pos < 0 || (pos >> cache.page_shift) >= cache.table_stride) {
      record_fault(status, kFaultBadLength);
    } else {
      token = static_cast<int>(pos);
      page = cache.table[seq * cache.table_stride + (pos >> cache.page_shift)];
      if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(cache.pages)) {
        record_fault(status, kFaultBadPage);
        page = -1;
      }
    }
  }
  const bool store = page >= 0;
  const int mine = store ? lanes : 0, lead = store ? lane : -1;   // lead: lane 0 of a stored row writes the scale
  const int64_t at = store ? token_offset(cache, page, token, head) : 0;
  const int64_t sat = store && E4M3 ? scale_offset(cache, page, token, head) : 0;
  constexpr int kBytes = E4M3 ? 1 : 2;
  store_row<T, E4M3, LANES>(k, lead < 0 ? LANES : lead, mine, cache.k + at * kBytes, cache.k_scale + sat);
  store_row<T, E4M3, LANES>(v, lead < 0 ? LANES : lead, mine, cache.v + at * kBytes, cache.v_scale + sat);
}

// Eight codes times the row's scale, rounded once to T.
template <typename T> __device__ __forceinline__ uint4 decode8(uint2 codes, float scale) {
  T out[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = e4m3x2_to_f32(((i < 2 ? codes.x : codes.y) >> ((i & 1) * 16)) & 0xFFFFu);
    out[2 * i] = from_f32<T>(f.x * scale);
    out[2 * i + 1] = from_f32<T>(f.y * scale);
  }
  return *reinterpret_cast<const uint4*>(out);
}

template <typename T, bool E4M3, int LANES>
__global__ void __launch_bounds__(256) kv_cache_read_kernel(PagedCache cache, DenseRows out, const int32_t* __restrict__ cu_kv,
                                                            int n_seqs, int rows, int heads, int lanes, int* status) {
  const int64_t unit = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / LANES;
  const int lane = threadIdx.x & (LANES - 1);
  if (unit >= static_cast<int64_t>(rows) * heads || lane >= lanes) return;
  const int row = static_cast<int>(unit / heads), head = static_cast<int>(unit - static_cast<int64_t>(row) * heads);
  const int seq = sequence_of_row(cu_kv, n_seqs, row);
  if (seq < 0) return;
  const int64_t pos = static_cast<int64_t>(row) - cu_kv[seq];
  if (pos < 0 || (pos >> cache.page_shift) >= cache.table_stride) {
    record_fault(status, kFaultBadLength);
    return;
  }
  const int token = static_cast<int>(pos);
  const int page = cache.table[seq * cache.table_stride + (pos >> cache.page_shift)];
  if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(cache.pages)) {
    record_fault(status, kFaultBadPage);
    return;
  }
  const int64_t at = token_offset(cache, page, token, head);
  uint4 k, v;
  if constexpr (E4M3) {
    const int64_t sat = scale_offset(cache, page, token, head);
    const uint2 kc = *reinterpret_cast<const uint2*>(cache.k + at + lane * 8);
    const uint2 vc = *reinterpret_cast<const uint2*>(cache.v + at + lane * 8);
    k = decode8<T>(kc, scale_of_byte(cache.k_scale[sat]));
    v = decode8<T>(vc, scale_of_byte(cache.v_scale[sat]));
  } else {
    k = *reinterpret_cast<const uint4*>(cache.k + at * 2 + lane * 16);
    v = *reinterpret_cast<const uint4*>(cache.v + at * 2 + lane * 16);
  }
  *(reinterpret_cast<uint4*>(out.k + 2 * (row * out.k_token + head * out.k_head)) + lane) = k;
  *(reinterpret_cast<uint4*>(out.v + 2 * (row * out.v_token + head * out.v_head)) + lane) = v;
}

static int check_rows(const char* what, const fb200_kv_cache* cache, const void* k, int64_t kt, int64_t kh, const void* v,
                      int64_t vt, int64_t vh, const int32_t* cu, const int32_t* table, int64_t table_stride,
                      int64_t n_seqs, int64_t rows, int dtype) {
  if (int rc = check_kv_cache(what, cache, dtype)) return rc;
  if (n_seqs < 0 || n_seqs > INT_MAX - 1 || rows < 0 || rows > kMostTokens || table_stride < 0) {
    return set_error(FB200_INVALID_ARGUMENT, "%s: bad size (%lld sequences, %lld rows, table stride %lld)", what,
                     (long long)n_seqs, (long long)rows, (long long)table_stride);
  }
  if (n_seqs == 0 || rows == 0) return FB200_OK;
  if (!k || !v || !cu || !table) return set_error(FB200_INVALID_ARGUMENT, "%s: null argument", what);
  if (!aligned16(k) || !aligned16(v) || kt % 8 || kh % 8 || vt % 8 || vh % 8 || kt < cache->head_dim ||
      kh < cache->head_dim || vt < cache->head_dim || vh < cache->head_dim) {
    return set_error(FB200_INVALID_ARGUMENT,
                     "%s: k and v must be 16-byte aligned, their strides multiples of 8 elements and at least head_dim", what);
  }
  if (rows * cache->kv_heads > (int64_t(1) << 34)) return set_error(FB200_INVALID_ARGUMENT, "%s: too many rows", what);
  return FB200_OK;
}

}  // namespace fb200

using namespace fb200;

// Lanes per row: 8 cover head_dim 64, 16 cover 128 (one 16-byte vector of the dense side each).
#define FB200_KV_DISPATCH(KERNEL, ...)                                                                    \
  do {                                                                                                    \
    const int lanes = static_cast<int>(cache->head_dim / 8), group = lanes <= 8 ? 8 : 16;                 \
    const unsigned grid = static_cast<unsigned>((rows * cache->kv_heads * group + 255) / 256);            \
    const int heads = static_cast<int>(cache->kv_heads);                                                  \
    cudaStream_t s = as_stream(stream);                                                                   \
    auto go = [&](auto kernel) { kernel<<<grid, 256, 0, s>>>(__VA_ARGS__, heads, lanes, status); };       \
    const bool bf = dtype == FB200_BF16, e4m3 = cache->dtype == FB200_U8;                                 \
    if (group == 8) {                                                                                     \
      if (!e4m3) go(KERNEL<__nv_bfloat16, false, 8>);                                                     \
      else if (bf) go(KERNEL<__nv_bfloat16, true, 8>);                                                    \
      else go(KERNEL<__half, true, 8>);                                                                   \
    } else {                                                                                              \
      if (!e4m3) go(KERNEL<__nv_bfloat16, false, 16>);                                                    \
      else if (bf) go(KERNEL<__nv_bfloat16, true, 16>);                                                   \
      else go(KERNEL<__half, true, 16>);                                                                  \
    }                                                                                                     \
  } while (0)

extern "C" int fb200_kv_cache_write(const fb200_kv_cache* cache, const void* k, int64_t k_token_stride, int64_t k_head_stride,
                                    const void* v, int64_t v_token_stride, int64_t v_head_stride, const int32_t* cu_q,
                                    const int32_t* kv_len, const int32_t* block_table, int64_t table_stride,
                                    int64_t n_seqs, int64_t rows, int dtype, fb200_stream stream) {
  if (int rc = check_rows("kv_cache_write", cache, k, k_token_stride, k_head_stride, v, v_token_stride, v_head_stride, cu_q,
                          block_table, table_stride, n_seqs, rows, dtype)) {
    return rc;
  }
  if (n_seqs == 0 || rows == 0) return FB200_OK;
  if (!kv_len) return set_error(FB200_INVALID_ARGUMENT, "kv_cache_write: null argument");
  PagedCache c;
  if (int rc = make_paged_cache(cache, block_table, table_stride, &c)) return rc;
  int* status = nullptr;
  if (int rc = device_status_word(&status)) return rc;
  const DenseRows in{static_cast<uint8_t*>(const_cast<void*>(k)), static_cast<uint8_t*>(const_cast<void*>(v)),
                     k_token_stride, k_head_stride, v_token_stride, v_head_stride};
  FB200_KV_DISPATCH(kv_cache_write_kernel, c, in, cu_q, kv_len, static_cast<int>(n_seqs), static_cast<int>(rows));
  return after_launch("kv_cache_write_kernel");
}

extern "C" int fb200_kv_cache_read(const fb200_kv_cache* cache, void* k, int64_t k_token_stride, int64_t k_head_stride,
                                   void* v, int64_t v_token_stride, int64_t v_head_stride, const int32_t* cu_kv,
                                   const int32_t* block_table, int64_t table_stride, int64_t n_seqs, int64_t rows,
                                   int dtype, fb200_stream stream) {
  if (int rc = check_rows("kv_cache_read", cache, k, k_token_stride, k_head_stride, v, v_token_stride, v_head_stride, cu_kv,
                          block_table, table_stride, n_seqs, rows, dtype)) {
    return rc;
  }
  if (n_seqs == 0 || rows == 0) return FB200_OK;
  PagedCache c;
  if (int rc = make_paged_cache(cache, block_table, table_stride, &c)) return rc;
  int* status = nullptr;
  if (int rc = device_status_word(&status)) return rc;
  const DenseRows out{static_cast<uint8_t*>(k), static_cast<uint8_t*>(v), k_token_stride, k_head_stride, v_token_stride,
                      v_head_stride};
  FB200_KV_DISPATCH(kv_cache_read_kernel, c, out, cu_kv, static_cast<int>(n_seqs), static_cast<int>(rows));
  return after_launch("kv_cache_read_kernel");
}
