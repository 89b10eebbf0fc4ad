// Paged key/value cache: storing new tokens (16-bit, or e4m3 codes with a power-of-two scale per
// token and head) and reading whole sequences back.  The reference has no cache.
//
// Write, per token-head row x of head_dim numbers:
//   e = min { e >= -126 : max|x| <= 448 * 2^e },  code = e4m3(x * 2^-e) to nearest even,  byte = e + 127.
// A power of two keeps every product exact, so the codes do not depend on how the division is done,
// and code * 2^e is exact in bfloat16 when it is read.  A relative step of 2^-4 is all e4m3 has either
// way; the scale only has to keep small numbers out of its denormals.
// Read: code * 2^e, rounded once, at most the type's largest finite number.
// Both are bound by HBM: (2 + 1) bytes a number either way, 1/head_dim more for the scales.  A lane group
// (16 bytes a lane on the dense side) takes four heads of one token: the token's place, a binary search and two
// dependent loads, is found once for eight vectors in flight (figures at dispatch_rows).
#include "kv_cache.cuh"

#include <climits>
#include <type_traits>

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

// Largest magnitude of eight numbers as 16 bits.  Without their signs the bits are ordered like the
// magnitudes, infinities above everything finite and NaNs above them.
__device__ __forceinline__ uint32_t top_of(const uint4& x) {
  const uint32_t m = 0x7FFF7FFFu;
  const uint32_t t = __vmaxu2(__vmaxu2(x.x & m, x.y & m), __vmaxu2(x.z & m, x.w & m));
  return max(t & 0xFFFFu, t >> 16);
}
template <typename T> __device__ __forceinline__ uint32_t f32_bits_of(uint32_t bits16) {
  const uint16_t b = static_cast<uint16_t>(bits16);
  return __float_as_uint(to_f32(*reinterpret_cast<const T*>(&b)));
}
// Eight numbers of a row whose largest magnitude is `top` (16 bits), as codes.
template <typename T> __device__ __forceinline__ uint2 encode8(const uint4& raw, uint32_t byte) {
  if (byte == 255u) return make_uint2(0u, 0u);   // not finite
  // 2^-e = 2^(127 - byte): exponent field 254 - byte, above 0 (amax < 2^128 gives at most byte 247)
  const float inv = __uint_as_float((254u - byte) << 23);
  const T* x = reinterpret_cast<const T*>(&raw);
  uint32_t out[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t pair = __nv_cvt_float2_to_fp8x2(make_float2(to_f32(x[2 * i]) * inv, to_f32(x[2 * i + 1]) * inv), __NV_SATFINITE, __NV_E4M3);
    out[i >> 1] |= pair << ((i & 1) * 16);
  }
  return make_uint2(out[0], out[1]);
}

// The token and the heads a lane group works on.
struct Unit {
  int row, head, heads;   // heads: how many from `head` on, 0 past the end
};
template <int LANES, int HEADS> __device__ __forceinline__ Unit unit_of(int rows, int heads) {
  const int64_t unit = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / LANES;
  const int per_row = (heads + HEADS - 1) / HEADS;
  if (unit >= static_cast<int64_t>(rows) * per_row) return {0, 0, 0};
  const int row = static_cast<int>(unit / per_row), head = static_cast<int>(unit - static_cast<int64_t>(row) * per_row) * HEADS;
  return {row, head, min(HEADS, heads - head)};
}
// Page of token `pos` of sequence seq, or -1 (recorded) if it has no place.
__device__ __forceinline__ int place_of(const PagedCache& cache, int seq, int64_t pos, int* status) {
  if (pos < 0 || (pos >> cache.page_shift) >= cache.table_stride) {
    record_fault(status, kFaultBadLength);
    return -1;
  }
  const int page = cache.table[seq * cache.table_stride + (pos >> cache.page_shift)];
  if (static_cast<uint32_t>(page) < static_cast<uint32_t>(cache.pages)) return page;
  record_fault(status, kFaultBadPage);
  return -1;
}

template <typename T, bool E4M3, int LANES, int HEADS>
__global__ void __launch_bounds__(256) kv_cache_write_kernel(PagedCache cache, DenseRows in, const int32_t* __restrict__ cu_q,
                                                             const int32_t* __restrict__ kv_len, int n_seqs, int rows,
                                                             int heads, int lanes, int* status) {
  const int lane = threadIdx.x & (LANES - 1);
  const Unit u = unit_of<LANES, HEADS>(rows, heads);
  // the loads do not wait for the lookups of where the row goes
  uint4 k[HEADS], v[HEADS];
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    k[i] = v[i] = make_uint4(0, 0, 0, 0);
    if (i < u.heads && lane < lanes) {
      k[i] = __ldg(reinterpret_cast<const uint4*>(in.k + 2 * (u.row * in.k_token + (u.head + i) * in.k_head)) + lane);
      v[i] = __ldg(reinterpret_cast<const uint4*>(in.v + 2 * (u.row * in.v_token + (u.head + i) * in.v_head)) + lane);
    }
  }
  const int seq = u.heads > 0 ? sequence_of_row(cu_q, n_seqs, u.row) : -1;
  const int64_t pos = seq >= 0 ? static_cast<int64_t>(kv_len[seq]) - cu_q[seq + 1] + u.row : 0;
  if (seq >= 0 && !span_fits(cu_q, seq, rows)) record_fault(status, kFaultBadLength);
  const int page = seq >= 0 ? place_of(cache, seq, pos, status) : -1;
  constexpr int kBytes = E4M3 ? 1 : 2;
  const int64_t at = page >= 0 ? token_offset(cache, page, static_cast<int>(pos), u.head) * kBytes : 0;
  const int64_t sat = page >= 0 && E4M3 ? scale_offset(cache, page, static_cast<int>(pos), u.head) : 0;
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    const bool store = page >= 0 && i < u.heads && lane < lanes;   // the others only take part in the maximum
    const int64_t to = at + i * cache.head_stride * kBytes;
    if constexpr (E4M3) {
      uint32_t top = top_of(k[i]) | top_of(v[i]) << 16;   // both rows' maxima in one word
#pragma unroll
      for (int d = LANES / 2; d > 0; d >>= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, d, LANES));
      const uint32_t kb = scale_byte_of(f32_bits_of<T>(top & 0xFFFFu)), vb = scale_byte_of(f32_bits_of<T>(top >> 16));
      if (store) {
        *reinterpret_cast<uint2*>(cache.k + to + lane * 8) = encode8<T>(k[i], kb);
        *reinterpret_cast<uint2*>(cache.v + to + lane * 8) = encode8<T>(v[i], vb);
        if (lane == 0) {
          cache.k_scale[sat + i * cache.scale_head_stride] = static_cast<uint8_t>(kb);
          cache.v_scale[sat + i * cache.scale_head_stride] = static_cast<uint8_t>(vb);
        }
      }
    } else if (store) {
      *reinterpret_cast<uint4*>(cache.k + to + lane * 16) = k[i];
      *reinterpret_cast<uint4*>(cache.v + to + lane * 16) = v[i];
    }
  }
}

// Eight codes times the row's scale, rounded once to T (at most its largest finite number).
template <typename T> __device__ __forceinline__ uint4 decode8(uint2 codes, float scale) {
  uint32_t out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = e4m3x2_to_f32(((i < 2 ? codes.x : codes.y) >> ((i & 1) * 16)) & 0xFFFFu);
    out[i] = pack_finite<T>(f.x * scale, f.y * scale);
  }
  return make_uint4(out[0], out[1], out[2], out[3]);
}

template <typename T, bool E4M3, int LANES, int HEADS>
__global__ void __launch_bounds__(256) kv_cache_read_kernel(PagedCache cache, DenseRows out, const int32_t* __restrict__ cu_kv,
                                                            int n_seqs, int rows, int heads, int lanes, int* status) {
  const int lane = threadIdx.x & (LANES - 1);
  const Unit u = unit_of<LANES, HEADS>(rows, heads);
  if (u.heads == 0 || lane >= lanes) return;
  const int seq = sequence_of_row(cu_kv, n_seqs, u.row);
  if (seq < 0) return;
  if (!span_fits(cu_kv, seq, rows)) record_fault(status, kFaultBadLength);
  const int64_t pos = static_cast<int64_t>(u.row) - cu_kv[seq];
  const int page = place_of(cache, seq, pos, status);
  if (page < 0) return;
  using Raw = typename std::conditional<E4M3, uint2, uint4>::type;   // eight numbers
  const int64_t at = token_offset(cache, page, static_cast<int>(pos), u.head) * (E4M3 ? 1 : 2) + lane * sizeof(Raw);
  const int64_t step = cache.head_stride * (E4M3 ? 1 : 2);
  Raw k[HEADS], v[HEADS];
  uint32_t ks[HEADS], vs[HEADS];
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    if (i >= u.heads) break;
    k[i] = *reinterpret_cast<const Raw*>(cache.k + at + i * step);
    v[i] = *reinterpret_cast<const Raw*>(cache.v + at + i * step);
    if constexpr (E4M3) {
      const int64_t sat = scale_offset(cache, page, static_cast<int>(pos), u.head + i);
      ks[i] = cache.k_scale[sat];
      vs[i] = cache.v_scale[sat];
    }
  }
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    if (i >= u.heads) break;
    uint4* const to_k = reinterpret_cast<uint4*>(out.k + 2 * (u.row * out.k_token + (u.head + i) * out.k_head)) + lane;
    uint4* const to_v = reinterpret_cast<uint4*>(out.v + 2 * (u.row * out.v_token + (u.head + i) * out.v_head)) + lane;
    if constexpr (E4M3) {
      *to_k = decode8<T>(k[i], scale_of_byte(ks[i]));
      *to_v = decode8<T>(v[i], scale_of_byte(vs[i]));
    } else {
      *to_k = k[i];
      *to_v = v[i];
    }
  }
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

// Lanes per row: 8 cover head_dim 64, 16 cover 128 (one 16-byte vector of the dense side each).  Four heads a
// group when that still leaves two groups' worth of work for every thread slot of the GPU (16 prompts of up to
// 4000 tokens, 8 heads: write 44 -> 35 us), one where the call is too small for it (32 single tokens: 3.1 us
// against 4.7).
template <typename Go>
static void dispatch_rows(const fb200_kv_cache* cache, int64_t rows, int dtype, Go go) {
  const int lanes = static_cast<int>(cache->head_dim / 8), group = lanes <= 8 ? 8 : 16;
  const bool wide = rows * cache->kv_heads * group >= int64_t(2) * kNumSMs * 2048 && cache->kv_heads >= 4;
  const int64_t per_row = wide ? (cache->kv_heads + 3) / 4 : cache->kv_heads;
  const unsigned grid = static_cast<unsigned>((rows * per_row * group + 255) / 256);
  auto heads = [&](auto type, auto e4m3, auto width) {
    if (wide) go(type, e4m3, width, std::integral_constant<int, 4>(), grid, lanes);
    else go(type, e4m3, width, std::integral_constant<int, 1>(), grid, lanes);
  };
  auto width = [&](auto type, auto e4m3) {
    if (group == 8) heads(type, e4m3, std::integral_constant<int, 8>());
    else heads(type, e4m3, std::integral_constant<int, 16>());
  };
  if (cache->dtype != FB200_U8) width(__nv_bfloat16(), std::false_type());   // 16 bits move as they are
  else if (dtype == FB200_BF16) width(__nv_bfloat16(), std::true_type());
  else width(__half(), std::true_type());
}

}  // namespace fb200

using namespace fb200;

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
  dispatch_rows(cache, rows, dtype, [&](auto type, auto e4m3, auto width, auto heads, unsigned grid, int lanes) {
    kv_cache_write_kernel<decltype(type), decltype(e4m3)::value, decltype(width)::value, decltype(heads)::value>
        <<<grid, 256, 0, as_stream(stream)>>>(c, in, cu_q, kv_len, static_cast<int>(n_seqs), static_cast<int>(rows),
                                              static_cast<int>(cache->kv_heads), lanes, status);
  });
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
  dispatch_rows(cache, rows, dtype, [&](auto type, auto e4m3, auto width, auto heads, unsigned grid, int lanes) {
    kv_cache_read_kernel<decltype(type), decltype(e4m3)::value, decltype(width)::value, decltype(heads)::value>
        <<<grid, 256, 0, as_stream(stream)>>>(c, out, cu_kv, static_cast<int>(n_seqs), static_cast<int>(rows),
                                              static_cast<int>(cache->kv_heads), lanes, status);
  });
  return after_launch("kv_cache_read_kernel");
}
