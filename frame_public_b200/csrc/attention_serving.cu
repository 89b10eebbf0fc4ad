// Entry points of attention over packed sequences: checks, and the choice between the two kernels.
#include "attention_serving.cuh"

#include <climits>

namespace fb200 {

int check_attention_params(const char* what, const fb200_attention_params* p) {
  if (p == nullptr) return set_error(FB200_INVALID_ARGUMENT, "%s: null params", what);
  if (p->n_seqs < 0 || p->n_seqs > INT_MAX - 1 || p->q_rows < 0 || p->q_rows > kMostTokens || p->kv_rows < 0 ||
      p->kv_rows > kMostTokens || p->max_q < 0 || p->max_kv < 0) {
    return set_error(FB200_INVALID_ARGUMENT, "%s: a size is negative or past 2^30", what);
  }
  if (p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads || p->heads > 65535) {
    return set_error(FB200_INVALID_ARGUMENT, "%s: heads (%lld) must be a multiple of kv_heads (%lld)", what,
                     (long long)p->heads, (long long)p->kv_heads);
  }
  if (p->dtype != FB200_BF16 && p->dtype != FB200_F16) {
    return set_error(FB200_UNIMPLEMENTED, "%s: needs bfloat16 or float16 (got dtype %d)", what, p->dtype);
  }
  if (p->head_dim < 16 || p->head_dim > 128 || p->head_dim % 16 || p->heads / p->kv_heads > 64) {
    return set_error(FB200_UNIMPLEMENTED,
                     "%s: needs head_dim a multiple of 16 up to 128 and at most 64 query heads per kv head (got %lld, %lld)",
                     what, (long long)p->head_dim, (long long)(p->heads / p->kv_heads));
  }
  if (!(p->scale > 0.0f) || p->scale > 2.0e38f) {   // times log2(e) it still has to be finite
    return set_error(FB200_INVALID_ARGUMENT, "%s: the score scale must be positive and at most 2e38", what);
  }
  const int64_t strides[4] = {p->q_token_stride, p->q_head_stride, p->o_token_stride, p->o_head_stride};
  for (int64_t s : strides) {
    if (s % 8 || s < p->head_dim) {
      return set_error(FB200_INVALID_ARGUMENT, "%s: strides must be multiples of 8 elements and at least head_dim", what);
    }
  }
  return FB200_OK;
}

static ServingProblem make_problem(const fb200_attention_params* p, const void* q, void* o, float* lse, const int32_t* cu_q) {
  ServingProblem r{};
  r.q = static_cast<const uint8_t*>(q);
  r.o = static_cast<uint8_t*>(o);
  r.lse = lse;
  r.cu_q = cu_q;
  r.q_token = p->q_token_stride;
  r.q_head = p->q_head_stride;
  r.o_token = p->o_token_stride;
  r.o_head = p->o_head_stride;
  r.n_seqs = static_cast<int>(p->n_seqs);
  r.q_rows = static_cast<int>(p->q_rows);
  r.kv_rows = static_cast<int>(p->kv_rows);
  r.heads = static_cast<int>(p->heads);
  r.group = static_cast<int>(p->heads / p->kv_heads);
  r.kv_heads = static_cast<int>(p->kv_heads);
  r.dim = static_cast<int>(p->head_dim);
  r.max_q = static_cast<int>(p->max_q < p->q_rows ? p->max_q : p->q_rows);
  r.max_kv = static_cast<int>(p->max_kv < kMostTokens ? p->max_kv : kMostTokens);
  r.dtype = p->dtype;
  r.causal = p->causal != 0;
  r.scale = p->scale;
  return r;
}

}  // namespace fb200

using namespace fb200;

extern "C" int fb200_attention_prompt(const fb200_attention_params* params, const void* q, const void* k, const void* v,
                                      void* o, float* lse, const int32_t* cu_q, const int32_t* cu_kv, fb200_stream stream) {
  if (int rc = check_attention_params("attention_prompt", params)) return rc;
  const int64_t strides[4] = {params->k_token_stride, params->k_head_stride, params->v_token_stride, params->v_head_stride};
  for (int64_t s : strides) {
    if (s % 8 || s < params->head_dim) {
      return set_error(FB200_INVALID_ARGUMENT, "attention_prompt: strides must be multiples of 8 elements and at least head_dim");
    }
  }
  if (params->n_seqs == 0 || params->q_rows == 0) return FB200_OK;
  if (!q || !o || !cu_q || !cu_kv || (params->kv_rows > 0 && (!k || !v))) {
    return set_error(FB200_INVALID_ARGUMENT, "attention_prompt: null argument");
  }
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o)) {
    return set_error(FB200_INVALID_ARGUMENT, "attention_prompt: q, k, v and o must be 16-byte aligned");
  }
  ServingProblem r = make_problem(params, q, o, lse, cu_q);
  r.k = static_cast<const uint8_t*>(k);
  r.v = static_cast<const uint8_t*>(v);
  r.cu_kv = cu_kv;
  r.k_token = params->k_token_stride;
  r.k_head = params->k_head_stride;
  r.v_token = params->v_token_stride;
  r.v_head = params->v_head_stride;
  return launch_attention_tiles(r, nullptr, false, nullptr, as_stream(stream));
}

static int check_paged(const char* what, const fb200_attention_params* p, const fb200_kv_cache* c) {
  if (int rc = check_attention_params(what, p)) return rc;
  if (int rc = check_kv_cache(what, c, p->dtype)) return rc;
  if (c->kv_heads != p->kv_heads || c->head_dim != p->head_dim) {
    return set_error(FB200_INVALID_ARGUMENT, "%s: the cache's heads and head_dim are not the call's", what);
  }
  return FB200_OK;
}

extern "C" int fb200_attention_paged_workspace(const fb200_attention_params* params, const fb200_kv_cache* cache, size_t* bytes) {
  if (bytes == nullptr) return set_error(FB200_INVALID_ARGUMENT, "attention_paged_workspace: null out pointer");
  *bytes = 0;
  if (int rc = check_paged("attention_paged_workspace", params, cache)) return rc;
  const ServingProblem r = make_problem(params, nullptr, nullptr, nullptr, nullptr);
  *bytes = attention_decode_takes(r) ? attention_decode_workspace(r) : attention_tiles_workspace(r);
  return FB200_OK;
}

extern "C" int fb200_attention_paged(const fb200_attention_params* params, const fb200_kv_cache* cache, const void* q, void* o,
                                     float* lse, const int32_t* cu_q, const int32_t* kv_len, const int32_t* block_table,
                                     int64_t table_stride, void* workspace, size_t workspace_bytes, fb200_stream stream) {
  if (int rc = check_paged("attention_paged", params, cache)) return rc;
  if (table_stride < 0) return set_error(FB200_INVALID_ARGUMENT, "attention_paged: negative table stride");
  if (params->n_seqs == 0 || params->q_rows == 0) return FB200_OK;
  if (!q || !o || !cu_q || !kv_len || (table_stride > 0 && !block_table)) {
    return set_error(FB200_INVALID_ARGUMENT, "attention_paged: null argument");
  }
  if (cache->pages == 0 && table_stride > 0) return set_error(FB200_INVALID_ARGUMENT, "attention_paged: a cache without pages");
  if (!aligned16(q) || !aligned16(o)) return set_error(FB200_INVALID_ARGUMENT, "attention_paged: q and o must be 16-byte aligned");
  size_t need = 0;
  if (int rc = fb200_attention_paged_workspace(params, cache, &need)) return rc;
  if (workspace_bytes < need || (need > 0 && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256))) {
    return set_error(FB200_INVALID_ARGUMENT, "attention_paged: needs a 256-byte aligned workspace of %zu bytes (got %zu)", need, workspace_bytes);
  }
  PagedCache c;
  if (int rc = make_paged_cache(cache, block_table, table_stride, &c)) return rc;
  ServingProblem r = make_problem(params, q, o, lse, cu_q);
  r.kv_len = kv_len;
  if (attention_decode_takes(r)) return launch_attention_decode(r, c, cache->dtype == FB200_U8, workspace, as_stream(stream));
  return launch_attention_tiles(r, &c, cache->dtype == FB200_U8, workspace, as_stream(stream));
}
