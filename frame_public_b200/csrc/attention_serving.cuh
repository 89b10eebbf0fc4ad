// One call of fb200_attention_prompt or fb200_attention_paged, as the kernels see it.
#pragma once

#include "kv_cache.cuh"

namespace fb200 {

struct ServingProblem {
  const uint8_t* q;
  uint8_t* o;
  float* lse;
  const uint8_t* k;   // dense keys and values; a paged call reads them through PagedCache
  const uint8_t* v;
  const int32_t* cu_q;
  const int32_t* cu_kv;    // prompt
  const int32_t* kv_len;   // paged
  int64_t q_token, q_head, o_token, o_head, k_token, k_head, v_token, v_head;   // elements
  int n_seqs, q_rows, kv_rows, heads, kv_heads, group, dim, max_q, max_kv, causal, dtype;
  float scale;
};

// Query rows and keys of sequence s, cut to the extents.
template <bool PAGED>
__device__ __forceinline__ void serving_lengths(const ServingProblem& p, const PagedCache& c, int s, int& q0, int& lq, int& k0, int& lk) {
  sequence_span(p.cu_q, s, p.q_rows, q0, lq);
  if constexpr (PAGED) {
    k0 = 0;
    lk = cached_length(p.kv_len[s], c.table_stride, c.page_shift);
  } else {
    sequence_span(p.cu_kv, s, p.kv_rows, k0, lk);
  }
}

// The front of every workspace: the decode kernel's counters, zero between calls; no other kernel touches it.
constexpr size_t kServingCounterBytes = 4096;

int launch_attention_tiles(const ServingProblem& p, const PagedCache* cache, bool e4m3, void* workspace, cudaStream_t stream);
size_t attention_tiles_workspace(const ServingProblem& p);
bool attention_decode_takes(const ServingProblem& p);
size_t attention_decode_workspace(const ServingProblem& p);
int launch_attention_decode(const ServingProblem& p, const PagedCache& cache, bool e4m3, void* workspace, cudaStream_t stream);

}  // namespace fb200
