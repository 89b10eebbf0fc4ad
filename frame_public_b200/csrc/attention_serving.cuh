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

// Whether serving_lengths takes those of sequence s as they are.  keys: kv_len where PAGED, else cu_kv, and
// most_keys what they are cut to.  The keys of a sequence without rows (an empty place of a padded batch) may be
// anything.
template <bool PAGED>
__device__ __forceinline__ bool lengths_fit(const int32_t* cu_q, const int32_t* keys, int s, int q_rows, int most_keys) {
  if (!span_fits(cu_q, s, q_rows)) return false;
  if (cu_q[s] == cu_q[s + 1]) return true;
  if constexpr (PAGED) return keys[s] >= 0 && keys[s] <= most_keys;
  else return span_fits(keys, s, most_keys);
}

// cudaFuncSetAttribute(MaxDynamicSharedMemorySize) once per kernel and device.  (The kernels of one launch
// function have the same type, so a static in it is shared by all of them.)
struct SmemOptIn {
  static constexpr int kMost = 16;
  std::atomic<const void*> who[kMost] = {};
  std::atomic<uint64_t> done[kMost] = {};   // bit per device ordinal
  template <typename K> int once(K kernel, size_t bytes) {
    int device = 0, at = 0;
    FB200_CUDA_OK(cudaGetDevice(&device));
    const void* const f = reinterpret_cast<const void*>(kernel);
    for (; at < kMost; ++at) {   // this kernel's place, or the first free one
      const void* seen = nullptr;
      if (who[at].load(std::memory_order_relaxed) == f || who[at].compare_exchange_strong(seen, f) || seen == f) break;
    }
    const uint64_t bit = device < 64 ? uint64_t(1) << device : 0;
    if (at < kMost && (done[at].load(std::memory_order_acquire) & bit)) return FB200_OK;
    FB200_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
    if (at < kMost) done[at].fetch_or(bit, std::memory_order_release);
    return FB200_OK;
  }
};

// The front of every workspace: the decode kernel's counters, zero between calls; no other kernel touches it.
constexpr size_t kServingCounterBytes = 4096;

int launch_attention_tiles(const ServingProblem& p, const PagedCache* cache, bool e4m3, void* workspace, cudaStream_t stream);
size_t attention_tiles_workspace(const ServingProblem& p);
bool attention_decode_takes(const ServingProblem& p);
size_t attention_decode_workspace(const ServingProblem& p);
int launch_attention_decode(const ServingProblem& p, const PagedCache& cache, bool e4m3, void* workspace, cudaStream_t stream);

}  // namespace fb200
