// Attention of few query rows over a paged cache: decoding steps and short drafts, where a kv head's
// rows (new tokens x the query heads that share it) fit the 16 rows of one mma.sync tile.
//
// Bound by HBM: every cached key and value is read once and used for 4 * 16 FLOP a number, a few
// percent of what even the warp-level tensor instructions do in the time of the read, so tcgen05's
// 128-row tiles would only add latency.  What counts is that all SMs stream evenly to the end and
// keep enough bytes in flight:
//   * The work is the list of (sequence, kv head) pairs in tiles of keys, dealt out in equal contiguous
//     ranges to two CTAs per SM, whatever the lengths are.  A pair that lies in several ranges leaves
//     partial results (row maximum, sum, unnormalised O in fp32); the CTA that finishes last joins them in
//     the order of the keys, so results do not depend on timing and no second launch is needed.
//   * A warp streams slabs of keys of its own through a ring of three cp.async stages (8 KiB each at
//     head_dim 128: 128 KiB in flight per SM) and keeps its own running maximum, sum and O in registers; the
//     four warps of a CTA meet only at the end of a pair's range, and the ring runs on across it.
// e4m3 codes are turned into float16 operands in registers (exact, one conversion per two codes; bfloat16
// takes five instructions, which bound the kernel: 130 us where this takes 79 us, 8 sequences over up to
// 32000 keys); the scale of K multiplies the score, that of V the probability.  The contraction index of
// Q K^T and the columns of O are permuted so that a thread reads 16 codes of one row at a time.
#include <type_traits>

#include "attention_serving.cuh"

namespace fb200 {

int device_status_word(int** dev_ptr);

constexpr int kDecodeWarps = 4;
constexpr int kDecodeStages = 3;
constexpr int kDecodeCtasPerSm = 2;
constexpr int kDecodeJoinRows = 4;
constexpr int kDecodeMostCtas = kNumSMs * kDecodeCtasPerSm;
constexpr int kDecodeRows = 16;
constexpr int kDecodeSlabBytes = 4096;      // K or V of one slab at head_dim 65..128; half below
static_assert(kDecodeMostCtas * sizeof(uint32_t) <= kServingCounterBytes, "one counter per CTA");

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <bool TRANS> __device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
  if constexpr (TRANS) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  } else {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  }
}

template <typename T> __device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Position in the list of tiles: tile `tile` of [.., end) of pair (seq, head).
struct Cursor {
  int seq, head, tile, end;   // end: the pair's last tile + 1, or where this CTA's range ends
  int lk, tiles;              // keys and tiles of the sequence
  int64_t left;               // tiles of this CTA's range behind `end`
};

// Tiles a pair of sequence s takes; a sequence with rows but no keys takes one, which writes zeros.
template <int TILE>
__device__ __forceinline__ int pair_tiles(const ServingProblem& p, const PagedCache& c, int s, int& lk) {
  int q0, lq, k0;
  serving_lengths<true>(p, c, s, q0, lq, k0, lk);
  return lq == 0 ? 0 : lk <= TILE ? 1 : (lk - 1) / TILE + 1;
}

template <int TILE>
__device__ __forceinline__ void cursor_enter(const ServingProblem& p, const PagedCache& c, Cursor& at) {
  while (at.seq < p.n_seqs) {   // the next sequence that has tiles
    at.tiles = pair_tiles<TILE>(p, c, at.seq, at.lk);
    if (at.tiles > 0) break;
    ++at.seq;
  }
}
template <int TILE>
__device__ __forceinline__ void cursor_next(const ServingProblem& p, const PagedCache& c, Cursor& at) {
  if (++at.tile < at.end) return;
  at.tile = at.end = 0;
  if (at.left == 0) return;
  if (++at.head == p.kv_heads) {
    at.head = 0;
    ++at.seq;
    cursor_enter<TILE>(p, c, at);
  }
  at.end = at.left < at.tiles ? static_cast<int>(at.left) : at.tiles;
  at.left -= at.end;
}

// BIG: head_dim 65..128, else up to 64.  HALVES: 1 when a kv head has at most 8 rows (the tile's upper half
// stays empty and costs no softmax), else 2.
template <typename T, bool BIG, bool E4M3, int HALVES>
__global__ void __launch_bounds__(kDecodeWarps * 32, kDecodeCtasPerSm)
attention_decode_kernel(const ServingProblem p, const PagedCache cache, uint8_t* workspace, int* status) {
  constexpr int kSlab = E4M3 ? 32 : 16;                    // keys of a warp's slab
  constexpr int kTile = kSlab * kDecodeWarps;
  constexpr int kDim = BIG ? 128 : 64;
  constexpr int kSteps = kDim / 16;                        // k steps of Q K^T
  constexpr int kCols = kDim / 8;                          // column tiles of O
  constexpr int kRowBytes = kDim * (E4M3 ? 1 : 2);
  constexpr int kUnits = kRowBytes / 16;                   // 16-byte units of a row
  constexpr int kHalf = kSlab * kRowBytes;                 // K or V of a slab
  constexpr int kKeyTiles = kSlab / 8;
  using M = typename std::conditional<E4M3, __half, T>::type;   // type of the operands
  static_assert(kHalf <= kDecodeSlabBytes, "slab");

  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g4 = lane >> 2, t = lane & 3;
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * (kDecodeStages * 2 * kHalf);
  float* const join_o = reinterpret_cast<float*>(smem + kDecodeWarps * kDecodeStages * 2 * kHalf);   // [warps][kDecodeJoinRows][kDim]
  float* const join_m = join_o + kDecodeWarps * kDecodeJoinRows * kDim;                                            // [warps][16]
  float* const join_l = join_m + kDecodeWarps * kDecodeRows;
  __shared__ int last_flag;
  const int units = p.dim * (E4M3 ? 1 : 2) / 16, steps = p.dim / 16;

  // Where a lane reads in a slab of codes; rows are constants away (the swizzles depend on the lane alone).
  uint32_t lane_k[2] = {0, 0}, lane_v = 0;
  if constexpr (E4M3) {
    const int row_swap = BIG ? (g4 & 1) << 2 : 0;
    lane_k[0] = g4 * kRowBytes + ((t ^ row_swap) << 4);
    lane_k[1] = g4 * kRowBytes + (((4 + t) ^ row_swap) << 4);
    lane_v = t * 2 * kRowBytes + (BIG ? (g4 ^ (t * 2)) << 4 : (((g4 >> 1) ^ t) << 4) + (g4 & 1) * 8);
    if (units < kUnits) {   // what no copy fills reads as zeros
      for (int i = lane; i < kDecodeStages * 2 * kHalf / 16; i += 32) {
        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(ring + i * 16), "r"(0) : "memory");
      }
      __syncwarp();
    }
  }

  // ---- this CTA's range -----------------------------------------------------------------------------
  int64_t total = 0;
  {
    int64_t sum = 0;
    for (int s = lane; s < p.n_seqs; s += 32) {
      int lk;
      sum += pair_tiles<kTile>(p, cache, s, lk);
      if (blockIdx.x == 0 && warp == 0 && !lengths_fit<true>(p.cu_q, p.kv_len, s, p.q_rows, most_cached(cache.table_stride, cache.page_shift))) record_fault(status, kFaultBadLength);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    total = sum * p.kv_heads;
  }
  const int64_t ctas = total < gridDim.x ? total : gridDim.x;
  if (blockIdx.x >= ctas) return;
  auto range_start = [&](int64_t cta) { return total * cta / ctas; };
  const int64_t t0 = range_start(blockIdx.x), t1 = range_start(blockIdx.x + 1);
  Cursor take{};   // consumed next
  {
    int64_t before = 0;   // tiles of the sequences before s0
    for (int s0 = 0; s0 < p.n_seqs; s0 += 32) {
      int lk = 0;
      const int64_t n = s0 + lane < p.n_seqs ? static_cast<int64_t>(pair_tiles<kTile>(p, cache, s0 + lane, lk)) * p.kv_heads : 0;
      int64_t upto = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += x;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, before + upto > t0);
      if (hit) {
        const int src = __ffs(hit) - 1;
        const int64_t into = t0 - before - __shfl_sync(0xffffffffu, upto - n, src);
        take.seq = s0 + src;
        take.lk = __shfl_sync(0xffffffffu, lk, src);
        take.tiles = static_cast<int>(__shfl_sync(0xffffffffu, n, src) / p.kv_heads);
        take.head = static_cast<int>(into / take.tiles);
        take.tile = static_cast<int>(into - static_cast<int64_t>(take.head) * take.tiles);
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    const int64_t len = t1 - t0, room = take.tiles - take.tile;
    take.end = take.tile + static_cast<int>(len < room ? len : room);
    take.left = len - (take.end - take.tile);
  }
  Cursor load = take;   // fetched next
  int64_t to_load = t1 - t0;

  // The page of key `lane` of the slab that is fetched next, and the scale bytes of key `lane` of the slab
  // fetched last: loaded one slab ahead of their use, and not looked at before.
  auto page_ahead = [&]() -> int {
    const int key = load.tile * kTile + warp * kSlab + lane;
    return to_load > 0 && lane < kSlab && key < load.lk ? cache.table[load.seq * cache.table_stride + (key >> cache.page_shift)] : 0;
  };
  int page_raw = page_ahead();
  uint32_t k_scale_new = 0, v_scale_new = 0, k_scale_next = 0, v_scale_next = 0;
  auto fetch = [&](int stage) {
    if (to_load > 0) {
      const int key0 = load.tile * kTile + warp * kSlab, valid = load.lk - key0;
      const uint32_t dst = ring + stage * (2 * kHalf);
      int page = page_raw;
      if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(cache.pages)) {
        if (cache.pages > 0) record_fault(status, kFaultBadPage);
        page = 0;
      }
      if (valid > 0) {
        constexpr int kElem = E4M3 ? 1 : 2, kStepRows = 32 / kUnits;
        const int row0 = lane / kUnits, unit = lane % kUnits;
        auto copy = [&](int row, int64_t off) {
          const bool there = row < valid;   // rows behind the last key become zeros
          if (!there) off = 0;
          const int swz_k = E4M3 ? (BIG ? (row & 1) << 2 : 0) : row & (kUnits < 8 ? kUnits - 1 : 7);
          const int swz_v = E4M3 ? (BIG ? row & 6 : (row >> 1) & 3) : swz_k;
          if (unit < units) {
            cp_async16(dst + row * kRowBytes + ((unit ^ swz_k) << 4), cache.k + off, there);
            cp_async16(dst + kHalf + row * kRowBytes + ((unit ^ swz_v) << 4), cache.v + off, there);
          }
        };
        if ((1 << cache.page_shift) >= kSlab) {   // a slab lies in one page
          const int64_t step = cache.token_stride * (kStepRows * kElem);
          int64_t off = token_offset(cache, __shfl_sync(0xffffffffu, page, 0), key0 + row0, load.head) * kElem + unit * 16;
#pragma unroll
          for (int i = 0; i < kSlab / kStepRows; ++i, off += step) copy(row0 + i * kStepRows, off);
        } else {
#pragma unroll 1
          for (int i = 0; i < kSlab / kStepRows; ++i) {
            const int row = row0 + i * kStepRows;
            copy(row, token_offset(cache, __shfl_sync(0xffffffffu, page, row), key0 + row, load.head) * kElem + unit * 16);
          }
        }
      }
      if constexpr (E4M3) {
        if (lane < valid) {
          const int64_t at = scale_offset(cache, page, key0 + lane, load.head);
          k_scale_new = cache.k_scale[at];
          v_scale_new = cache.v_scale[at];
        }
      }
      --to_load;
      cursor_next<kTile>(p, cache, load);
      page_raw = page_ahead();
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kDecodeStages - 1; ++i) {
    k_scale_next = k_scale_new;
    v_scale_next = v_scale_new;
    fetch(i);
  }

  const float c = p.scale * 1.4426950408889634f;
  int stage = 0;
  for (int64_t todo = t1 - t0; todo > 0;) {
    // ---- one pair's share ---------------------------------------------------------------------------
    int q0, lq, k0, lk;
    serving_lengths<true>(p, cache, take.seq, q0, lq, k0, lk);
    const int shift = lk - lq;   // query i sees keys up to i + shift
    if (lq > p.max_q) {
      if (tid == 0) record_fault(status, kFaultBadLength);
      lq = p.max_q;
    }
    const int rows = lq * p.group, head = take.head, first_tile = take.tile, end_tile = take.end;
    const int pair_n = take.tiles;
    uint32_t q[kSteps][4] = {};
    int limit[2] = {0, 0};
    float lift[2] = {c, c};   // of the scores, to the exponent's units
#pragma unroll
    for (int half = 0; half < HALVES; ++half) {
      const int r = g4 + half * 8, i = r / p.group;
      limit[half] = r < rows ? (p.causal ? min(lk, i + shift + 1) : lk) : 0;
      const uint8_t* src = p.q + 2 * ((q0 + i) * p.q_token + (head * p.group + r - i * p.group) * p.q_head);
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) {
        if constexpr (E4M3) {
          const int d = (ks >> 2) * 64 + t * 16 + (ks & 3) * 4;   // four numbers in a row: k = 2t, 2t+1, 2t+8, 2t+9
          if (r < rows && d < p.dim) {
            const uint2 x = *reinterpret_cast<const uint2*>(src + d * 2);
            q[ks][half] = x.x;
            q[ks][half + 2] = x.y;
          }
        } else {
          if (r < rows && ks < steps) {
            q[ks][half] = *reinterpret_cast<const uint32_t*>(src + (ks * 16 + t * 2) * 2);
            q[ks][half + 2] = *reinterpret_cast<const uint32_t*>(src + (ks * 16 + t * 2 + 8) * 2);
          }
        }
      }
      if constexpr (E4M3 && !std::is_same<T, __half>::value) {   // bfloat16 rows to float16
        auto pair = [](uint32_t x) { return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xFFFF0000u)); };
        float amax = 0.0f;
#pragma unroll
        for (int ks = 0; ks < kSteps; ++ks) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 f = pair(q[ks][half + 2 * e]);
            amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        float up;
        lift[half] = c * query_lift(amax, up);
#pragma unroll
        for (int ks = 0; ks < kSteps; ++ks) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 f = pair(q[ks][half + 2 * e]);
            const __half2 h2 = __floats2half2_rn(f.x * up, f.y * up);
            q[ks][half + 2 * e] = *reinterpret_cast<const uint32_t*>(&h2);
          }
        }
      }
    }
    const int sure = p.causal ? shift + 1 : lk;   // keys every row sees
    float o[kCols][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < kCols; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;

    for (; take.tile < end_tile && todo > 0; --todo) {
      cp_async_wait<kDecodeStages - 2>();
      __syncwarp();
      const uint32_t k_scale = k_scale_next, v_scale = v_scale_next;
      k_scale_next = k_scale_new;
      v_scale_next = v_scale_new;
      fetch(stage == 0 ? kDecodeStages - 1 : stage - 1);   // into the stage consumed last
      const int key0 = take.tile * kTile + warp * kSlab;
      const uint32_t ks_at = ring + stage * (2 * kHalf), vs_at = ks_at + kHalf;
      stage = stage + 1 == kDecodeStages ? 0 : stage + 1;
      const bool last = take.tile + 1 == end_tile;
      if (last) {
        ++take.tile;   // the pair's share ends; the cursor itself moves on below
      } else {
        cursor_next<kTile>(p, cache, take);
      }
      if (key0 >= lk) continue;
      float s[kKeyTiles][4];
#pragma unroll
      for (int n = 0; n < kKeyTiles; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
      if constexpr (E4M3) {
#pragma unroll
        for (int n = 0; n < kKeyTiles; ++n) {
#pragma unroll
          for (int i = 0; i < kSteps / 4; ++i) {
            const uint4 x = lds128(ks_at + lane_k[i] + n * 8 * kRowBytes);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              mma16816<M>(s[n], q[i * 4 + k], codes_low(w[k]), codes_high(w[k]));
            }
          }
        }
      } else {
        const int row = (lane & 7) + ((lane >> 4) << 3);
        const uint32_t row_at = ks_at + row * kRowBytes;
        const int swz = row & (kUnits < 8 ? kUnits - 1 : 7);
#pragma unroll
        for (int ks = 0; ks < kSteps; ++ks) {
          if (ks < steps) {
            uint32_t b[4];
            ldmatrix_x4<false>(row_at + (((ks * 2 + ((lane >> 3) & 1)) ^ swz) << 4), b);
            mma16816<M>(s[0], q[ks], b[0], b[1]);
            mma16816<M>(s[1], q[ks], b[2], b[3]);
          }
        }
      }
      // ---- scale, mask, running maximum --------------------------------------------------------------
      float top[2] = {-INFINITY, -INFINITY};
      const bool edge = key0 + kSlab > sure;
      const float k_factor = scale_of_byte(k_scale), v_factor = scale_of_byte(v_scale), v_exp = scale_exponent(v_scale);   // of key `lane`
#pragma unroll
      for (int n = 0; n < kKeyTiles; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int at = n * 8 + t * 2 + e, key = key0 + at;
          float f = 1.0f, weight = 0.0f;
          if constexpr (E4M3) {
            f = __shfl_sync(0xffffffffu, k_factor, at);
            weight = __shfl_sync(0xffffffffu, v_exp, at);
          }
#pragma unroll
          for (int half = 0; half < HALVES; ++half) {
            float x = s[n][half * 2 + e] * lift[half];
            if constexpr (E4M3) x *= f;
            if (edge && key >= limit[half]) x = -INFINITY;
            s[n][half * 2 + e] = x;
            top[half] = fmaxf(top[half], x + weight);
          }
        }
      }
#pragma unroll
      for (int half = 0; half < HALVES; ++half) {
        top[half] = fmaxf(top[half], __shfl_xor_sync(0xffffffffu, top[half], 1));
        top[half] = fmaxf(top[half], __shfl_xor_sync(0xffffffffu, top[half], 2));
      }
      // O follows a row's maximum once it grew by more than 2^8 (or for the first time).
      if (__any_sync(0xffffffffu, top[0] - m[0] > 8.0f || (HALVES == 2 && top[1] - m[1] > 8.0f))) {
        float f[2] = {1.0f, 1.0f};
#pragma unroll
        for (int half = 0; half < HALVES; ++half) {
          const float next = fmaxf(m[half], top[half]);
          f[half] = next == -INFINITY ? 1.0f : exp2_fast(m[half] - next);
          m[half] = next;
          l[half] *= f[half];
        }
#pragma unroll
        for (int j = 0; j < kCols; ++j) {
          o[j][0] *= f[0];
          o[j][1] *= f[0];
          if (HALVES == 2) {
            o[j][2] *= f[1];
            o[j][3] *= f[1];
          }
        }
      }
      const float base[2] = {m[0] == -INFINITY ? 0.0f : m[0] - kProbLift<M>, m[1] == -INFINITY ? 0.0f : m[1] - kProbLift<M>};
      uint32_t pa[kKeyTiles / 2][4] = {};   // P as A operands of 16 keys each
#pragma unroll
      for (int n = 0; n < kKeyTiles; ++n) {
        float v0 = 1.0f, v1 = 1.0f;
        if constexpr (E4M3) {
          v0 = __shfl_sync(0xffffffffu, v_factor, n * 8 + t * 2);
          v1 = __shfl_sync(0xffffffffu, v_factor, n * 8 + t * 2 + 1);
        }
#pragma unroll
        for (int half = 0; half < HALVES; ++half) {
          float e0 = exp2_fast(s[n][half * 2] - base[half]), e1 = exp2_fast(s[n][half * 2 + 1] - base[half]);
          l[half] += e0 + e1;
          if constexpr (E4M3) {
            const int key = key0 + n * 8 + t * 2;
            // a masked key's scale may be NaN
            e0 = edge && key >= limit[half] ? 0.0f : e0 * v0;
            e1 = edge && key + 1 >= limit[half] ? 0.0f : e1 * v1;
          }
          if constexpr (std::is_same<M, __half>::value) {
            const __half2 h2 = __floats2half2_rn(e0, e1);
            pa[n >> 1][(n & 1) * 2 + half] = *reinterpret_cast<const uint32_t*>(&h2);
          } else {
            const __nv_bfloat162 h2 = __floats2bfloat162_rn(e0, e1);
            pa[n >> 1][(n & 1) * 2 + half] = *reinterpret_cast<const uint32_t*>(&h2);
          }
        }
      }
      // ---- O += P V ----------------------------------------------------------------------------------
      if constexpr (E4M3) {
        constexpr int kWords = kCols / 4;   // a thread's codes of one key: columns d = g4 * kCols + 0 .. kCols - 1
#pragma unroll
        for (int k = 0; k < kKeyTiles / 2; ++k) {
          uint32_t w[4][kWords];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t at = vs_at + lane_v + (k * 16 + (i & 1) + (i >> 1) * 8) * kRowBytes;
            if constexpr (BIG) {
              const uint4 x = lds128(at);
              w[i][0] = x.x, w[i][1] = x.y, w[i][2] = x.z, w[i][3] = x.w;
            } else {
              const uint2 x = lds64(at);
              w[i][0] = x.x, w[i][1] = x.y;
            }
          }
#pragma unroll
          for (int j = 0; j < kCols; j += 2) {   // bytes j, j + 1 of the one key and of the other, in turn
            const uint32_t sel = (j & 2) ? 0x7362 : 0x5140;
            const uint32_t x = __byte_perm(w[0][j >> 2], w[1][j >> 2], sel), y = __byte_perm(w[2][j >> 2], w[3][j >> 2], sel);
            mma16816<M>(o[j], pa[k], codes_low(x), codes_low(y));
            mma16816<M>(o[j + 1], pa[k], codes_high(x), codes_high(y));
          }
        }
      } else {
        const int row = lane & 15;
        const uint32_t row_at = vs_at + row * kRowBytes;
        const int swz = row & (kUnits < 8 ? kUnits - 1 : 7);
#pragma unroll
        for (int j = 0; j < kCols / 2; ++j) {
          if (j < steps) {
            uint32_t b[4];
            ldmatrix_x4<true>(row_at + (((j * 2 + (lane >> 4)) ^ swz) << 4), b);
            mma16816<M>(o[2 * j], pa[0], b[0], b[1]);
            mma16816<M>(o[2 * j + 1], pa[0], b[2], b[3]);
          }
        }
      }
      __syncwarp();
    }

    // ---- the four warps' shares meet ------------------------------------------------------------------
#pragma unroll
    for (int half = 0; half < HALVES; ++half) {
      l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
      l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
      if (t == 0) {
        join_m[warp * kDecodeRows + g4 + half * 8] = m[half];
        join_l[warp * kDecodeRows + g4 + half * 8] = l[half];
      }
    }
    const bool whole = first_tile == 0 && end_tile == pair_n;
    // The pair's tiles are [pair_t0, pair_t0 + pair_n) of the list; the CTAs first_cta .. last_cta hold them.
    const int64_t here = t1 - todo - (end_tile - first_tile);   // list index of first_tile
    const int64_t pair_t0 = here - first_tile;
    const int64_t first_cta = ((pair_t0 + 1) * ctas - 1) / total, last_cta = ((pair_t0 + pair_n) * ctas - 1) / total;
    auto slot_of = [&](int64_t cta) { return 2 * cta + (cta == first_cta && range_start(cta) < pair_t0 ? 1 : 0); };
    const int max_rows = p.max_q * p.group;
    float* const parts = reinterpret_cast<float*>(workspace + kServingCounterBytes);   // [slots][max_rows][dim]
    float2* const stats = reinterpret_cast<float2*>(parts + static_cast<int64_t>(2 * gridDim.x) * max_rows * p.dim);
    const int quads = p.dim / 4;
    auto store_row = [&](int r, int d, float4 x, float mr, float lr) {   // the pair's result
      const int i = r / p.group, h = head * p.group + r - i * p.group;
      const float inv = lr == 0.0f ? 0.0f : 1.0f / lr;
      if (lr == 0.0f) x = make_float4(0, 0, 0, 0);
      uint2 out;
      if constexpr (E4M3) {
        out = make_uint2(pack_finite<T>(x.x * inv, x.y * inv), pack_finite<T>(x.z * inv, x.w * inv));
      } else {
        const T four[4] = {from_f32<T>(x.x * inv), from_f32<T>(x.y * inv), from_f32<T>(x.z * inv), from_f32<T>(x.w * inv)};
        out = *reinterpret_cast<const uint2*>(four);
      }
      *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.o) + (q0 + i) * p.o_token + h * p.o_head + d) = out;
      if (d == 0 && p.lse != nullptr) {
        p.lse[static_cast<int64_t>(q0 + i) * p.heads + h] = lr == 0.0f ? -INFINITY : (mr - kProbLift<M>) * 0.6931471805599453f + logf(lr);
      }
    };
    for (int r0 = 0; r0 < rows; r0 += kDecodeJoinRows) {
      const int half = r0 >> 3;
      if (r0 > 0) __syncthreads();
      float* const mine = join_o + (warp * kDecodeJoinRows + (g4 & (kDecodeJoinRows - 1))) * kDim;
      const bool turn = (g4 & ~(kDecodeJoinRows - 1)) == (r0 & 7);
#pragma unroll
      for (int j = 0; turn && j < kCols; ++j) {
        const float x = half ? o[j][2] : o[j][0], y = half ? o[j][3] : o[j][1];
        if constexpr (E4M3) {
          mine[t * 2 * kCols + j] = x;
          mine[(t * 2 + 1) * kCols + j] = y;
        } else {
          *reinterpret_cast<float2*>(mine + j * 8 + t * 2) = make_float2(x, y);
        }
      }
      __syncthreads();
      for (int i = tid; i < kDecodeJoinRows * quads; i += kDecodeWarps * 32) {
        const int rr = i / quads, r = r0 + rr, d = (i - rr * quads) * 4;
        if (r >= rows) break;
        float mr = -INFINITY, lr = 0.0f;
        for (int w = 0; w < kDecodeWarps; ++w) mr = fmaxf(mr, join_m[w * kDecodeRows + r]);
        float4 sum = make_float4(0, 0, 0, 0);
        for (int w = 0; w < kDecodeWarps; ++w) {
          const float mw = join_m[w * kDecodeRows + r], f = mw == -INFINITY ? 0.0f : exp2_fast(mw - mr);
          const float4 x = *reinterpret_cast<const float4*>(join_o + (w * kDecodeJoinRows + rr) * kDim + d);
          lr += f * join_l[w * kDecodeRows + r];
          sum.x += f * x.x;
          sum.y += f * x.y;
          sum.z += f * x.z;
          sum.w += f * x.w;
        }
        if (whole) {
          store_row(r, d, sum, mr, lr);
        } else {
          const int64_t at = slot_of(blockIdx.x) * max_rows + r;
          *reinterpret_cast<float4*>(parts + at * p.dim + d) = sum;
          if (d == 0) stats[at] = make_float2(mr, lr);
        }
      }
    }
    if (!whole) {
      __threadfence();
      __syncthreads();
      const int n = static_cast<int>(last_cta - first_cta) + 1;
      if (tid == 0) last_flag = atomicInc(reinterpret_cast<uint32_t*>(workspace) + first_cta, n - 1) == static_cast<uint32_t>(n - 1);
      __syncthreads();
      if (last_flag) {   // every other share is there: the counter is back at zero
        __threadfence();
        for (int i = tid; i < rows * quads; i += kDecodeWarps * 32) {
          const int r = i / quads, d = (i - r * quads) * 4;
          float mr = -INFINITY, lr = 0.0f;
          float4 sum = make_float4(0, 0, 0, 0);
          constexpr int kTogether = 8;   // shares in flight: one after the other, 37 of them took 15 us
          for (int64_t cta0 = first_cta; cta0 <= last_cta; cta0 += kTogether) {
            float2 ml[kTogether];
            float4 x[kTogether];
#pragma unroll
            for (int e = 0; e < kTogether; ++e) {
              ml[e] = make_float2(-INFINITY, 0.0f);
              x[e] = make_float4(0, 0, 0, 0);
              if (cta0 + e <= last_cta) {
                const int64_t at = slot_of(cta0 + e) * max_rows + r;
                ml[e] = __ldcg(&stats[at]);
                x[e] = __ldcg(reinterpret_cast<const float4*>(parts + at * p.dim + d));
              }
            }
            float next = mr;
#pragma unroll
            for (int e = 0; e < kTogether; ++e) next = fmaxf(next, ml[e].x);
            const float keep = mr == -INFINITY ? 0.0f : exp2_fast(mr - next);
            mr = next;
            lr *= keep;
            sum = make_float4(sum.x * keep, sum.y * keep, sum.z * keep, sum.w * keep);
#pragma unroll
            for (int e = 0; e < kTogether; ++e) {
              const float f = ml[e].x == -INFINITY ? 0.0f : exp2_fast(ml[e].x - mr);
              lr += f * ml[e].y;
              sum.x += f * x[e].x;
              sum.y += f * x[e].y;
              sum.z += f * x[e].z;
              sum.w += f * x[e].w;
            }
          }
          store_row(r, d, sum, mr, lr);
        }
      }
    }
    __syncthreads();   // join_o and join_m are free for the next pair
    if (todo > 0) {
      --take.tile;   // the share's last tile: the cursor leaves the pair
      cursor_next<kTile>(p, cache, take);
    }
  }
  cp_async_wait<0>();
}

bool attention_decode_takes(const ServingProblem& p) { return static_cast<int64_t>(p.max_q) * p.group <= kDecodeRows; }

size_t attention_decode_workspace(const ServingProblem& p) {
  const size_t rows = static_cast<size_t>(2 * kDecodeMostCtas) * p.max_q * p.group;
  return kServingCounterBytes + rows * p.dim * sizeof(float) + rows * sizeof(float2);
}

int launch_attention_decode(const ServingProblem& p, const PagedCache& cache, bool e4m3, void* workspace, cudaStream_t stream) {
  int* status = nullptr;
  if (int rc = device_status_word(&status)) return rc;
  const bool big = p.dim > 64;
  const size_t smem = static_cast<size_t>(kDecodeWarps) * (kDecodeStages * 2 * (big ? 4096 : 2048) + kDecodeJoinRows * (big ? 128 : 64) * 4 + 2 * kDecodeRows * 4);
  auto launch = [&](auto kernel) -> int {
    static SmemOptIn opted;
    if (int rc = opted.once(kernel, smem)) return rc;
    kernel<<<kDecodeMostCtas, kDecodeWarps * 32, smem, stream>>>(p, cache, static_cast<uint8_t*>(workspace), status);
    return FB200_OK;
  };
  auto rows = [&](auto type, auto big_dim, auto codes) -> int {
    using T = decltype(type);
    constexpr bool kBig = decltype(big_dim)::value, kCodes = decltype(codes)::value;
    return p.max_q * p.group <= 8 ? launch(attention_decode_kernel<T, kBig, kCodes, 1>) : launch(attention_decode_kernel<T, kBig, kCodes, 2>);
  };
  auto dims = [&](auto type, auto codes) -> int { return big ? rows(type, std::true_type(), codes) : rows(type, std::false_type(), codes); };
  auto kind = [&](auto type) -> int { return e4m3 ? dims(type, std::true_type()) : dims(type, std::false_type()); };
  const int rc = p.dtype == FB200_BF16 ? kind(__nv_bfloat16()) : kind(__half());
  if (rc != FB200_OK) return rc;
  return after_launch("attention_decode_kernel");
}

}  // namespace fb200
