// Attention of packed sequences on the tensor cores: 128 query rows at a time over tiles of 128 keys,
//   S = Q K^T,  m' = max(m, rowmax S),  P = 2^(c S - c m'),  l = l 2^(c m - c m') + rowsum P,
//   O = O 2^(c m - c m') + P V,  result O / l,   c = scale * log2(e),
// one pass over the keys with the running maximum and sum in fp32.
//
// A row is a (token, query head) pair: the query heads that share a kv head lie next to each other in
// the tile (128 / group tokens of `group` heads), so a key tile is read once for all of them and short
// chunks of new tokens still fill the tensor core's 128 rows.
//
// A CTA holds two such tiles ("stages") and walks the keys both see.  Roles:
//   warps 0-7, 8-15  softmax of stage 0 and 1, two threads per row = TMEM lane with 64 keys each:
//                    tcgen05.ld of the scores, maximum, exponentials, tcgen05.st of P (16 bit); an eighth of
//                    the exponentials is a polynomial on the FMA pipe instead of ex2 on the XU pipe (none:
//                    134 us where this takes 123, 2x4096 d64; a quarter: 126)
//   warp 16          every tcgen05.mma: S_s = Q_s K^T (both operands in shared memory), O_s += P_s V with
//                    P as the A operand in TMEM, so P never passes through shared memory
//   warp 17          TMA: Q once, K and V tiles through a ring; a paged cache one box per page
// While the threads of one stage compute exponentials the tensor core works for the other one.  TMEM has
// 512 columns.  head_dim up to 64: S0, S1 (128 each), O0, O1, P0, P1 (64 each), and the scores of the next
// tile are computed as soon as the threads have read those of this one.  Above: S0, S1, O0, O1 (128 each)
// leave no room, P lies over S, and the next scores follow P V; P is handed over in halves so that only
// the second half of P V lies between the two.
// O is only rescaled when a row's maximum grew by more than 2^8 since the last time (P stays below 2^8 then,
// float16 P, which is taken times 2^7, below 2^15: fp32 sums and the 16-bit types hold that).
//
// Bounds: 4 * pairs * head_dim FLOP against the tensor pipe; one exponential per pair against the
// XU pipe (16 per SM and cycle: 1024 cycles for a 128 x 128 tile whose two products take 512 to 1024).
// Shared memory is next: a score instruction of N columns reads (128 + N) * 32 bytes at 128 bytes per cycle,
// which for N = 64 is 48 cycles against 32 in the tensor pipe (measured), for N = 128 the 64 of both.  So
// scores are computed 128 keys at a time (steps of 64 took 584 us where these take 518, 2x8192 d128).
#include <cuda.h>

#include <type_traits>

#include "attention_serving.cuh"
#include "sm100_ptx.cuh"

namespace fb200 {

int make_tmap_4d(CUtensorMap* map, const void* ptr, int dtype, const int64_t (&dims)[4], const int64_t (&stride_bytes)[3],
                 const int (&box)[4]);
int device_status_word(int** dev_ptr);

using namespace sm100;

constexpr int kTileRows = 128;
constexpr int kTileKeys = 128;
constexpr int kSoftmaxWarps = 16;             // two threads per row of each stage, 64 of the 128 keys each
constexpr int kMmaWarp = kSoftmaxWarps, kCopyWarp = kSoftmaxWarps + 1;
constexpr int kCodeWarp = kCopyWarp + 1, kCodeWarps = 2;   // of an e4m3 cache (20 warps are five per scheduler, as 18 are)
constexpr int kRawSlots = 3;                  // tiles of codes on their way
__host__ __device__ constexpr int tiles_threads(bool e4m3) { return (kSoftmaxWarps + 2 + (e4m3 ? kCodeWarps : 0)) * 32; }
__host__ __device__ constexpr int tiles_slots(int spans, bool e4m3) { return spans == 1 ? (e4m3 ? 6 : 8) : e4m3 ? 3 : 5; }
constexpr int kScaleTiles = 4;                // tiles whose scales are kept: a tile's are read until the scores two tiles on
constexpr int kHalfKeys = kTileKeys / 2;
constexpr int kSpanBytes = kTileRows * 128;   // 128 rows of 64 16-bit elements
constexpr float kRescaleStep = 8.0f;          // log2 of the growth of a row's maximum that O follows at once

enum TilesFault : int {
  kFaultTilesQuery = 331,
  kFaultTilesKeys = 332,
  kFaultTilesScores = 333,
  kFaultTilesProbs = 334,
  kFaultTilesRing = 335,
  kFaultTilesOutput = 336,
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^x without the XU pipe: x = n + f with f in [-1/2, 1/2] by adding 1.5 * 2^23 (n stands in the low bits of
// the sum), 2^f by the polynomial of degree 5 with the least largest relative error (1.6e-7 in fp32
// arithmetic; found by reweighted least squares, constant term 1), times 2^n from its exponent field.  From
// -127 down that field is 0, and so is the result.  A NaN stays one in every step: whatever the bits of n are
// then, the last one multiplies with them (adding n to the polynomial's exponent made a finite number of it).
__device__ __forceinline__ float2 exp2_poly(float2 x) {
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x.x));   // -127
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x.y));
  const float2 big = make_float2(12582912.0f, 12582912.0f), t = __fadd2_rn(x, big);
  const float2 n = __fadd2_rn(t, make_float2(-12582912.0f, -12582912.0f));
  const float2 f = __fadd2_rn(x, make_float2(-n.x, -n.y));
  auto poly = [](float z) {   // scalar: the coefficients are immediates, where packed pairs would hold them in registers
    float y = fmaf(0.0013264727f, z, 0.009671513f);
    y = fmaf(y, z, 0.055507336f);
    y = fmaf(y, z, 0.24022242f);
    y = fmaf(y, z, 0.693147f);
    return fmaf(y, z, 1.0f);
  };
  auto power = [](float z) { return __uint_as_float((__float_as_uint(z) << 23) + 0x3F800000u); };
  return __fmul2_rn(make_float2(poly(f.x), poly(f.y)), make_float2(power(t.x), power(t.y)));
}
template <typename T> __device__ __forceinline__ uint32_t pack_pair(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack_pair<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack_pair<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T, bool E4M3> __device__ __forceinline__ uint32_t pack_result(float lo, float hi) {
  return E4M3 ? pack_finite<T>(lo, hi) : pack_pair<T>(lo, hi);
}

// A CTA's share of the work.
struct TilesItem {
  int seq, block, q0, lq, rows, k0, lk;   // rows: of the lq query rows, those that are computed
};

// Keys that the block ending before token `end` sees.
__device__ __forceinline__ int keys_seen(int causal, int end, int lq, int lk) {
  return causal ? max(0, min(lk, end + lk - lq)) : lk;
}

// Item `rank` of the blocks of `tokens` query tokens of all sequences in order of falling cost (tiles of
// keys): the long ones start first, so that the last CTAs to run are short ones.  The number of blocks
// that cost more than c tiles is a closed form per sequence; a binary search over c finds the cost of
// the rank, a scan over the sequences the block.  A sequence has blocks for its first max_q rows only, so that
// one with more rows takes no other's place in the grid.  Run by one warp; returns false past the last item.
template <bool PAGED>
__device__ bool find_item(const ServingProblem& p, const PagedCache& cache, int rank, int tokens, uint32_t tokens_inverse,
                          TilesItem& item) {
  const int lane = threadIdx.x & 31;
  // y / tokens for 0 <= y < 2^31: tokens_inverse = floor(2^32 / tokens) gives it or one less
  auto over_tokens = [&](int y) {
    const int q = static_cast<int>(__umulhi(static_cast<uint32_t>(y), tokens_inverse));
    return q + (y - q * tokens >= tokens ? 1 : 0);
  };
  struct Seq {
    int q0, lq, rows, k0, lk, blocks;
  };
  auto load = [&](int s) {
    Seq q{0, 0, 0, 0, 0, 0};
    if (s < p.n_seqs) {
      serving_lengths<PAGED>(p, cache, s, q.q0, q.lq, q.k0, q.lk);
      q.rows = min(q.lq, p.max_q);
      q.blocks = over_tokens(q.rows + tokens - 1);
    }
    return q;
  };
  const Seq mine = load(lane);   // sequence `lane` stays in registers
  auto sequence = [&](int s) { return s < 32 ? mine : load(s); };
  // blocks of a sequence that see more than 128 * c keys
  auto above = [&](const Seq& q, int c) {
    if (c < 0) return q.blocks;
    if (q.lk <= c * kTileKeys) return 0;
    if (!p.causal) return q.blocks;
    const int y = c * kTileKeys - q.lk + q.lq;   // blocks that end at or before token y see no more
    return y >= q.rows ? 0 : q.blocks - over_tokens(max(y, 0));
  };
  auto total = [&](int c) {
    int sum = above(mine, c);
    for (int s = lane + 32; s < p.n_seqs; s += 32) sum += above(load(s), c);
    return __reduce_add_sync(0xffffffffu, sum);
  };
  int most = mine.lk;
  for (int s = lane + 32; s < p.n_seqs; s += 32) most = max(most, load(s).lk);
  const int longest = __reduce_max_sync(0xffffffffu, most);
  if (rank >= total(-1)) return false;
  int lo = -1, hi = (longest + kTileKeys - 1) / kTileKeys;   // total(lo) > rank >= total(hi)
  int below = 0;                                             // total(hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1, n = total(mid);
    if (n > rank) lo = mid;
    else { hi = mid; below = n; }
  }
  // items of cost hi exactly, in sequence order: `rank - below` of them lie before this one
  int left = rank - below;
  for (int s0 = 0; s0 < p.n_seqs; s0 += 32) {
    const Seq q = sequence(s0 + lane);
    const int more = above(q, hi), n = above(q, hi - 1) - more;
    int upto = n;   // inclusive scan
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += x;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, upto > left);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const int block = q.blocks - more - n + (left - (upto - n));
      item.seq = s0 + src;
      item.block = __shfl_sync(0xffffffffu, block, src);
      item.q0 = __shfl_sync(0xffffffffu, q.q0, src);
      item.lq = __shfl_sync(0xffffffffu, q.lq, src);
      item.rows = __shfl_sync(0xffffffffu, q.rows, src);
      item.k0 = __shfl_sync(0xffffffffu, q.k0, src);
      item.lk = __shfl_sync(0xffffffffu, q.lk, src);
      return true;
    }
    left -= __shfl_sync(0xffffffffu, upto, 31);
  }
  return false;
}

// Records sequences that are cut.  Run by one warp of the call, out of line: inlined it took registers from the
// loops over the tiles (2 x 8192 538 -> 547 us, e4m3 chunks of float16 405 -> 421).
template <bool PAGED>
__device__ __noinline__ void check_lengths(const int32_t* cu_q, const int32_t* keys, int n_seqs, int q_rows, int most_keys, int max_q, int* status) {
  for (int s = threadIdx.x & 31; s < n_seqs; s += 32) {
    if (!lengths_fit<PAGED>(cu_q, keys, s, q_rows, most_keys) || cu_q[s + 1] - cu_q[s] > max_q) record_fault(status, kFaultBadLength);
  }
}

// Barriers, the swap of row maxima and an e4m3 cache's scales, in front of the tiles.
__host__ __device__ constexpr uint32_t tiles_small_bytes(int spans, bool e4m3) {
  return 320 + (spans == 1 ? 2 : 1) * 4 * kTileRows * 4 + (e4m3 ? kScaleTiles * 3 * kTileKeys * 4 : 0);
}

// Few blocks over many keys: the keys of a block go to several CTAs, `tiles` of 128 to each, which leave
// unnormalised O, maximum (in the exponent's units) and sum for attention_tiles_join_kernel.
struct TilesSplit {
  int parts, tiles;   // CTAs per block, tiles per CTA; parts 1: not split
  float* o;           // [parts][q_rows][heads][dim]
  float2* stats;      // [parts][q_rows][heads]
};

// A place in the ring; K and V tiles alternate, so each steps by two.
struct RingPos {
  int slot;
  uint32_t phase;
  __device__ __forceinline__ void next(int slots) {
    slot += 2;
    if (slot >= slots) {
      slot -= slots;
      phase ^= 1u;
    }
  }
};

template <typename T, int SPANS, bool PAGED, bool E4M3>
__global__ void __launch_bounds__(tiles_threads(E4M3), 1)
attention_tiles_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                       const __grid_constant__ CUtensorMap tmap_v, const ServingProblem p, const PagedCache cache,
                       const TilesSplit split, int tile_tokens, uint32_t tokens_inverse, int box_keys, int* status) {
  using M = typename std::conditional<E4M3, __half, T>::type;   // type of the operands
  constexpr bool kLift = E4M3 && !std::is_same<T, __half>::value;   // the query rows become float16
  constexpr uint32_t kFmt = std::is_same<M, __half>::value ? kFmtF16 : kFmtBF16;
  constexpr int kSlotBytes = SPANS * kSpanBytes;
  constexpr int kSlots = tiles_slots(SPANS, E4M3);
  constexpr bool kApart = SPANS == 1;   // P has columns of its own
  constexpr uint32_t kTmemO = 2 * kTileKeys, kTmemP = kApart ? kTmemO + 128 : 0, kTmemPStage = kApart ? 64 : kTileKeys;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t bars = smem_u32(smem_raw), base = (bars + tiles_small_bytes(SPANS, E4M3) + 1023u) & ~1023u;   // swizzle atoms are 1024 bytes
  uint8_t* base_ptr = smem_raw + (base - bars);
  const uint32_t q_s = base, ring = base + 2 * kSlotBytes;
  const uint32_t bar_q = bars, full = bars + 8, freed = full + 8 * kSlots, bar_s = freed + 8 * kSlots, bar_r = bar_s + 16,
                 bar_p = bar_r + 16, bar_o = bar_p + 32, raw_full = bar_o + 16, raw_freed = raw_full + 8 * kRawSlots, bar_lift = raw_freed + 8 * kRawSlots, tmem_slot = bar_lift + 8;
  const uint32_t raw_ring = ring + kSlots * kSlotBytes;
  uint8_t* const after = smem_raw + (tmem_slot - bars);
  volatile uint32_t* const tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(after);
  TilesItem* const item_ptr = reinterpret_cast<TilesItem*>(after + 16);
  int* const found_ptr = reinterpret_cast<int*>(after + 16 + sizeof(TilesItem));
  float* const share = reinterpret_cast<float*>(smem_raw + 320);   // [tile parity, P apart only][stage][half][row]: maxima, then sums
  float* const scales = share + (kApart ? 2 : 1) * 4 * kTileRows;          // [tile % kScaleTiles][K, V, exponent of V][key]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = blockIdx.x % split.parts, pair = blockIdx.x / split.parts, head = pair % p.kv_heads;
  // of the softmax threads, worked out while the item is looked for
  const int row = threadIdx.x & 127, in_tile = row / p.group;
  if (warp == 0) {
    TilesItem it;
    const bool found = find_item<PAGED>(p, cache, pair / p.kv_heads, 2 * tile_tokens, tokens_inverse, it);
    if (lane == 0) {
      if (found) *item_ptr = it;
      *found_ptr = found;
    }
  } else if (warp == kMmaWarp && lane == 0) {
    mbar_init(bar_q, 1);
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(full + 8 * i, E4M3 ? kCodeWarps : 1);
      mbar_init(freed + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_s + 8 * i, 1);
      mbar_init(bar_r + 8 * i, kSoftmaxWarps / 2);
      mbar_init(bar_p + 16 * i, 4);
      mbar_init(bar_p + 16 * i + 8, 4);
      mbar_init(bar_o + 8 * i, 1);
    }
    mbar_init(bar_lift, kSoftmaxWarps);
    for (int i = 0; E4M3 && i < kRawSlots; ++i) {
      mbar_init(raw_full + 8 * i, 1);
      mbar_init(raw_freed + 8 * i, kCodeWarps);
    }
    mbar_fence_init();
  } else if (warp == kCopyWarp) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tcgen05_fence_before_sync();
  __syncthreads();
  tcgen05_fence_after_sync();
  const uint32_t tmem = __reduce_max_sync(0xffffffffu, *tmem_slot_ptr);
  const TilesItem item = *item_ptr;
  const bool found = *found_ptr != 0;
  const int token0 = item.block * 2 * tile_tokens;
  int tiles[2];   // of keys that each stage's rows see
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int first = token0 + s * tile_tokens;
    tiles[s] = found && first < item.rows
                   ? (keys_seen(p.causal, min(item.rows, first + tile_tokens), item.lq, item.lk) + kTileKeys - 1) / kTileKeys
                   : 0;
  }
  const int all = max(tiles[0], tiles[1]);   // stage 1's rows come later: it sees as much, unless it has none
  // this CTA's part of them
  const bool parted = split.parts > 1 && all > split.tiles;
  const int tile0 = part * split.tiles, key0 = tile0 * kTileKeys;
  const bool work = found && (part == 0 || tile0 < all);
  if (split.parts > 1) {
    const int room = part == split.parts - 1 ? 0x7fffffff : split.tiles;   // the last part takes what max_kv did not foresee
    tiles[0] = max(0, min(tiles[0] - tile0, room));
    tiles[1] = max(0, min(tiles[1] - tile0, room));
  }
  const int most = max(tiles[0], tiles[1]);

  if (warp == kCopyWarp) {
    // ---- copies ----------------------------------------------------------------------------------
    if (most > 0) {
      if (lane == 0) {
        const int live_stages = (tiles[0] > 0) + (tiles[1] > 0);
        mbar_arrive_expect_tx(bar_q, static_cast<uint32_t>(live_stages * tile_tokens * p.group * 128 * SPANS));
        for (int s = 0; s < 2; ++s) {
          if (tiles[s] == 0) continue;
          for (int x = 0; x < SPANS; ++x) {
            tma_load_4d(q_s + s * kSlotBytes + x * kSpanBytes, &tmap_q, bar_q, x * 64, 0, item.q0 + token0 + s * tile_tokens, head);
          }
        }
      }
      __syncwarp();
      bool live = true;
      // K and V of tile n / 2 in turn: into the ring, or as codes into the raw ring
      constexpr int kInto = E4M3 ? kRawSlots : kSlots, kIntoBytes = E4M3 ? kSpanBytes : kSlotBytes, kBoxes = E4M3 ? 1 : SPANS;
      const uint32_t into = E4M3 ? raw_ring : ring, into_full = E4M3 ? raw_full : full, into_freed = E4M3 ? raw_freed : freed;
      for (int n = 0; live && n < 2 * most; ++n) {
        const int slot = n % kInto, use = n / kInto;
        const uint32_t dst = into + slot * kIntoBytes, bar = into_full + 8 * slot;
        const void* map = (n & 1) ? static_cast<const void*>(&tmap_v) : &tmap_k;
        const int key = key0 + (n >> 1) * kTileKeys + lane * box_keys;
        const bool mine = lane * box_keys < kTileKeys && (!PAGED || key < item.lk);
        const int boxes = __popc(__ballot_sync(0xffffffffu, mine));
        int page = 0, row = item.k0 + key;
        if (PAGED && mine) {
          page = page_number(cache, item.seq, key >> cache.page_shift, status);
          row = key & ((1 << cache.page_shift) - 1);
        }
        if (use > 0) live = mbar_wait_lanes(into_freed + 8 * slot, (use - 1) & 1, status, kFaultTilesRing);
        if (!live) break;
        if (lane == 0) mbar_arrive_expect_tx(bar, static_cast<uint32_t>(boxes * box_keys * 128 * kBoxes));
        __syncwarp();
        if (mine) {
          for (int x = 0; x < kBoxes; ++x) {
            tma_load_4d(dst + x * kSpanBytes + lane * box_keys * 128, map, bar, x * 64, row, head, page);
          }
        }
      }
    }
    if (blockIdx.x == 0) {   // here it delays nothing: the last copies are on their way
      check_lengths<PAGED>(p.cu_q, PAGED ? p.kv_len : p.cu_kv, p.n_seqs, p.q_rows, PAGED ? most_cached(cache.table_stride, cache.page_shift) : p.kv_rows, p.max_q, status);
    }
    __syncwarp();
  } else if (E4M3 && warp >= kCodeWarp) {
    // ---- codes into float16 operands, rows behind the last key zero ------------------------------------
    if constexpr (E4M3) {
      constexpr int kUnits = SPANS * 4;   // 16 codes each
      const int me = (warp - kCodeWarp) * 32 + lane;
      // Scale bytes of keys me and me + 64, fetched one tile ahead, and the pages they lie in, two tiles ahead.
      int page_raw[2] = {0, 0};
      uint32_t k_scale[2], v_scale[2], k_scale_next[2], v_scale_next[2];
      auto pages_ahead = [&](int first) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int key = first + me + i * 64;
          page_raw[i] = key < item.lk ? cache.table[item.seq * cache.table_stride + (key >> cache.page_shift)] : 0;
        }
      };
      auto scales_ahead = [&](int first) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int key = first + me + i * 64;
          k_scale_next[i] = v_scale_next[i] = 0;
          if (key < item.lk) {   // (a page outside the cache is recorded by the copy warp)
            const int page = static_cast<uint32_t>(page_raw[i]) < static_cast<uint32_t>(cache.pages) ? page_raw[i] : 0;
            const int64_t at = scale_offset(cache, page, key, head);
            k_scale_next[i] = cache.k_scale[at];
            v_scale_next[i] = cache.v_scale[at];
          }
        }
      };
      if (most > 0) {
        pages_ahead(key0);
        scales_ahead(key0);
        pages_ahead(key0 + kTileKeys);
      }
      bool live = true;
      for (int n = 0; live && n < 2 * most; ++n) {
        const int slot = n % kSlots, use = n / kSlots, from = n % kRawSlots, key_tile = key0 + (n >> 1) * kTileKeys;
        if (!(n & 1)) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            k_scale[i] = k_scale_next[i];
            v_scale[i] = v_scale_next[i];
          }
          scales_ahead(key_tile + kTileKeys);
          pages_ahead(key_tile + 2 * kTileKeys);
        }
        if (use > 0) live = mbar_wait_lanes(freed + 8 * slot, (use - 1) & 1, status, kFaultTilesRing);
        live = live && mbar_wait_lanes(raw_full + 8 * from, (n / kRawSlots) & 1, status, kFaultTilesKeys);
        if (!live) break;
        uint8_t* const to = base_ptr + (ring - base) + slot * kSlotBytes;
        const uint8_t* const raw = base_ptr + (raw_ring - base) + from * kSpanBytes;
        // The rows a thread takes are multiples of 8 apart, so the swizzle is the same for all of them and
        // every address is a constant away from the first.
        constexpr int kApartRows = kCodeWarps * 32 / kUnits, kTakes = kTileKeys / kApartRows, kAhead = 8;
        const int row0 = me / kUnits, unit = me % kUnits, left = item.lk - key_tile - row0;   // rows from row0 on that exist
        const uint8_t* const in = raw + row0 * 128 + ((unit ^ (row0 & 7)) << 4);
        uint8_t* const out = to + (unit >> 2) * kSpanBytes + row0 * 128;
        const int out0 = (((unit & 3) * 2) ^ (row0 & 7)) << 4, out1 = (((unit & 3) * 2 + 1) ^ (row0 & 7)) << 4;
#pragma unroll
        for (int i0 = 0; i0 < kTakes; i0 += kAhead) {
          uint4 codes[kAhead];
#pragma unroll
          for (int i = 0; i < kAhead; ++i) codes[i] = *reinterpret_cast<const uint4*>(in + (i0 + i) * kApartRows * 128);
#pragma unroll
          for (int i = 0; i < kAhead; ++i) {
            const uint4 w = (i0 + i) * kApartRows < left ? codes[i] : make_uint4(0, 0, 0, 0);
            uint8_t* const at = out + (i0 + i) * kApartRows * 128;
            *reinterpret_cast<uint4*>(at + out0) = make_uint4(codes_low(w.x), codes_high(w.x), codes_low(w.y), codes_high(w.y));
            *reinterpret_cast<uint4*>(at + out1) = make_uint4(codes_low(w.z), codes_high(w.z), codes_low(w.w), codes_high(w.w));
          }
        }
        if (!(n & 1)) {
          float* const sc = scales + ((n >> 1) % kScaleTiles) * 3 * kTileKeys;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            sc[me + i * 64] = scale_of_byte(k_scale[i]);
            sc[kTileKeys + me + i * 64] = scale_of_byte(v_scale[i]);
            sc[2 * kTileKeys + me + i * 64] = scale_exponent(v_scale[i]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(raw_freed + 8 * from);
          mbar_arrive(full + 8 * slot);
        }
      }
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    // ---- products --------------------------------------------------------------------------------
    // Straight-line issue: descriptors and ring positions advance by additions in warp-uniform code (a
    // division per tile and a rolled loop over the k steps took 2900 cycles per 128 x 128 x 128 pair of
    // products, three times what the tensor core needs for it).
    // Equal in all lanes; a warp reduction leaves its result in a uniform register, which is where the
    // descriptors, addresses and loop bounds of the tensor instructions have to be.
    auto uniform = [](int x) { return __reduce_max_sync(0xffffffffu, x); };
    const int u_most = uniform(most), u_tiles[2] = {uniform(tiles[0]), uniform(tiles[1])}, keys_left = uniform(item.lk - key0);
    if (u_most > 0) {
      const int k_steps = p.dim / 16;
      const uint32_t idesc_s = make_instr_desc(kFmt, 0, 0, kTileRows, kTileKeys);
      const uint32_t idesc_o = make_instr_desc(kFmt, 0, 1, kTileRows, static_cast<uint32_t>(p.dim));
      const uint64_t q_desc = make_smem_desc_sw128(q_s, 16, 1024);
      const uint64_t k_desc = make_smem_desc_sw128(ring, 16, 1024);
      const uint64_t v_desc = make_smem_desc(ring, kSpanBytes, 1024, kLayoutSw128);
      bool live = mbar_wait_lanes(kLift ? bar_lift : bar_q, 0, status, kFaultTilesQuery);
      if constexpr (kLift) tcgen05_fence_after_sync();
      RingPos kp{0, 0}, vp{1, 0};   // of the K and the V tile that come next
      auto scores = [&](int s) {
        const uint64_t a = q_desc + static_cast<uint64_t>(s * (kSlotBytes / 16)), b = k_desc + static_cast<uint64_t>(kp.slot * (kSlotBytes / 16));
        const uint32_t d = tmem + s * kTileKeys;
        constexpr uint64_t kSpanUnits = kSpanBytes / 16;
#pragma unroll
        for (int x = 0; x < SPANS; ++x) {
          if (k_steps >= x * 4 + 4) {
            mma_f16_elect_x4<2, 2>(d, a + x * kSpanUnits, b + x * kSpanUnits, idesc_s, x > 0 ? 1u : 0u);
          } else {   // a head_dim that is no multiple of 64 ends inside a span
            for (int k = x * 4; k < k_steps; ++k) {
              const uint64_t at = x * kSpanUnits + (k & 3) * 2;
              mma_f16_elect(d, a + at, b + at, idesc_s, k > 0 ? 1u : 0u);
            }
          }
        }
        mma_commit_elect(bar_s + 8 * s);
      };
      auto values = [&](int s, int j) {
        const uint64_t b = v_desc + static_cast<uint64_t>(vp.slot * (kSlotBytes / 16));
        const uint32_t d = tmem + kTmemO + s * (SPANS * 64), a = tmem + kTmemP + s * kTmemPStage;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          live = live && mbar_wait_lanes(bar_p + 16 * s + 8 * half, j & 1, status, kFaultTilesProbs);
          if (!live) return;
          tcgen05_fence_after_sync();
          mma_f16_ts_elect_x4<8, 128>(d, a + half * 32, b + half * 512, idesc_o, (j > 0 || half > 0) ? 1u : 0u);
        }
        mma_commit_elect(bar_o + 8 * s);
      };
      live = live && mbar_wait_lanes(full, 0, status, kFaultTilesKeys);
      tcgen05_fence_after_sync();
      if (live) {
        if (u_tiles[0] > 0) scores(0);
        if (u_tiles[1] > 0) scores(1);
        mma_commit_elect(freed);
        kp.next(kSlots);
      }
      for (int j = 0; live && j < u_most; ++j) {
        const bool more = j + 1 < u_most;
        if (kApart && more) live = mbar_wait_lanes(full + 8 * kp.slot, kp.phase, status, kFaultTilesKeys);
        if (kApart && more && live) {
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            if (j + 1 >= u_tiles[s]) continue;
            live = live && mbar_wait_lanes(bar_r + 8 * s, j & 1, status, kFaultTilesScores);
            tcgen05_fence_after_sync();
            if (live) scores(s);
          }
        }
        live = live && mbar_wait_lanes(full + 8 * vp.slot, vp.phase, status, kFaultTilesKeys);
        if (!live) break;
        const int there = keys_left - j * kTileKeys;
        if (!E4M3 && there < kTileKeys) {
          // Rows behind the last key hold another sequence's values or none: their P is 0, but 0 times a
          // NaN is not.
          for (int i = lane; i < (kTileKeys - there) * 8 * SPANS; i += 32) {
            const int row = there + (i >> 3) % (kTileKeys - there), span = (i >> 3) / (kTileKeys - there);
            *reinterpret_cast<uint4*>(base_ptr + (ring - base) + vp.slot * kSlotBytes + span * kSpanBytes + row * 128 + (i & 7) * 16) =
                make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if (live && j < u_tiles[s]) values(s, j);
          if (!kApart && s == 0 && more) live = live && mbar_wait_lanes(full + 8 * kp.slot, kp.phase, status, kFaultTilesKeys);
          if (!kApart && live && j + 1 < u_tiles[s]) scores(s);
        }
        if (!live) break;
        mma_commit_elect(freed + 8 * vp.slot);
        vp.next(kSlots);
        if (more) {
          mma_commit_elect(freed + 8 * kp.slot);
          kp.next(kSlots);
        }
      }
    }
    __syncwarp();
  } else {
    // ---- softmax ---------------------------------------------------------------------------------
    const int s = warp >> 3, half = (warp >> 2) & 1, token = token0 + s * tile_tokens + in_tile;
    const int h = head * p.group + row - in_tile * p.group;
    const bool there = work && in_tile < tile_tokens && token < item.rows;
    const int limit = there ? keys_seen(p.causal, token + 1, item.lq, item.lk) - key0 : 0;   // keys this row sees from key0 on
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t t_s = lanes + s * kTileKeys + half * kHalfKeys, t_p = lanes + kTmemP + s * kTmemPStage + half * (kHalfKeys / 2);
    const uint32_t t_o = lanes + kTmemO + s * (SPANS * 64);
    float* const mine = share + (s * 2 + half) * kTileRows + row;
    const float* const other = share + (s * 2 + 1 - half) * kTileRows + row;
    // The two warps that hold the halves of the same 32 rows meet; true if both are still live, so that they
    // give up at the same tile.
    auto pair_sync = [&](bool ok) {
      uint32_t all;
      asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\tbar.red.and.pred q, %1, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}\n"
                   : "=r"(all) : "r"(1 + s * 4 + (warp & 3)), "r"(ok ? 1u : 0u) : "memory");
      return all != 0;
    };
    float c = p.scale * 1.4426950408889634f, m = -INFINITY, l = 0.0f;
    bool live = true;
    if constexpr (kLift) {   // this half of the row to float16, in place
      uint4* const q_row = reinterpret_cast<uint4*>(base_ptr + s * kSlotBytes + row * 128 + half * (SPANS == 2 ? kSpanBytes : 64));
      float amax = 0.0f;
      if (tiles[s] > 0) {
        live = mbar_wait_lanes(bar_q, 0, status, kFaultTilesQuery);
#pragma unroll
        for (int i = 0; i < SPANS * 4; ++i) {
          const uint4 x = q_row[i];
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(w[e] << 16)), fabsf(__uint_as_float(w[e] & 0xFFFF0000u))));
        }
      }
      *mine = amax;
      live = pair_sync(live);
      amax = fmaxf(amax, *other);
      live = pair_sync(live);   // read before it is written again
      float up;
      c *= query_lift(amax, up);
      if (tiles[s] > 0) {
#pragma unroll
        for (int i = 0; i < SPANS * 4; ++i) {
          const uint4 x = q_row[i];
          uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = pack_pair<__half>(__uint_as_float(w[e] << 16) * up, __uint_as_float(w[e] & 0xFFFF0000u) * up);
          q_row[i] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        fence_proxy_async_smem();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_lift);
    }
    const float to_exp = E4M3 ? 1.0f : c;   // of the maximum and the scores below to the exponent's units
    for (int j = 0; j < tiles[s]; ++j) {
      live = mbar_wait_lanes(bar_s + 8 * s, j & 1, status, kFaultTilesScores);
      tcgen05_fence_after_sync();
      uint32_t r[2][32];
      tmem_ld_32x32b_x32(t_s, r[0]);
      tmem_ld_32x32b_x32(t_s + 32, r[1]);
      tmem_ld_wait(r[0]);
      tmem_ld_wait(r[1]);
      if constexpr (kApart) {   // the next tile's scores may come
        tcgen05_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_r + 8 * s);
      }
      const float* const sc = scales + (j % kScaleTiles) * 3 * kTileKeys + half * kHalfKeys;
      if constexpr (E4M3) {   // the scale of K is the score's, that of V the probability's
        const float2 c2 = make_float2(c, c);
#pragma unroll
        for (int i = 0; i < kHalfKeys; i += 4) {
          const float4 k4 = *reinterpret_cast<const float4*>(sc + i);
          uint32_t* const x = &r[i >> 5][i & 31];
          const float2 lo = __fmul2_rn(__fmul2_rn(make_float2(__uint_as_float(x[0]), __uint_as_float(x[1])), c2), make_float2(k4.x, k4.y));
          const float2 hi = __fmul2_rn(__fmul2_rn(make_float2(__uint_as_float(x[2]), __uint_as_float(x[3])), c2), make_float2(k4.z, k4.w));
          x[0] = __float_as_uint(lo.x), x[1] = __float_as_uint(lo.y), x[2] = __float_as_uint(hi.x), x[3] = __float_as_uint(hi.y);
        }
      }
      const int visible = limit - j * kTileKeys - half * kHalfKeys;
      if (__any_sync(0xffffffffu, visible < kHalfKeys)) {
#pragma unroll
        for (int i = 0; i < kHalfKeys; ++i) {
          if (i >= visible) r[i >> 5][i & 31] = 0xFF800000u;   // -inf
        }
      }
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; E4M3 && i < kHalfKeys; i += 4) {   // of probability times value scale: see kScaleFloor
        const float4 e4 = *reinterpret_cast<const float4*>(sc + 2 * kTileKeys + i);
        const uint32_t* const x = &r[i >> 5][i & 31];
        const float2 lo = __fadd2_rn(make_float2(__uint_as_float(x[0]), __uint_as_float(x[1])), make_float2(e4.x, e4.y));
        const float2 hi = __fadd2_rn(make_float2(__uint_as_float(x[2]), __uint_as_float(x[3])), make_float2(e4.z, e4.w));
        top[(i >> 1) & 3] = fmaxf(top[(i >> 1) & 3], fmaxf(lo.x, lo.y));
        top[((i >> 1) & 3) + 1] = fmaxf(top[((i >> 1) & 3) + 1], fmaxf(hi.x, hi.y));
      }
#pragma unroll
      for (int i = 0; !E4M3 && i < kHalfKeys; i += 2) {
        top[(i >> 1) & 3] = fmaxf(top[(i >> 1) & 3], fmaxf(__uint_as_float(r[i >> 5][i & 31]), __uint_as_float(r[i >> 5][(i & 31) + 1])));
      }
      float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
      // P apart: the product of the tile before is done, so P's columns and O are free.  (P over S: the scores
      // of this tile were issued behind it.)
      if (kApart && j > 0) {
        live = mbar_wait_lanes(bar_o + 8 * s, (j - 1) & 1, status, kFaultTilesOutput) && live;
        tcgen05_fence_after_sync();
      }
      // The row's maximum: the halves swap theirs.  With P over S this also keeps one half's P from reaching
      // columns that the other has not read.  (A place of the swap is written again two tiles on, or, with P
      // over S, behind the next scores, which wait for both halves' P.)
      const int swap = kApart ? (j & 1) * 4 * kTileRows : 0;
      mine[swap] = mx;
      if constexpr (!kApart) tcgen05_fence_before_sync();
      live = pair_sync(live);
      if (!live) break;
      if constexpr (!kApart) tcgen05_fence_after_sync();
      mx = fmaxf(mx, other[swap]);
      if (j == 0) {
        m = mx;
      } else if (__any_sync(0xffffffffu, (mx - m) * to_exp > kRescaleStep)) {   // -inf - -inf compares false
        const float next = fmaxf(m, mx);
        const float f = next == -INFINITY ? 1.0f : ex2((m - next) * to_exp);
        m = next;
        l *= f;
        // the first half's threads do it, whose P the tensor core waits for before anything else
        for (int i = 0; half == 0 && i < p.dim; i += 16) {
          uint32_t x[16];
          tmem_ld_32x32b_x16(t_o + i, x);
          tmem_ld_wait(x);
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * f);
          tmem_st_32x32b_x16(t_o + i, x);
        }
      }
      const float mc = m == -INFINITY ? 0.0f : m * to_exp - kProbLift<M>;
      float2 sum = make_float2(0.0f, 0.0f);
      const float2 c2 = make_float2(c, c), nm2 = make_float2(-mc, -mc);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t out[16];
        float4 v4;   // scales of V
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          if (E4M3 && !(e & 2)) v4 = *reinterpret_cast<const float4*>(sc + kTileKeys + i * 32 + e);
          float2 x = make_float2(__uint_as_float(r[i][e]), __uint_as_float(r[i][e + 1]));
          x = E4M3 ? __fadd2_rn(x, nm2) : __ffma2_rn(x, c2, nm2);
          if ((e & 15) == 14) {
            x = exp2_poly(x);
          } else {
            x.x = ex2(x.x);
            x.y = ex2(x.y);
          }
          sum = __fadd2_rn(sum, x);
          if constexpr (E4M3) x = __fmul2_rn(x, (e & 2) ? make_float2(v4.z, v4.w) : make_float2(v4.x, v4.y));
          out[e >> 1] = pack_pair<M>(x.x, x.y);
        }
        tmem_st_32x32b_x16(t_p + i * 16, out);
      }
      l += sum.x + sum.y;
      tmem_st_wait();
      tcgen05_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_p + 16 * s + 8 * half);
    }
    const bool any = tiles[s] > 0;
    // (The wait before this one's phase is past: above, or by the scores of the last tile.)
    if (live && any) live = mbar_wait_lanes(bar_o + 8 * s, (tiles[s] - 1) & 1, status, kFaultTilesOutput);
    live = pair_sync(live);   // the last swap has been read
    *mine = l;
    live = pair_sync(live);
    l += *other;
    if (live) {
      tcgen05_fence_after_sync();
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const int64_t at = static_cast<int64_t>(item.q0 + token) * p.heads + h;
      // Rows go out through the stage's Q tile, which nothing reads any more (the last product is done, and the
      // scores before it): a warp that stored its 32 rows from registers, 16 bytes of each at a time, took
      // 3 K cycles a tile at head_dim 128.
      uint8_t* const rows = base_ptr + s * kSlotBytes;
      for (int i = half * 16; i < p.dim; i += 32) {
        uint32_t x[16];
        if (any) {
          tmem_ld_32x32b_x16(t_o + i, x);
          tmem_ld_wait(x);
        }
        if (parted) {
          float* const to = split.o + (part * static_cast<int64_t>(p.q_rows) * p.heads + at) * p.dim + i;
#pragma unroll
          for (int e = 0; there && any && e < 16; e += 4) *reinterpret_cast<uint4*>(to + e) = make_uint4(x[e], x[e + 1], x[e + 2], x[e + 3]);
        } else {
          uint32_t out[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            out[e] = l == 0.0f ? 0u : pack_result<T, E4M3>(__uint_as_float(x[2 * e]) * inv, __uint_as_float(x[2 * e + 1]) * inv);
          }
          uint8_t* const to = rows + (i >> 6) * kSpanBytes + row * 128;
          const int chunk = (i >> 3) & 7;
          *reinterpret_cast<uint4*>(to + ((chunk ^ (row & 7)) << 4)) = make_uint4(out[0], out[1], out[2], out[3]);
          *reinterpret_cast<uint4*>(to + (((chunk + 1) ^ (row & 7)) << 4)) = make_uint4(out[4], out[5], out[6], out[7]);
        }
      }
      if (!parted) {
        live = pair_sync(live);   // both halves of the 32 rows are there; each warp stores 16 of them
        const int64_t to = (static_cast<int64_t>(item.q0 + token) * p.o_token + h * p.o_head) * 2;
        constexpr int kChunks = SPANS * 8, kRowsAtOnce = 32 / kChunks;
        const int chunk = lane % kChunks;
#pragma unroll
        for (int i = 0; i < 16 / kRowsAtOnce; ++i) {
          const int from = half * 16 + i * kRowsAtOnce + lane / kChunks;   // lane that knows the row
          const int r = (warp & 3) * 32 + from;
          const int64_t dst = __shfl_sync(0xffffffffu, to, from);
          const bool wanted = __shfl_sync(0xffffffffu, there ? 1 : 0, from) != 0;
          const uint4 x = *reinterpret_cast<const uint4*>(rows + (chunk >> 3) * kSpanBytes + r * 128 + (((chunk & 7) ^ (r & 7)) << 4));
          if (wanted && chunk * 8 < p.dim) *reinterpret_cast<uint4*>(p.o + dst + chunk * 16) = x;
        }
      }
      if (there && half == 0) {
        if (parted) split.stats[part * static_cast<int64_t>(p.q_rows) * p.heads + at] = make_float2(any ? m * to_exp - kProbLift<M> : -INFINITY, l);
        else if (p.lse != nullptr) p.lse[at] = l == 0.0f ? -INFINITY : (m * to_exp - kProbLift<M>) * 0.6931471805599453f + logf(l);
      }
    }
  }
  tcgen05_fence_before_sync();
  __syncthreads();
  if (warp == kCopyWarp) {
    __syncwarp();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of split blocks in the order of the keys: one warp per (row, head).
template <typename T, bool E4M3>
__global__ void __launch_bounds__(256) attention_tiles_join_kernel(const ServingProblem p, const PagedCache cache, const TilesSplit split,
                                                                   int tile_tokens) {
  const int64_t at = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (at >= static_cast<int64_t>(p.q_rows) * p.heads) return;
  const int row = static_cast<int>(at / p.heads), h = static_cast<int>(at - static_cast<int64_t>(row) * p.heads);
  const int s = sequence_of_row(p.cu_q, p.n_seqs, row);
  if (s < 0) return;
  int q0, lq, k0, lk;
  serving_lengths<true>(p, cache, s, q0, lq, k0, lk);
  if (row - q0 >= p.max_q) return;   // not computed
  const int end = min(min(lq, p.max_q), ((row - q0) / (2 * tile_tokens) + 1) * 2 * tile_tokens);   // of the row's block
  const int tiles = (keys_seen(p.causal, end, lq, lk) + kTileKeys - 1) / kTileKeys;
  if (tiles <= split.tiles) return;   // written by its CTA
  const int parts = min(split.parts, (tiles + split.tiles - 1) / split.tiles);
  const int64_t stride = static_cast<int64_t>(p.q_rows) * p.heads;
  float m = -INFINITY;
  for (int i = lane; i < parts; i += 32) m = fmaxf(m, split.stats[i * stride + at].x);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  float4 sum = make_float4(0, 0, 0, 0);
  float l = 0.0f;
  const bool mine = lane * 4 < p.dim;
#pragma unroll 4
  for (int i = 0; i < parts; ++i) {
    const float2 ml = split.stats[i * stride + at];
    // Saw no key.  (A part whose scores are all NaN has no maximum either, but its sum is NaN and reaches the
    // result: ex2(-inf - m) is 0 or NaN.)
    if (ml.x == -INFINITY && ml.y == 0.0f) continue;
    const float f = ex2(ml.x - m);
    l += f * ml.y;
    if (mine) {
      const float4 x = *reinterpret_cast<const float4*>(split.o + (i * stride + at) * p.dim + lane * 4);
      sum.x += f * x.x;
      sum.y += f * x.y;
      sum.z += f * x.z;
      sum.w += f * x.w;
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (mine) {
    const uint2 out = l == 0.0f ? make_uint2(0, 0) : make_uint2(pack_result<T, E4M3>(sum.x * inv, sum.y * inv), pack_result<T, E4M3>(sum.z * inv, sum.w * inv));
    *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.o) + static_cast<int64_t>(row) * p.o_token + h * p.o_head + lane * 4) = out;
  }
  if (lane == 0 && p.lse != nullptr) p.lse[at] = l == 0.0f ? -INFINITY : m * 0.6931471805599453f + logf(l);
}

// Blocks of `tokens` query tokens there can be.
static int64_t most_blocks(const ServingProblem& p, int64_t tokens) {
  const int64_t by_rows = p.q_rows / tokens + p.n_seqs;
  const int64_t by_seq = static_cast<int64_t>(p.n_seqs) * ((p.max_q + tokens - 1) / tokens);
  return by_rows < by_seq ? by_rows : by_seq;
}

// How a call over a cache is split.  A block per SM or more is left whole (cutting 256 blocks of up to 94
// tiles cost 248 us against 216: partial results of every row for little better balance); with fewer the
// keys are cut into parts of at least eight tiles (1024 keys) so that there are about two CTAs per SM,
// whatever the lengths are: short sequences simply have fewer parts (16 sequences of 5 new tokens over up
// to 8000 keys: 127 -> 78 us, one such sequence 124 -> 33 us).
static void tiles_split_shape(const ServingProblem& p, int& parts, int& tiles) {
  const int64_t blocks = most_blocks(p, 2 * (kTileRows / p.group)) * p.kv_heads, all = (static_cast<int64_t>(p.max_kv) + kTileKeys - 1) / kTileKeys;
  parts = 1;
  tiles = 0;
  if (blocks == 0 || blocks >= kNumSMs || all <= 8) return;
  const int64_t each = (all * blocks + 2 * kNumSMs - 1) / (2 * kNumSMs);
  tiles = static_cast<int>(each < 8 ? 8 : each);
  parts = static_cast<int>((all + tiles - 1) / tiles);
}

size_t attention_tiles_workspace(const ServingProblem& p) {
  int parts, tiles;
  tiles_split_shape(p, parts, tiles);
  if (parts == 1) return 0;
  return kServingCounterBytes + static_cast<size_t>(parts) * p.q_rows * p.heads * (static_cast<size_t>(p.dim) * sizeof(float) + sizeof(float2));
}

int launch_attention_tiles(const ServingProblem& p, const PagedCache* cache, bool e4m3, void* workspace, cudaStream_t stream) {
  const int tile_tokens = kTileRows / p.group;
  TilesSplit split{1, 0, nullptr, nullptr};
  if (cache != nullptr) {
    tiles_split_shape(p, split.parts, split.tiles);
    split.o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kServingCounterBytes);
    split.stats = reinterpret_cast<float2*>(split.o + static_cast<size_t>(split.parts) * p.q_rows * p.heads * p.dim);
  }
  int64_t grid = most_blocks(p, 2 * tile_tokens) * p.kv_heads * split.parts;
  if (grid > 0x7fffffff) return set_error(FB200_INVALID_ARGUMENT, "attention: too many tiles");
  if (grid == 0) grid = 1;   // max_q is 0: one CTA looks whether any sequence has rows all the same
  const int spans = p.dim > 64 ? 2 : 1;
  CUtensorMap tq, tk, tv;
  const int64_t qd[4] = {p.dim, p.group, p.q_rows, p.kv_heads}, qs[3] = {p.q_head * 2, p.q_token * 2, p.q_head * p.group * 2};
  const int qb[4] = {64, p.group, tile_tokens, 1};
  if (int rc = make_tmap_4d(&tq, p.q, p.dtype, qd, qs, qb)) return rc;
  int box_keys = kTileKeys;
  tk = tv = tq;   // without keys nothing is copied through these maps
  if (cache != nullptr) {
    const int64_t page = int64_t(1) << cache->page_shift;
    if (page < box_keys) box_keys = static_cast<int>(page);
    const int64_t d[4] = {p.dim, page, p.kv_heads, cache->pages};
    const int64_t st[3] = {cache->token_stride * 2, cache->head_stride * 2, cache->page_stride * 2};
    const int64_t st8[3] = {cache->token_stride, cache->head_stride, cache->page_stride};
    const int b[4] = {64, box_keys, 1, 1}, b8[4] = {128, box_keys, 1, 1};   // a row of codes is one span
    if (cache->pages > 0) {
      if (int rc = make_tmap_4d(&tk, cache->k, e4m3 ? FB200_U8 : p.dtype, d, e4m3 ? st8 : st, e4m3 ? b8 : b)) return rc;
      if (int rc = make_tmap_4d(&tv, cache->v, e4m3 ? FB200_U8 : p.dtype, d, e4m3 ? st8 : st, e4m3 ? b8 : b)) return rc;
    }
  } else if (p.kv_rows > 0) {
    const int64_t d[4] = {p.dim, p.kv_rows, p.kv_heads, 1};
    const int64_t ks[3] = {p.k_token * 2, p.k_head * 2, p.k_token * 2}, vs[3] = {p.v_token * 2, p.v_head * 2, p.v_token * 2};
    const int b[4] = {64, box_keys, 1, 1};
    if (int rc = make_tmap_4d(&tk, p.k, p.dtype, d, ks, b)) return rc;
    if (int rc = make_tmap_4d(&tv, p.v, p.dtype, d, vs, b)) return rc;
  }
  int* status = nullptr;
  if (int rc = device_status_word(&status)) return rc;
  const PagedCache view = cache != nullptr ? *cache : PagedCache{};
  auto launch = [&](auto kernel) -> int {
    const size_t smem = ((tiles_small_bytes(spans, e4m3) + 1023) & ~1023u) + static_cast<size_t>(spans * kSpanBytes) * (2 + tiles_slots(spans, e4m3)) + (e4m3 ? kRawSlots * kSpanBytes : 0);
    static SmemOptIn opted;
    if (int rc = opted.once(kernel, smem)) return rc;
    kernel<<<static_cast<unsigned>(grid), tiles_threads(e4m3), smem, stream>>>(tq, tk, tv, p, view, split, tile_tokens,
                                                                             static_cast<uint32_t>((uint64_t(1) << 32) / (2 * tile_tokens)), box_keys, status);
    return FB200_OK;
  };
  auto pick = [&](auto type) -> int {
    using T = decltype(type);
    if (cache == nullptr) return spans == 2 ? launch(attention_tiles_kernel<T, 2, false, false>) : launch(attention_tiles_kernel<T, 1, false, false>);
    if (e4m3) return spans == 2 ? launch(attention_tiles_kernel<T, 2, true, true>) : launch(attention_tiles_kernel<T, 1, true, true>);
    return spans == 2 ? launch(attention_tiles_kernel<T, 2, true, false>) : launch(attention_tiles_kernel<T, 1, true, false>);
  };
  if (int rc = p.dtype == FB200_BF16 ? pick(__nv_bfloat16()) : pick(__half())) return rc;
  if (int rc = after_launch("attention_tiles_kernel")) return rc;
  if (split.parts == 1) return FB200_OK;
  const int64_t joins = (static_cast<int64_t>(p.q_rows) * p.heads + 7) / 8;
  auto join = [&](auto kernel) { kernel<<<static_cast<unsigned>(joins), 256, 0, stream>>>(p, view, split, tile_tokens); };
  if (p.dtype == FB200_BF16) e4m3 ? join(attention_tiles_join_kernel<__nv_bfloat16, true>) : join(attention_tiles_join_kernel<__nv_bfloat16, false>);
  else e4m3 ? join(attention_tiles_join_kernel<__half, true>) : join(attention_tiles_join_kernel<__half, false>);
  return after_launch("attention_tiles_join_kernel");
}

}  // namespace fb200
