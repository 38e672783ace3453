// Attention of prompts in the expanded form: keys of 128 values a head and 64
// for all heads, values of 128.
//
//   out[i,h] = softmax_j((q[i,h,:128] . k[j,h] + q[i,h,128:] . k_rope[j]) scale) . v[j,h]
//
// Two CTAs (a cluster, on neighbouring SMs) take a block of one head's queries. A
// product spans both: each has 128 of its 256 queries, and brings half of the keys
// (64 of 128) and half of the values (64 of the 128 of each token), so that an SM reads
// 40 KiB for a tile of 128 keys where it would read 80 by itself: then the copies'
// latency was what bounded the products, at 2250 cycles for a tile whose products
// take 1280.
//   S_t = Q_t K^T   256 x 128 x 192, both from shared memory
//   O_t += P_t V    256 x 128 x 128, P over S in tensor memory, rounded to the
//                   inputs' type: the products take nothing wider beside V, and a
//                   second term would double them. Its sum takes the unrounded
//                   weights: over values of either sign the rounded ones would
//                   cancel little of it. Errors (rms, relative) are 0.0021 in bf16,
//                   of which the output's own rounding is 0.0016; f16 0.00025, 0.0002.
// t counts two such pairs of S and O, which take all 512 columns of tensor memory: the
// softmax of one runs while the products of the other do, in the order
// O_0(j) S_0(j+1) O_1(j) S_1(j+1). A block has 512 queries, 256 for each t, that share
// the keys; where that would leave SMs without work it has 256, and t = 0 and 1 take its
// even and odd tiles of keys, joined at the end.
//
// Softmax: a thread has a row, its scores in registers; references are lazy (a row
// passes its own by 2^15, all that f16 weights hold, before O is rescaled; theirs sits
// 2^7 below the row's largest score, so that they are whole down to 2^-21 of the
// largest), sums in fp32. The first 64 weights are taken against the reference as it stands while the
// tile's largest score is looked for, and handed to the products while the others are
// taken.
//
// A weight of 0 times an infinity or NaN would not be 0 in the product: values past
// a sequence's end are cleared in shared memory, and on tiles that some query sees
// in part, values that are not finite are cleared and added to the rows that see
// them at the end (two warps look for them while the scores are under way).
//
// Between the CTAs: a thread of the odd one tells the even one's products what its
// copies have brought (released and acquired at the cluster's scope), and stays until
// the products' last arrivals have come. Where only tensor memory is handed over,
// ordered by the tcgen05 fences, arrivals are relaxed.
//
// Measured: 16384 tokens, 16 heads, causal: 1.01 ms, 1370 TFLOP/s, a turn of t at 1760
// cycles with 1280 of products: the softmax (125 for the scores, 840 to the first
// weights handed over, 650 to the rest), the products of a turn after it and their
// latency make a chain of 3500 for two turns. A block costs another 10000 cycles to
// start and to end, a tile that some query sees in part 1500. One that a single SM takes
// by itself (80 KiB a tile, ring of 8 x 16 KiB) runs at 900 TFLOP/s.
//
// Every wait is bounded; a CTA that gives up records it in the device error word,
// waits for its own copies and products, frees its tensor memory and returns.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <atomic>

#include "../../include/qsa_b200.h"
#include "qsa_latent.cuh"
#include "qsa_latent_tc.cuh"

namespace qsa {
namespace {

constexpr int kLpTile = 128;                 // queries of a CTA in a product, and keys
constexpr int kLpChunk = kLpTile * 128;      // bytes of 128 tokens of 64 values
constexpr int kLpThreads = 384;
constexpr int kLpLoadWarp = 8, kLpMmaWarp = 9, kLpFixWarp = 10;
constexpr int kLpHeads = 8;                   // heads whose blocks of an entry follow one another
constexpr float kLpMost = 15.f;              // log2 of the largest weight
constexpr float kLowest = -3.402823466e38f;
constexpr uint64_t kLpDrainNs = 20000000ull;  // for copies, whose announcement a failure can keep from coming
constexpr uint64_t kLpDoneNs = 1000000000ull;  // for the products' last arrivals, which always come

// Queries of a block, and shared memory: [Q tiles][3 chunks], then the stages. Stage n
// brings what a turn needs: keys n (3 half chunks) and values n - kAhead (one chunk).
template <bool kSplit>
struct Lp {
  static constexpr int kBlock = kSplit ? 2 * kLpTile : 4 * kLpTile;
  static constexpr int kQTiles = kSplit ? 1 : 2, kStages = kSplit ? 4 : 3, kAhead = kSplit ? 2 : 1;
  static constexpr int kStage = 5 * (kLpChunk / 2), kV = 3 * (kLpChunk / 2);
  static constexpr int kRing = kQTiles * 3 * kLpChunk;
  static constexpr int kStats = kRing + kStages * kStage;  // [t][128] references and sums
  static constexpr int kBars = kStats + 2 * kLpTile * 8;
  static constexpr int kMisc = kBars + 8 * (4 * kStages + 1 + 2 + 4 + 2 + 1);
  static constexpr int kSmem = kMisc + 64 + 1024;
  static_assert(kSmem + 256 <= 232448 && kMisc % 8 == 0 && kV % 1024 == 0 && kStage % 1024 == 0, "shared memory");
};

constexpr uint32_t kLpTmemS = 0, kLpTmemO = 256;  // columns, 128 for each t

struct LpMaps {
  CUtensorMap q, k, k_rope, v;
};

// A block's entry and place: queries q0 .. of `n` (the first at token q_at), m keys from k_at.
struct LpBlock {
  int q_at, n, k_at, m, first, head;
};

__device__ __forceinline__ void mbar_expect(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];\n" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y)
      : "memory");
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <typename T, bool kSplit>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kLpThreads, 1)
    qsa_latent_prefill_kernel(const __grid_constant__ LatentPrefillParams p, const __grid_constant__ LpMaps maps) {
  using L = Lp<kSplit>;
  constexpr int kStages = L::kStages, kAhead = L::kAhead;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr float kSits = kBf16 ? 0.f : 7.f;  // log2 of the largest weight where the reference has just moved
  constexpr uint32_t kExp = kBf16 ? 0x7f80u : 0x7c00u;  // exponent bits of an infinity or NaN
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_s = smem_u32(smem_raw);
  const uint32_t base_s = (raw_s + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base_s - raw_s);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_rank();  // the products are issued by rank 0

  // In rank 0 what both CTAs have to be done with counts an arrival of each; the
  // products' arrivals go to both.
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBars);  // [stages] copies (of both) -> products
  uint64_t* empty = full + kStages;                               // [stages] products -> copies
  uint64_t* v_here = empty + kStages;                             // [stages] this CTA's values -> fixers, on tiles that they go through
  uint64_t* fixed = v_here + kStages;                             // [stages] fixers of both -> products, results
  uint64_t* q1_full = fixed + kStages;                            // copies of Q_1 (of both) -> products; Q_0 comes with stage 0
  uint64_t* s_full = q1_full + 1;                                 // [2] products -> softmax
  uint64_t* p_full = s_full + 2;                                  // [2][2 halves] softmax of both -> products
  uint64_t* o_full = p_full + 4;                                  // [2] products -> softmax
  uint64_t* drain = o_full + 2;
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(smem + L::kMisc);
  const uint32_t tries = tries_of(p.wait_limit_ns);
  volatile int* stages_loaded = reinterpret_cast<volatile int*>(smem + L::kMisc + 8);  // as far as the loader has come
  volatile int* odd_values = reinterpret_cast<volatile int*>(smem + L::kMisc + 12);    // values that were cleared
  LpBlock* found = reinterpret_cast<LpBlock*>(smem + L::kMisc + 16);

  const int at_block = (int)(blockIdx.x >> 1);
  if (tid == 0) {
    const int both = rank == 0 ? 2 : 1;
    for (int i = 0; i < kStages; ++i) {
      mbar_init(full + i, both);
      mbar_init(empty + i, 1);
      mbar_init(v_here + i, 1);
      mbar_init(fixed + i, 4);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(s_full + t, 1);
      mbar_init(p_full + 2 * t, 8);
      mbar_init(p_full + 2 * t + 1, 8);
      mbar_init(o_full + t, 1);
    }
    mbar_init(q1_full, both);
    mbar_init(drain, 1);
    *stages_loaded = 0;
    *odd_values = 0;
    *found = LpBlock{0, 0, 0, 0, -1, 0};  // a block past the last one
    fence_mbar_init();
  }
  // The entry that the block belongs to: those with the most keys first where there are
  // no more than a warp has lanes, in their order otherwise. An entry's blocks run over
  // some heads at a time, so that their keys and values are still in the L2 when the next
  // block reads them, and for those from its end, the longest first.
  auto bounds = [&](int e, LpBlock& b) -> int {  // of an entry, and its blocks
    b.q_at = b.n = b.k_at = b.m = 0;
    if (e < p.entries) {
      b.q_at = max(__ldg(p.cu_q + e), 0);
      b.n = max(min(__ldg(p.cu_q + e + 1), p.q_tokens) - b.q_at, 0);
      b.k_at = min(max(__ldg(p.cu_k + e), 0), p.k_tokens);
      b.m = max(min(__ldg(p.cu_k + e + 1), p.k_tokens) - b.k_at, 0);
    }
    return (b.n + L::kBlock - 1) / L::kBlock;
  };
  auto place = [&](int64_t before, int blocks, LpBlock& b) {  // the block of an entry that follows so many
    const int local = (int)(at_block - before * p.heads);
    const int first_head = local / (blocks * kLpHeads) * kLpHeads;
    const int of_them = local - first_head * blocks, some = min(p.heads - first_head, kLpHeads);
    b.first = (blocks - 1 - of_them / some) * L::kBlock;
    b.head = first_head + of_them % some;
  };
  LpBlock b;
  __syncwarp();
  if (p.entries <= 32) {
    int blocks = bounds(lane, b);
    int64_t before = 0;
#pragma unroll 1
    for (int e = 0; e < p.entries; ++e) {
      const int keys = __shfl_sync(0xffffffffu, b.m, e), others = __shfl_sync(0xffffffffu, blocks, e);
      before += keys > b.m || (keys == b.m && e < lane) ? others : 0;
    }
    const uint32_t mine = __ballot_sync(0xffffffffu, at_block >= before * p.heads && at_block < (before + blocks) * p.heads);
    const int from = mine ? __ffs(mine) - 1 : 0;
    b.q_at = __shfl_sync(0xffffffffu, b.q_at, from);
    b.n = __shfl_sync(0xffffffffu, b.n, from);
    b.k_at = __shfl_sync(0xffffffffu, b.k_at, from);
    b.m = __shfl_sync(0xffffffffu, b.m, from);
    blocks = __shfl_sync(0xffffffffu, blocks, from);
    before = __shfl_sync(0xffffffffu, before, from);
    if (mine) place(before, blocks, b);
    else b.first = -1;
    __syncthreads();  // the barriers are ready
  } else {
    __shared__ int warp_sum[kLpThreads / 32];
    int before = 0;  // blocks of the entries looked through
    __syncthreads();
    for (int e0 = 0; e0 < p.entries; e0 += kLpThreads) {
      const int blocks = bounds(e0 + tid, b);
      int upto = blocks;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      if (lane == 31) warp_sum[warp] = upto;
      __syncthreads();
      int total = 0;
#pragma unroll
      for (int w = 0; w < kLpThreads / 32; ++w) {
        if (w < warp) upto += warp_sum[w];
        total += warp_sum[w];
      }
      upto += before;
      const int64_t others = upto - blocks;
      if (at_block >= others * p.heads && at_block < (int64_t)upto * p.heads) {
        place(others, blocks, b);
        *found = b;
      }
      before += total;
      __syncthreads();
      if (at_block < (int64_t)before * p.heads) break;
    }
    b = *found;
  }
  if (b.first < 0) return;  // a block past the last one, for both CTAs
  const int head = b.head;
  bool failed = false;
  // tiles of keys that the last query of t sees
  auto key_tiles = [&](int t) -> int {
    const int first = b.first + (kSplit ? 0 : t * 2 * kLpTile), rows = min(b.n - first, 2 * kLpTile);
    if (rows <= 0) return 0;
    const int seen = p.causal ? min((int64_t)b.m, (int64_t)first + rows + b.m - b.n) : b.m;
    return seen > 0 ? (seen + kLpTile - 1) / kLpTile : 0;
  };
  const int last0 = key_tiles(0), last1 = key_tiles(1), nk = max(last0, last1);
  const int nk0 = kSplit ? (nk + 1) / 2 : last0, nk1 = kSplit ? nk / 2 : last1;  // tiles that t takes
  auto key_of = [](int t, int i) -> int { return kSplit ? 2 * i + t : i; };      // the i-th of them
  // tiles from here on hold a key that some query of the block does not see, or
  // that lies past the sequence
  const int whole = min(p.causal ? max(b.first + (b.m - b.n) + 1, 0) : b.m, b.m) / kLpTile;
  // stages, the first whose values the fixers go through, and the phase of their n-th use
  const int stages = nk > 0 ? nk + kAhead : 0, fix_from = whole + kAhead;
  auto parity_of = [](int n) -> uint32_t { return (uint32_t)((n / kStages) & 1); };

  // queries of t, and stage n's keys and values
  auto load_queries = [&](int t, uint64_t* bar) {
    for (int c = 0; c < 3; ++c)
      tma_3d(base_s + (3 * t + c) * kLpChunk, &maps.q, bar, 64 * c, head, b.q_at + b.first + (2 * t + (int)rank) * kLpTile);
  };
  auto load = [&](int n) {
    const int st = n % kStages, j = n - kAhead;  // the values' tile
    const uint32_t dst = base_s + L::kRing + st * L::kStage;
    // values for the fixers land on a barrier of their own, each phase of which
    // they wait for; the products wait for the fixers then
    const bool fix = n >= fix_from;
    mbar_expect(full + st, (n == 0 && nk0 > 0 ? 3 * kLpChunk : 0) + (n < nk ? 3 * (kLpChunk / 2) : 0) + (j >= 0 && !fix ? kLpChunk : 0));
    if (n == 0 && nk0 > 0) load_queries(0, full);  // else the results' zeros are written there
    if (n < nk) {
      const int at = b.k_at + n * kLpTile + (int)rank * (kLpTile / 2);
      for (int c = 0; c < 2; ++c) tma_3d(dst + c * (kLpChunk / 2), &maps.k, full + st, 64 * c, head, at);
      tma_2d(dst + 2 * (kLpChunk / 2), &maps.k_rope, full + st, 0, at);
    }
    if (j >= 0) {
      if (fix) mbar_expect(v_here + st, kLpChunk);
      tma_3d(dst + L::kV, &maps.v, fix ? v_here + st : full + st, 64 * (int)rank, head, b.k_at + j * kLpTile);
    }
  };
  const bool queries1 = !kSplit && nk1 > 0;
  int loaded = 0;
  if (warp == kLpLoadWarp && lane == 0) {  // the first copies are under way while the CTAs find one another
#pragma unroll 1
    for (; loaded < min(stages, kStages); ++loaded) {
      load(loaded);
      if (loaded == 0 && queries1) mbar_expect(q1_full, 3 * kLpChunk), load_queries(1, q1_full);
    }
  }
  if (warp == kLpMmaWarp) {
    pair_tmem_alloc(tmem_at, 512);
    tc_fence_before();
  }
  __syncwarp();
  cluster_sync();
  tc_fence_after();
  constexpr uint32_t tmem = 0;  // all of it is these blocks'

  if (warp >= kLpLoadWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;\n");
    if (warp == kLpLoadWarp && lane == 0 && nk > 0) {
      // ================================ TMA =================================
#pragma unroll 1
      for (; loaded < stages; ++loaded) {
        failed = !wait_tries(empty + loaded % kStages, parity_of(loaded - kStages), tries);
        if (failed) break;
        load(loaded);
        *stages_loaded = loaded;
      }
      const int n = loaded;
      // all copies have landed before the block leaves (the usual end: the products took them)
      if (queries1 && !mbar_wait_bounded(q1_full, 0u, kLpDrainNs)) failed = true;
      for (int m = max(n - kStages, 0); m < n; ++m) {
        if (!mbar_wait_bounded(full + m % kStages, parity_of(m), kLpDrainNs)) failed = true;
        if (m >= fix_from && !mbar_wait_bounded(v_here + m % kStages, parity_of(m - fix_from), kLpDrainNs)) failed = true;
      }
    } else if (warp == kLpMmaWarp && rank == 0 && nk > 0) {
      // ============================== products ==============================
      constexpr uint32_t kIdescS = idesc_f16(2 * kLpTile, kLpTile, kBf16, false), kIdescO = idesc_f16(2 * kLpTile, 128, kBf16, true);
      auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        if (!__all_sync(0xffffffffu, wait_tries(bar, parity, tries))) return false;
        tc_fence_after();
        return true;
      };
      // what the other CTA's threads tell of its shared memory
      auto wait_pair = [&](uint64_t* bar, uint32_t parity) -> bool {
        if (!__all_sync(0xffffffffu, cluster_wait_tries(bar, parity, tries))) return false;
        tc_fence_after();
        return true;
      };
      auto scores = [&](int t, int st) {  // S_t = Q_t K^T
        const uint32_t a0 = desc_low(base_s) + (kSplit ? 0 : t) * 3 * (kLpChunk / 16);
        const uint32_t b0 = desc_low(base_s + L::kRing) + st * (L::kStage / 16);
#pragma unroll
        for (int c = 0; c < 3; ++c)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            pair_mma_f16_ss(tmem + kLpTmemS + t * 128, a0 + c * (kLpChunk / 16) + kk * 2, b0 + c * (kLpChunk / 32) + kk * 2, kIdescS, c + kk > 0 ? 1u : 0u);
        pair_commit(s_full + t);
      };
      auto weigh = [&](int t, int i, int st) -> bool {  // O_t += P_t V, the first 64 tokens' weights first
        const uint32_t d = tmem + kLpTmemO + t * 128, a = tmem + kLpTmemS + t * 128;
        const uint32_t b0 = desc_low(base_s + L::kRing + L::kV) + st * (L::kStage / 16);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (!wait(p_full + 2 * t + h, (uint32_t)(i & 1))) return false;
#pragma unroll
          for (int kk = 4 * h; kk < 4 * h + 4; ++kk) pair_mma_f16_ts(d, a + kk * 8, b0 + kk * 128, kIdescO, kk > 0 ? 1u : i > 0);
        }
        return true;
      };
      // turn i of t: the weighted values of its tile i, the scores of the next. Scores
      // that have arrived tell that the values before are in.
#pragma unroll 1
      for (int i = -1; i < max(nk0, nk1) && !failed; ++i)
#pragma unroll 1
        for (int t = 0; t < 2 && !failed; ++t) {
          const int tiles = t == 0 ? nk0 : nk1, n = key_of(t, i) + kAhead, st = n % kStages;
          if (i < tiles && tiles > 0) {
            failed = !wait_pair(full + st, parity_of(n)) || (!kSplit && t == 1 && i < 0 && !wait_pair(q1_full, 0u)) ||
                     (n >= fix_from && !wait_pair(fixed + st, parity_of(n - fix_from))) ||
                     (i >= 0 && !weigh(t, i, st));
            if (failed) break;
            if (i + 1 < tiles) scores(t, st);
            else pair_commit(o_full + t);
          }
          if (kSplit ? n < stages : t == 1) pair_commit(empty + st);  // the last to use it
        }
      pair_commit(drain);
      if (!mbar_wait_bounded(drain, 0u, kLpDoneNs)) failed = true;
    } else if (warp == kLpMmaWarp && nk > 0) {
      // ================== this CTA's copies, told to the products =================
      auto tell = [&](uint64_t* bar, uint32_t parity) {
        if (!failed) failed = !wait_tries(bar, parity, tries);
        if (!failed) cluster_arrive(smem_of(bar, 0));
      };
      if (lane == 0) {
#pragma unroll 1
        for (int n = 0; n < stages && !failed; ++n) {
          tell(full + n % kStages, parity_of(n));
          if (n == 0 && queries1) tell(q1_full, 0u);
        }
        // the products' arrivals here have come before the block leaves its memory
        if (!mbar_wait_bounded(drain, 0u, kLpDoneNs)) failed = true;
      }
    } else if (warp >= kLpFixWarp) {
      // ====================== values that must not count ====================
      const int at = tid - 32 * kLpFixWarp;  // of 64 threads
      const uint32_t other = rank ^ 1;
#pragma unroll 1
      for (int j = whole; j < nk; ++j) {
        bool any = false;
        const int st = (j + kAhead) % kStages;
        // the first comes when all whole tiles have gone through: the limit is for a time
        // in which the loader has not brought another stage
        for (int seen = __shfl_sync(0xffffffffu, *stages_loaded, 0);;) {
          failed = !__all_sync(0xffffffffu, wait_tries(v_here + st, parity_of(j - whole), tries));
          const int now = __shfl_sync(0xffffffffu, *stages_loaded, 0);
          if (!failed || now == seen) break;
          seen = now;
        }
        if (failed) break;
        uint8_t* v = smem + L::kRing + st * L::kStage + L::kV;
#pragma unroll 4
        for (int i = at; i < kLpChunk / 16; i += 64) {  // 16 bytes of row i / 8; all of a row are treated alike
          uint4* x = reinterpret_cast<uint4*>(v + i * 16);
          uint4 w = *x;
          const bool past = j * kLpTile + i / 8 >= b.m;
          uint32_t words[4] = {w.x, w.y, w.z, w.w};
          bool odd = false;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if ((words[k] & kExp) == kExp) words[k] &= 0xffff0000u, odd = true;
            if ((words[k] & (kExp << 16)) == (kExp << 16)) words[k] &= 0xffffu, odd = true;
          }
          if (past) *x = make_uint4(0u, 0u, 0u, 0u);
          else if (odd) *x = make_uint4(words[0], words[1], words[2], words[3]), any = true;
        }
        if (any) {
          *odd_values = 1;
          asm volatile("st.shared::cluster.u32 [%0], %1;\n" ::"r"(smem_of(const_cast<int*>(odd_values), other)), "r"(1) : "memory");
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane < 2) cluster_arrive(smem_of(fixed + st, lane));
      }
    }
    __syncwarp();
  } else {
    // ========================== softmax, results ===========================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;\n");
    const int t = warp >> 2;
    const int tiles = t == 0 ? nk0 : nk1;
    const int q4 = warp & 3, row = q4 * 32 + lane;
    const uint32_t lane_base = (uint32_t)(q4 * 32) << 16;
    const uint32_t s_at = tmem + lane_base + kLpTmemS + t * 128, o_at = tmem + lane_base + kLpTmemO + t * 128;
    const int i = b.first + (kSplit ? 0 : t * 2 * kLpTile) + (int)rank * kLpTile + row;  // the thread's query
    const int64_t seen = p.causal ? min((int64_t)b.m, (int64_t)i + b.m - b.n + 1) : b.m;  // keys that it sees
    const bool valid = i < b.n;
    const uint32_t told = smem_of(p_full + 2 * t, 0);
    float r = kLowest, l = 0.f;
#pragma unroll 1
    for (int j = 0; j < tiles; ++j) {
      failed = __any_sync(0xffffffffu, !wait_tries(s_full + t, (uint32_t)(j & 1), tries));
      if (failed) break;
      tc_fence_after();
      float s[4][32];
      tmem_ld_2x32_wait(s_at, s_at + 32, s[0], s[1]);
      tmem_ld_2x32_wait(s_at + 64, s_at + 96, s[2], s[3]);
      const int left = (int)max((int64_t)0, min((int64_t)kLpTile, seen - (int64_t)key_of(t, j) * kLpTile));  // visible columns of the tile
      if (p.negative) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int k = 0; k < 32; ++k) s[c][k] = -s[c][k];
      }
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (__any_sync(0xffffffffu, left < 32 * c + 32)) {
#pragma unroll
          for (int k = 0; k < 32; ++k) s[c][k] = 32 * c + k < left ? s[c][k] : -INFINITY;
        }
      // Weights of the first half against the row's reference as it is, while the tile's
      // largest score is found; where that passes it, the reference moves and they are
      // taken again.
      uint64_t sum[2];
      uint32_t w[32];
      const uint64_t scale2 = pair2(p.score_scale_log2, p.score_scale_log2);
      auto weights = [&](int c) {  // of 64 keys
        const uint64_t back2 = pair2(-r, -r);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            float a, d;
            unpair2(fma2(pair2(s[c + h][k], s[c + h][k + 1]), scale2, back2), a, d);
            a = ex2(a), d = ex2(d);
            sum[h] = add2(sum[h], pair2(a, d));
            w[16 * h + k / 2] = pack2<T>(a, d);
          }
      };
      auto hand_over = [&](int c) {
        tmem_st(s_at + 16 * c, w);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) cluster_arrive_relaxed(told + 4 * c);
      };
#pragma unroll 1
      for (;;) {
        float tops[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) tops[c] = max3_nan(s[c][0], s[c][1], s[c][2]);
#pragma unroll
        for (int k = 3; k < 31; k += 2)
#pragma unroll
          for (int c = 0; c < 4; ++c) tops[c] = max3_nan(tops[c], s[c][k], s[c][k + 1]);
#pragma unroll
        for (int c = 0; c < 4; ++c) tops[c] = fmaxf(tops[c], s[c][31]);
        const float top = fmaxf(max3(tops[0], tops[1], tops[2]), tops[3]) * p.score_scale_log2;
        sum[0] = sum[1] = 0;
        weights(0);
        const bool moves = top > r + kLpMost;
        if (!__any_sync(0xffffffffu, moves)) break;
        const float next = moves ? top - kSits : r;
        const float f = ex2(r - next);
        r = next;
        l *= f;
        if (j > 0) {
#pragma unroll 1
          for (int c = 0; c < 8; ++c) {
            float x[16];
            uint32_t y[16];
            tmem_ld_wait<16>(o_at + 16 * c, x);
#pragma unroll
            for (int k = 0; k < 16; ++k) y[k] = __float_as_uint(x[k] * f);
            tmem_st(o_at + 16 * c, y);
          }
        }
      }
      hand_over(0);
      weights(2);
      hand_over(2);
      float a, d;
      unpair2(add2(sum[0], sum[1]), a, d);
      l += a + d;
    }
    if (tiles > 0 && !failed) failed = !wait_tries(o_full + t, 0u, tries);
    for (int j = max(nk - kStages, whole); j < nk; ++j)
      if (!failed) failed = !cluster_wait_tries(fixed + (j + kAhead) % kStages, parity_of(j - whole), tries);
    failed = __any_sync(0xffffffffu, failed);
    tc_fence_after();
    float f0 = 1.f, f1 = 0.f;  // what the parts count for
    if (kSplit) {
      float2* stats = reinterpret_cast<float2*>(smem + L::kStats);
      stats[t * kLpTile + row] = make_float2(r, l);
      tc_fence_before();
      failed = bar_vote(1, 256, failed);
      tc_fence_after();
      const float2 x = stats[row], y = stats[kLpTile + row];
      const float top = fmaxf(x.x, y.x);
      f0 = ex2(x.x - top), f1 = ex2(y.x - top);
      l = x.y * f0 + y.y * f1;
    }
    if (!failed) {
      const float inv = l == 0.f ? 0.f : 1.0f / l;  // 0 for a row without scores
      const bool odd = *odd_values != 0;
      const int c0 = kSplit ? 2 * t : 0, c1 = kSplit ? 2 * t + 2 : 4;
      // rows of a warp's results go through shared memory (the queries', which are done
      // with), 16 bytes at a time in places that spread over the banks, and leave whole:
      // a thread that wrote its own row would take a transaction for every 16 bytes
      constexpr int kUnits = kSplit ? 8 : 16;  // of a row
      uint8_t* stage = smem + (kSplit ? warp * 32 * 16 * kUnits : t * 3 * kLpChunk + q4 * 32 * 16 * kUnits);
#pragma unroll 1
      for (int c = c0; c < c1; ++c) {
        __syncwarp();  // the loads below are the whole warp's
        float x[32];
        if (kSplit ? nk0 > 0 : tiles > 0) {
          tmem_ld_wait<32>((kSplit ? o_at - t * 128 : o_at) + 32 * c, x);
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) x[k] = 0.f;
        }
        if (kSplit && nk1 > 0) {
          float y[32];
          tmem_ld_wait<32>(o_at + (1 - t) * 128 + 32 * c, y);
#pragma unroll
          for (int k = 0; k < 32; ++k) x[k] = x[k] * f0 + y[k] * f1;
        }
#pragma unroll
        for (int k = 0; k < 32; ++k) x[k] *= inv;
        if (odd && valid) {  // what was cleared counts where it is seen
          for (int64_t j = (int64_t)whole * kLpTile; j < seen; ++j) {
            const T* v = static_cast<const T*>(p.v) + (b.k_at + j) * p.v_stride + head * p.v_head_stride + 32 * c;
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              const float y = latent_to_float(v[k]);
              if (!(fabsf(y) <= 3.402823466e38f)) x[k] += y;
            }
          }
        }
#pragma unroll
        for (int k = 0; k < 32; k += 8) {
          const int u = 4 * (c - c0) + k / 8;
          *reinterpret_cast<uint4*>(stage + (lane * kUnits + (u ^ (lane & 7))) * 16) =
              make_uint4(pack2<T>(x[k], x[k + 1]), pack2<T>(x[k + 2], x[k + 3]), pack2<T>(x[k + 4], x[k + 5]), pack2<T>(x[k + 6], x[k + 7]));
        }
      }
      __syncwarp();
      T* out = static_cast<T*>(p.out) + ((int64_t)(b.q_at + i - lane) * p.heads + head) * 128 + 32 * c0;
#pragma unroll 4
      for (int k = lane; k < 32 * kUnits; k += 32) {
        const int of = k / kUnits, u = k % kUnits;  // row, unit
        if (i - lane + of < b.n)
          *reinterpret_cast<uint4*>(out + (int64_t)of * p.heads * 128 + 8 * u) =
              *reinterpret_cast<const uint4*>(stage + (of * kUnits + (u ^ (of & 7))) * 16);
      }
    }
  }

  if (failed) {
    if (p.err) atomicOr(p.err, 1);
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync();  // nothing of the other CTA's is read or told any more
  if (warp == kLpMmaWarp) {
    tc_fence_after();
    pair_tmem_free(tmem, 512);
  }
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static std::atomic<void*> fn{nullptr};
  void* f = fn.load(std::memory_order_acquire);
  if (!f) {
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return nullptr;
    fn.store(f, std::memory_order_release);
  }
  return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
}

// [tokens, heads, values] (heads = 0: [tokens, values]) as boxes of 64 values of
// some tokens of a head, 128-byte swizzled; tokens past the end read zeros.
bool encode(CUtensorMap* map, bool bf16, const void* base, int values, int heads, int tokens, int64_t head_stride,
            int64_t stride, int rows) {
  auto fn = encode_fn();
  if (!fn) return false;
  const bool flat = heads == 0;
  const cuuint64_t dims[3] = {(cuuint64_t)values, (cuuint64_t)(flat ? tokens : heads), (cuuint64_t)tokens};
  const cuuint64_t strides[2] = {(cuuint64_t)(flat ? stride : head_stride) * 2, (cuuint64_t)stride * 2};
  const cuuint32_t box[3] = {64u, flat ? (cuuint32_t)rows : 1u, (cuuint32_t)rows};
  const cuuint32_t step[3] = {1u, 1u, 1u};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, flat ? 2 : 3, const_cast<void*>(base),
            dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, bool kSplit>
cudaError_t launch(const LatentPrefillParams& p, int64_t blocks, cudaStream_t stream) {
  // the shared memory beyond the default limit, once per device
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(ready.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(qsa_latent_prefill_kernel<T, kSplit>, cudaFuncAttributeMaxDynamicSharedMemorySize, Lp<kSplit>::kSmem);
    if (e != cudaSuccess) return e;
    ready.fetch_or(bit, std::memory_order_acq_rel);
  }
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  // without keys no block loads any, and the maps stand for the queries
  const bool none = p.k_tokens == 0;
  const int k_tokens = none ? 1 : p.k_tokens;
  LpMaps m;
  if (!encode(&m.q, kBf16, p.q, 192, p.heads, p.q_tokens, p.q_head_stride, p.q_stride, kLpTile) ||
      !encode(&m.k, kBf16, none ? p.q : p.k, 128, p.heads, k_tokens, none ? p.q_head_stride : p.k_head_stride, none ? p.q_stride : p.k_stride, kLpTile / 2) ||
      !encode(&m.k_rope, kBf16, none ? p.q : p.k_rope, 64, 0, k_tokens, 0, none ? p.q_stride : p.k_rope_stride, kLpTile / 2) ||
      !encode(&m.v, kBf16, none ? p.q : p.v, 128, p.heads, k_tokens, none ? p.q_head_stride : p.v_head_stride, none ? p.q_stride : p.v_stride, kLpTile))
    return cudaErrorInvalidValue;
  const int64_t grid = blocks * p.heads * 2;
  if (grid > 0x7fffffffll) return cudaErrorInvalidValue;
  qsa_latent_prefill_kernel<T, kSplit><<<(unsigned)grid, kLpThreads, Lp<kSplit>::kSmem, stream>>>(p, m);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_latent_prefill(const LatentPrefillParams& p, cudaStream_t stream) {
  // An entry's blocks are its length over theirs, rounded up. Large blocks bring keys
  // and values for twice the queries, but a pair of SMs each has to have some: 8192
  // tokens take 136 us in large and 82 in small blocks of 4 heads (64 large ones), 138
  // and 130 of 6, 140 and 159 of 8, 276 and 305 of 16; five chunks of up to 700 over up
  // to 2700 keys, 16 heads, 76 and 61.
  const int64_t most = p.entries < p.q_tokens ? p.entries : p.q_tokens;
  const int64_t large = p.q_tokens / Lp<false>::kBlock + most, small = p.q_tokens / Lp<true>::kBlock + most;
  const bool bf16 = p.dtype == QSA_B200_DTYPE_BF16;
  if (large * p.heads * 8 <= latent_sm_count() * 7)
    return bf16 ? launch<__nv_bfloat16, true>(p, small, stream) : launch<__half, true>(p, small, stream);
  return bf16 ? launch<__nv_bfloat16, false>(p, large, stream) : launch<__half, false>(p, large, stream);
}

}  // namespace qsa
