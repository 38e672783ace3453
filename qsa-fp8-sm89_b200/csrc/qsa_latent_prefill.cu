// Attention of prompts in the expanded form: keys of 128 values a head and 64
// for all heads, values of 128.
//
//   out[i,h] = softmax_j((q[i,h,:128] . k[j,h] + q[i,h,128:] . k_rope[j]) scale) . v[j,h]
//
// A CTA takes 256 queries of one head in two tiles of 128 that share every key
// and value, so that the softmax of one tile runs while the products of the other
// do:
//   S_t = Q_t K^T   128 x 128 x 192, both from shared memory
//   O_t += P_t V    128 x 128 x 128, P (rounded to the inputs' type, the usual
//                   choice: its sum is taken in fp32) over S in tensor memory
// Tensor memory holds two S and two O, all of its 512 columns. Keys and values come
// by TMA, 16 KiB (128 tokens of 64 values) at a time, into a ring of 8 slots in the
// order K(0) V(0) K(1) ...; the products run PV_0(j) S_0(j+1) PV_1(j) S_1(j+1).
//
// Softmax: a thread has a row, its scores in registers; references are lazy (a row
// passes its own by 2^8 before O is rescaled), sums in fp32.
//
// A weight of 0 times an infinity or NaN would not be 0 in the product: values past
// a sequence's end are cleared in shared memory, and on tiles that some query sees
// in part, values that are not finite are cleared and added to the rows that see
// them at the end (two warps look for them while the scores are under way).
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

constexpr int kLpTile = 128;                 // queries of a tile, and keys
constexpr int kLpBlock = 2 * kLpTile;        // queries of a CTA
constexpr int kLpChunk = kLpTile * 128;      // bytes of 128 tokens of 64 values
constexpr int kLpSlots = 8;
constexpr int kLpThreads = 384;
constexpr int kLpLoadWarp = 8, kLpMmaWarp = 9, kLpFixWarp = 10;
constexpr float kLpLazy = 8.f;               // log2 by which a score may pass its row's reference
constexpr float kLowest = -3.402823466e38f;
constexpr uint64_t kLpDrainNs = 1000000000ull;

constexpr int kLpQ = 0;                              // [tile][3 chunks]
constexpr int kLpRing = kLpQ + 6 * kLpChunk;
constexpr int kLpBars = kLpRing + kLpSlots * kLpChunk;
constexpr int kLpNumBars = 2 * kLpSlots + 2 + 2 + 2 + 2 + 2 + 1 + 1;
constexpr int kLpMisc = kLpBars + kLpNumBars * 8;
constexpr int kLpSmem = kLpMisc + 64 + 1024;
static_assert(kLpSmem + 256 <= 232448 && kLpMisc % 8 == 0, "shared memory");

constexpr uint32_t kLpTmemS = 0, kLpTmemO = 256;  // columns, 128 for each tile

struct LpMaps {
  CUtensorMap q, k, k_rope, v;
};

// A block's entry and place: queries q0 .. of `n` (the first at token q_at), m keys from k_at.
struct LpBlock {
  int q_at, n, k_at, m, first;
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

template <typename T>
__global__ void __launch_bounds__(kLpThreads, 1)
    qsa_latent_prefill_kernel(const __grid_constant__ LatentPrefillParams p, const __grid_constant__ LpMaps maps) {
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t kExp = kBf16 ? 0x7f80u : 0x7c00u;  // exponent bits of an infinity or NaN
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_s = smem_u32(smem_raw);
  const uint32_t base_s = (raw_s + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base_s - raw_s);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kLpBars);
  uint64_t* full = bars;               // [slots] TMA -> products
  uint64_t* empty = full + kLpSlots;   // [slots] products -> TMA
  uint64_t* q_full = empty + kLpSlots; // [2]
  uint64_t* s_full = q_full + 2;       // [2] products -> softmax
  uint64_t* p_full = s_full + 2;       // [2] softmax -> products
  uint64_t* o_full = p_full + 2;       // [2] products -> softmax
  uint64_t* v_full = o_full + 2;       // [2] TMA -> fixers: the values of a tile that they go through
  uint64_t* fixed = v_full + 2;        // fixers -> products, softmax
  uint64_t* drain = fixed + 1;
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(smem + kLpMisc);
  const uint32_t tries = tries_of(p.wait_limit_ns);
  volatile int* odd_values = reinterpret_cast<volatile int*>(smem + kLpMisc + 12);  // values that were cleared
  LpBlock* found = reinterpret_cast<LpBlock*>(smem + kLpMisc + 16);

  const int head = (int)(blockIdx.x % p.heads), block = (int)(blockIdx.x / p.heads);
  if (tid == 0) {
    for (int i = 0; i < kLpSlots; ++i) mbar_init(full + i, 1), mbar_init(empty + i, 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(q_full + t, 1);
      mbar_init(s_full + t, 1);
      mbar_init(p_full + t, 128);
      mbar_init(o_full + t, 1);
      mbar_init(v_full + t, 1);
    }
    mbar_init(fixed, 64);
    mbar_init(drain, 1);
    *odd_values = 0;
    *found = LpBlock{0, 0, 0, 0, -1};  // a block past the last one
    fence_mbar_init();
  }
  if (warp == kLpMmaWarp) {
    tmem_alloc(tmem_at, 512);
    tmem_relinquish();
    tc_fence_before();
  }
  // the entry that the block belongs to: blocks of an entry run from its end, the
  // longest first
  {
    __shared__ int warp_sum[kLpThreads / 32];
    int before = 0;  // blocks of the entries before this round's
    __syncwarp();
    __syncthreads();
    for (int e0 = 0; e0 < p.entries; e0 += kLpThreads) {
      const int e = e0 + tid;
      int q0 = 0, n = 0;
      if (e < p.entries) {
        q0 = max(__ldg(p.cu_q + e), 0);
        n = max(min(__ldg(p.cu_q + e + 1), p.q_tokens) - q0, 0);
      }
      const int mine = (n + kLpBlock - 1) / kLpBlock;
      int upto = mine;
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
      if (block >= upto - mine && block < upto) {
        const int k0 = min(max(__ldg(p.cu_k + e), 0), p.k_tokens);
        LpBlock b;
        b.q_at = q0, b.n = n, b.k_at = k0;
        b.m = max(min(__ldg(p.cu_k + e + 1), p.k_tokens) - k0, 0);
        b.first = (upto - 1 - block) * kLpBlock;
        *found = b;
      }
      before += total;
      __syncthreads();
      if (block < before) break;
    }
  }
  __syncwarp();
  __syncthreads();
  tc_fence_after();
  constexpr uint32_t tmem = 0;  // all of it is this block's
  const LpBlock b = *found;
  bool failed = false;
  // keys that tile t's last query sees, in tiles of 128
  auto key_tiles = [&](int t) -> int {
    const int rows = min(b.n - b.first - t * kLpTile, kLpTile);
    if (b.first < 0 || rows <= 0) return 0;
    const int seen = p.causal ? min((int64_t)b.m, (int64_t)b.first + t * kLpTile + rows + b.m - b.n) : b.m;
    return seen > 0 ? (seen + kLpTile - 1) / kLpTile : 0;
  };
  const int nk0 = key_tiles(0), nk1 = key_tiles(1), nk = max(nk0, nk1);
  // tiles from here on hold a key that some query of the block does not see, or
  // that lies past the sequence
  const int whole = min(p.causal ? max(b.first + (b.m - b.n) + 1, 0) : b.m, b.m) / kLpTile;

  if (warp >= kLpLoadWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;\n");
    if (warp == kLpLoadWarp && lane == 0 && nk > 0) {
      // ================================ TMA =================================
      for (int t = 0; t < 2; ++t) {
        if ((t == 0 ? nk0 : nk1) == 0) continue;
        mbar_expect(q_full + t, 3 * kLpChunk);
        for (int c = 0; c < 3; ++c)
          tma_3d(base_s + kLpQ + (3 * t + c) * kLpChunk, &maps.q, q_full + t, 64 * c, head, b.q_at + b.first + t * kLpTile);
      }
      int pos = 0;
      for (int j = 0; j < nk && !failed; ++j)
        for (int c = 0; c < 5; ++c, ++pos) {
          const int s = pos % kLpSlots;
          const bool fix = c >= 3 && j >= whole;
          // a tile's values are brought both or not at all
          for (int at = pos; at <= (c == 3 ? pos + 1 : pos) && !failed; ++at)
            failed = at >= kLpSlots &&
                     !wait_tries(empty + at % kLpSlots, (uint32_t)((at / kLpSlots - 1) & 1), tries);
          if (failed) break;
          // values for the fixers land on a barrier of their own, each phase of which
          // they wait for; the products wait for the fixers then
          uint64_t* bar = fix ? v_full + (j - whole) % 2 : full + s;
          if (!fix || c == 3) mbar_expect(bar, fix ? 2 * kLpChunk : kLpChunk);
          if (fix) mbar_arrive(full + s);
          const uint32_t dst = base_s + kLpRing + s * kLpChunk;
          const int at = b.k_at + j * kLpTile;
          if (c < 2)
            tma_3d(dst, &maps.k, bar, 64 * c, head, at);
          else if (c == 2)
            tma_2d(dst, &maps.k_rope, bar, 0, at);
          else
            tma_3d(dst, &maps.v, bar, 64 * (c - 3), head, at);
        }
      const int fix_tiles = pos >= 5 * whole + 5 ? pos / 5 - whole : 0;  // whose two copies are both under way
      // all copies have landed before the block leaves (the usual end: the products took them)
      for (int t = 0; t < 2; ++t)
        if ((t == 0 ? nk0 : nk1) > 0 && !mbar_wait_bounded(q_full + t, 0u, kLpDrainNs)) failed = true;
      for (int s = 0; s < kLpSlots; ++s) {
        const int fills = pos > s ? (pos - s + kLpSlots - 1) / kLpSlots : 0;
        if (fills > 0 && !mbar_wait_bounded(full + s, (uint32_t)((fills - 1) & 1), kLpDrainNs)) failed = true;
      }
      for (int f = max(fix_tiles - 2, 0); f < fix_tiles; ++f)
        if (!mbar_wait_bounded(v_full + f % 2, (uint32_t)((f / 2) & 1), kLpDrainNs)) failed = true;
    } else if (warp == kLpMmaWarp && nk > 0) {
      // ============================== products ==============================
      constexpr uint32_t kIdescS = idesc_f16(128, kLpTile, kBf16, false);
      constexpr uint32_t kIdescO = idesc_f16(128, 128, kBf16, true), kIdescHalf = idesc_f16(128, 64, kBf16, true);
      auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        if (!__all_sync(0xffffffffu, wait_tries(bar, parity, tries))) return false;
        tc_fence_after();
        return true;
      };
      auto wait_slot = [&](int pos) -> bool { return wait(full + pos % kLpSlots, (uint32_t)((pos / kLpSlots) & 1)); };
      auto scores = [&](int t, int j) -> bool {  // S_t = Q_t K(j)^T
        const bool last = t == 1 || j >= nk1;    // of the tile's users
#pragma unroll 1
        for (int c = 0; c < 3; ++c) {
          const int pos = 5 * j + c;
          if (!wait_slot(pos)) return false;
          const uint32_t a0 = desc_low(base_s + kLpQ) + (3 * t + c) * (kLpChunk / 16);
          const uint32_t b0 = desc_low(base_s + kLpRing) + pos % kLpSlots * (kLpChunk / 16);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_f16_ss(tmem + kLpTmemS + t * 128, a0 + kk * 2, b0 + kk * 2, kIdescS, kk > 0 ? 1u : c > 0);
          if (last) warp_commit(empty + pos % kLpSlots);
        }
        warp_commit(s_full + t);
        return true;
      };
      auto weigh = [&](int t, int j) -> bool {  // O_t += P_t V(j)
        const bool last = t == 1 || j >= nk1;
        if (!wait(p_full + t, (uint32_t)(j & 1))) return false;
        if (j >= whole && !wait(fixed, (uint32_t)((j - whole) & 1))) return false;
        const int pos = 5 * j + 3, s0 = pos % kLpSlots;
        if (!wait_slot(pos) || !wait_slot(pos + 1)) return false;
        const uint32_t d = tmem + kLpTmemO + t * 128, a = tmem + kLpTmemS + t * 128;
        if (s0 + 1 < kLpSlots) {  // both halves of the values in one product
          const uint32_t b0 = desc_low(base_s + kLpRing, kLpChunk) + s0 * (kLpChunk / 16);
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) mma_f16_ts(d, a + kk * 8, b0 + kk * 128, kIdescO, kk > 0 ? 1u : j > 0);
        } else {
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {
            const uint32_t b0 = desc_low(base_s + kLpRing) + (pos + c) % kLpSlots * (kLpChunk / 16);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk) mma_f16_ts(d + c * 64, a + kk * 8, b0 + kk * 128, kIdescHalf, kk > 0 ? 1u : j > 0);
          }
        }
        if (last) {
          warp_commit(empty + s0);
          warp_commit(empty + (pos + 1) % kLpSlots);
        }
        warp_commit(o_full + t);
        return true;
      };
      for (int t = 0; t < 2 && !failed; ++t)
        if ((t == 0 ? nk0 : nk1) > 0) failed = !(wait(q_full + t, 0u) && scores(t, 0));
#pragma unroll 1
      for (int j = 0; j < nk && !failed; ++j)
#pragma unroll 1
        for (int t = 0; t < 2 && !failed; ++t) {
          const int tiles = t == 0 ? nk0 : nk1;
          if (j < tiles) failed = !weigh(t, j) || (j + 1 < tiles && !scores(t, j + 1));
        }
      warp_commit(drain);
      if (!mbar_wait_bounded(drain, 0u, kLpDrainNs)) failed = true;
    } else if (warp >= kLpFixWarp) {
      // ====================== values that must not count ====================
      const int at = tid - 32 * kLpFixWarp;  // of 64 threads
#pragma unroll 1
      for (int j = whole; j < nk; ++j) {
        bool any = false;
        const int f = j - whole;
        failed = !__all_sync(0xffffffffu, wait_tries(v_full + f % 2, (uint32_t)((f / 2) & 1), tries));
        if (failed) break;
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          const int pos = 5 * j + 3 + c;
          uint8_t* v = smem + kLpRing + pos % kLpSlots * kLpChunk;
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
        }
        if (any) *odd_values = 1;
        fence_proxy_async_smem();
        mbar_arrive(fixed);
      }
    }
    __syncwarp();
  } else {
    // ========================== softmax, results ===========================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;\n");
    const int t = warp >> 2;
    const int tiles = t == 0 ? nk0 : nk1;
    const int q4 = warp & 3;
    const uint32_t lane_base = (uint32_t)(q4 * 32) << 16;
    const uint32_t s_at = tmem + lane_base + kLpTmemS + t * 128, o_at = tmem + lane_base + kLpTmemO + t * 128;
    const int i = b.first + t * kLpTile + q4 * 32 + lane;  // the thread's query
    const int64_t seen = p.causal ? min((int64_t)b.m, (int64_t)i + b.m - b.n + 1) : b.m;  // keys that it sees
    const bool valid = b.first >= 0 && i < b.n;
    float r = kLowest, l = 0.f;
#pragma unroll 1
    for (int j = 0; j < tiles; ++j) {
      if (!failed) failed = !wait_tries(s_full + t, (uint32_t)(j & 1), tries);
      failed = __any_sync(0xffffffffu, failed);
      if (failed) break;
      tc_fence_after();
      float s[4][32];
      tmem_ld_2x32_wait(s_at, s_at + 32, s[0], s[1]);
      tmem_ld_2x32_wait(s_at + 64, s_at + 96, s[2], s[3]);
      const int left = (int)min((int64_t)kLpTile, seen - (int64_t)j * kLpTile);  // visible columns of the tile
      if (p.negative) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int k = 0; k < 32; ++k) s[c][k] = -s[c][k];
      }
      if (__any_sync(0xffffffffu, left < kLpTile)) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int k = 0; k < 32; ++k) s[c][k] = 32 * c + k < left ? s[c][k] : -INFINITY;
      }
      float tops[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) tops[c] = max3(s[c][0], s[c][1], s[c][2]);
#pragma unroll
      for (int k = 3; k < 31; k += 2)
#pragma unroll
        for (int c = 0; c < 4; ++c) tops[c] = max3(tops[c], s[c][k], s[c][k + 1]);
#pragma unroll
      for (int c = 0; c < 4; ++c) tops[c] = fmaxf(tops[c], s[c][31]);
      const float top = fmaxf(max3(tops[0], tops[1], tops[2]), tops[3]) * p.score_scale_log2;
      const bool moves = top > r + kLpLazy;
      if (__any_sync(0xffffffffu, moves)) {
        const float next = moves ? top : r;
        const float f = ex2(r - next);
        r = next;
        l *= f;
        if (j > 0) {
          failed = !wait_tries(o_full + t, (uint32_t)((j - 1) & 1), tries);
          failed = __any_sync(0xffffffffu, failed);
          if (failed) break;
          tc_fence_after();
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
      uint64_t sum[2] = {0, 0};
      const uint64_t scale2 = pair2(p.score_scale_log2, p.score_scale_log2), back2 = pair2(-r, -r);
#pragma unroll
      for (int c = 0; c < 4; c += 2) {
        uint32_t w[32];
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
        tmem_st(s_at + 16 * c, w);
      }
      {
        float a, d;
        unpair2(add2(sum[0], sum[1]), a, d);
        l += a + d;
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(p_full + t);
    }
    if (tiles > 0 && !failed) failed = !wait_tries(o_full + t, (uint32_t)((tiles - 1) & 1), tries);
    if (nk > whole && !failed) failed = !wait_tries(fixed, (uint32_t)((nk - whole - 1) & 1), tries);
    failed = __any_sync(0xffffffffu, failed);
    if (!failed && b.first >= 0) {
      tc_fence_after();
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      const bool odd = *odd_values != 0;
      T* out = static_cast<T*>(p.out) + ((int64_t)(b.q_at + i) * p.heads + head) * 128;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        float x[32];
        if (tiles > 0) tmem_ld_wait<32>(o_at + 32 * c, x);
#pragma unroll
        for (int k = 0; k < 32; ++k) x[k] = tiles > 0 ? x[k] * inv : 0.f;
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
        if (valid) {
#pragma unroll
          for (int k = 0; k < 32; k += 8)
            *reinterpret_cast<uint4*>(out + 32 * c + k) = make_uint4(pack2<T>(x[k], x[k + 1]), pack2<T>(x[k + 2], x[k + 3]),
                                                                     pack2<T>(x[k + 4], x[k + 5]), pack2<T>(x[k + 6], x[k + 7]));
        }
      }
    }
  }

  if (failed) {
    if (p.err) atomicOr(p.err, 1);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kLpMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
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
// 128 tokens of a head, 128-byte swizzled; tokens past the end read zeros.
bool encode(CUtensorMap* map, bool bf16, const void* base, int values, int heads, int tokens, int64_t head_stride,
            int64_t stride) {
  auto fn = encode_fn();
  if (!fn) return false;
  const bool flat = heads == 0;
  const cuuint64_t dims[3] = {(cuuint64_t)values, (cuuint64_t)(flat ? tokens : heads), (cuuint64_t)tokens};
  const cuuint64_t strides[2] = {(cuuint64_t)(flat ? stride : head_stride) * 2, (cuuint64_t)stride * 2};
  const cuuint32_t box[3] = {64u, flat ? (cuuint32_t)kLpTile : 1u, (cuuint32_t)kLpTile};
  const cuuint32_t step[3] = {1u, 1u, 1u};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, flat ? 2 : 3, const_cast<void*>(base),
            dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T>
cudaError_t launch(const LatentPrefillParams& p, cudaStream_t stream) {
  // the shared memory beyond the default limit, once per device
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(ready.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(qsa_latent_prefill_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kLpSmem);
    if (e != cudaSuccess) return e;
    ready.fetch_or(bit, std::memory_order_acq_rel);
  }
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  // without keys no block loads any, and the maps stand for the queries
  const bool none = p.k_tokens == 0;
  LpMaps m;
  if (!encode(&m.q, kBf16, p.q, 192, p.heads, p.q_tokens, p.q_head_stride, p.q_stride) ||
      !encode(&m.k, kBf16, none ? p.q : p.k, 128, p.heads, none ? 1 : p.k_tokens, none ? p.q_head_stride : p.k_head_stride, none ? p.q_stride : p.k_stride) ||
      !encode(&m.k_rope, kBf16, none ? p.q : p.k_rope, 64, 0, none ? 1 : p.k_tokens, 0, none ? p.q_stride : p.k_rope_stride) ||
      !encode(&m.v, kBf16, none ? p.q : p.v, 128, p.heads, none ? 1 : p.k_tokens, none ? p.q_head_stride : p.v_head_stride, none ? p.q_stride : p.v_stride))
    return cudaErrorInvalidValue;
  // an entry's blocks are its length over 256, rounded up
  const int64_t blocks = (int64_t)p.q_tokens / kLpBlock + (p.entries < p.q_tokens ? p.entries : p.q_tokens);
  const int64_t grid = blocks * p.heads;
  if (grid > 0x7fffffffll) return cudaErrorInvalidValue;
  qsa_latent_prefill_kernel<T><<<(unsigned)grid, kLpThreads, kLpSmem, stream>>>(p, m);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_latent_prefill(const LatentPrefillParams& p, cudaStream_t stream) {
  return p.dtype == QSA_B200_DTYPE_BF16 ? launch<__nv_bfloat16>(p, stream) : launch<__half>(p, stream);
}

}  // namespace qsa
