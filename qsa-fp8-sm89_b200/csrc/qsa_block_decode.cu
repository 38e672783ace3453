// Attention over the block-scaled caches.
//
//   out[r,h] = softmax_t(q . K[t] ks[t] scale) . V[t] vs[t]  (*) sigmoid(gate)
//
// A CTA of 8 warps takes a range of one row's columns for up to 8 KV heads (a
// segment): it first turns its columns into physical slots (a table in shared
// memory), then brings them through a ring of stages by cp.async, 128 (token,
// KV head) rows of K and of V at a time: 16 tokens of 8 heads, or more tokens
// of fewer heads. A token's heads are neighbours in the cache, so a warp's loads
// run along 1 KiB. Each warp multiplies 16 tokens of one KV head with a set of
// up to 8 query heads, or two sets: a larger group goes as 2 or 4 virtual KV
// heads whose warps read the same rows of a stage. Warps that have the same
// heads and other tokens join their results in shared memory.
//
// Rows of up to 512 columns are a segment and a CTA each. Longer ones are
// planned: a scan over the rows' lengths gives every CTA of a grid that fills
// the GPU once the same number of tiles, whatever the lengths, as at most two
// pieces of rows and any whole rows between; the pieces are joined by their
// log-sums in a last kernel.
//
// The bytes bound it: 256 per token and head for 4 x 128 x group flops, so
// the tensor work is small against the rate that mma.sync reaches, while its
// register fragments take the codes from shared memory through one conversion
// (E4M3 -> f16, exact) into the product, with no operand written back:
//   S = K Q^T    m16n8k16: 16 tokens, 8 query heads. A thread's K fragments are
//                32 bytes of two tokens' rows; the order of the dims in the
//                product is theirs, and Q's fragments follow it.
//   O^T = V^T P^T  16 dims, 8 heads, 16 tokens. P goes from S's accumulator
//                layout to the operand's by movmatrix. A thread's V fragments
//                are 16 bytes of four tokens, interleaved by byte permutes.
// Measured on a B200: gathered 128-byte rows stream at 7.0 TB/s through
// cp.async (6.4 TB/s where each token's 1 KiB lies alone) while the heads of a
// token are fetched together, at 4.3 TB/s as one bulk copy a row; with a ring of
// its own for each warp, which lets the heads drift apart, this kernel lost 5 to
// 20 %. An E4M3 mma.sync is several instructions there, slower in this loop than
// the conversions with f16.
// Queries are scaled by a power of two to below 2^15 and held in f16: exact
// for a bf16 element down to 2^-28 of the head's largest. A probability times
// its token's V scale is rounded to f16 relative to a running reference W,
// held as 2^8 in f16's range: a weight keeps its 11 bits down to 2^-22 W and
// is off by 2^-33 W at most below that. Sums, maxima and accumulators are fp32.
//
// Softmax with lazy references: scores are taken against a reference m that
// moves only when one passes it by 8, weights p vs against a reference W that
// moves when one passes 128 W (2^15 in f16), so that scales may spread over any
// range. The usual tile needs one vote and no reduction. W is 2^-112 at least: a
// block of zero values has the scale 2^-126, and 2^8 over that passes fp32's range.
// With all scales at 2^-126 a weight keeps its 11 bits down to a probability of
// 2^-8 and is off by 2^-19 of the largest below that.
//
// Times: 8 rows of 90001 to 131072 tokens, 64 query on 8 KV heads: 287 us, 6.3
// TB/s of cache (a plain copy: 6.5; after some 10 ms of it the 1000 W limit lowers
// the clock and it takes 310 to 335 us); 512 rows of 64 to 2048 selected tokens:
// 234 us, 5.0 TB/s, 217 of them this kernel, where each row's start waits for its
// ring to fill, the rest planning and joining; 256 rows of 512: 57 us, 5.0 TB/s,
// one wave whose start and end (5 and 4 us) nothing covers; 4 rows of 64: 12 us,
// one chain of lookups, fetch, product and store.
#include <atomic>

#include "qsa_common.cuh"

namespace qsa {
namespace {

constexpr int kBdWarps = 8;
constexpr int kBdTile = 16;                         // tokens a warp takes at a time
constexpr int kBdTable = 2048;                      // slots of a CTA's table
static_assert(kBlockMaxColumns + kBdTable <= 0x7fffffffll, "the columns' counter");
constexpr int kBdColumns = 8;                       // columns that a thread looks up at once
constexpr int64_t kBdTwoSets = 1 << 19;             // (row, column, KV head)s from which a warp takes 16 query heads
constexpr int kBdDirect = 512;                      // columns of a row that are not planned
constexpr float kLazy = 8.f;                        // log2 by which a score may pass its reference
constexpr float kLazyW = 128.f;                     // factor by which a weight may pass its reference
constexpr float kOneW = 256.f;                      // what stands for W in f16
constexpr float kLeastW = 0x1p-112f;                // kOneW / W stays finite
constexpr float kLowest = -3.402823466e38f;

// The approximate forms (a few ulp) have no branches: 32 of the exact ones a
// thread took 3 us at the end of a segment. For x below -88 the divisor is past
// 2^126, where the approximate quotient is 0, as sigmoid rounds in bf16's range
// of normal values.
__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.0f, 1.0f + __expf(-x)); }
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ void cp_async_16_all(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_4_or_zero(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The two E4M3 codes in a word's low half as f16, exactly.
__device__ __forceinline__ uint32_t f16_of(uint32_t w) {
  uint32_t r;
  asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %1;\ncvt.rn.f16x2.e4m3x2 %0, lo;\n}\n" : "=r"(r) : "r"(w));
  return r;
}

// An 8 x 8 matrix of 16-bit elements, lane 4 i + j holding (i, 2j), (i, 2j + 1), transposed.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(x));
  return r;
}

// Of a chain of dependent launches: lets the next kernel start, and waits for
// all of the one before (nothing where the launch was an ordinary one).
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory"); }
__device__ __forceinline__ void wait_for_prerequisites() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// kSets: sets of 8 query heads of a warp. kParts: virtual KV heads of a cache
// head. kCh: cache heads of a CTA.
template <int kSets, int kParts, int kCh>
struct BdCfg {
  static constexpr int kHeads = kParts * kCh;                // virtual heads of a CTA
  static constexpr int kSplit = kBdWarps / kHeads;           // warps of a head
  static constexpr int kUnit = kSplit * kBdTile;             // tokens of a stage; the plan counts in them
  static constexpr int kRows = kUnit * kCh;                  // its K rows, and V rows: 128 / kParts
  static constexpr int kStageBytes = 2 * kRows * kHeadDim;
  static constexpr int kStages = kParts == 4 ? 6 : (kSets == 1 ? 3 : 2) * kParts;
  static constexpr int kThreads = 32 * kBdWarps;
  static constexpr int kScales = kStages * kStageBytes;             // float [stages][K, V][kRows]
  static constexpr int kTable = kScales + kStages * 2 * kRows * 4;  // int [kBdTable]
  // with two sets of heads the Q fragments lie here: uint4 [heads][k-steps][lanes]
  static constexpr int kQ = kTable + kBdTable * 4;
  static constexpr int kSmem = kQ + (kSets == 1 ? 0 : kHeads * 8 * 32 * 16);
  static constexpr int kLeft = (8 * kSets * (kHeadDim + 2) * 4 + 127) / 128 * 128;  // a warp's result
  static_assert(kHeads <= kBdWarps && kBdWarps * kLeft <= kSmem, "the warps' results fit in what is free at a segment's end");
  static_assert(2 * (kSmem + 1024) <= 228 * 1024, "two CTAs an SM");
};

template <int kSets, int kParts, int kCh>
__global__ void __launch_bounds__(32 * kBdWarps, 2) qsa_block_decode_kernel(const __grid_constant__ BlockDecodeParams p) {
  using C = BdCfg<kSets, kParts, kCh>;
  constexpr int kStages = C::kStages, kUnit = C::kUnit;
  constexpr int kRowStep = kCh * kHeadDim;  // from a token of a stage to the next
  extern __shared__ __align__(128) uint8_t smem[];
  int* table = reinterpret_cast<int*>(smem + C::kTable);
  const float* scales = reinterpret_cast<const float*>(smem + C::kScales);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int r = lane / 4, c = lane % 4;
  const uint32_t smem_s = smem_u32(smem);
  const int hgroups = p.num_kv_heads / kCh;
  const int part = warp / C::kHeads;                // this warp's share of a stage's tokens
  const int head_in = warp % C::kHeads;             // its virtual head in the CTA

  launch_dependents();
  // the CTA's range of the plan's units, and its first row
  int64_t at = 0, end = 1;
  int row = (int)(blockIdx.x / hgroups);
  if (p.plan) {
    wait_for_prerequisites();
    if ((int)blockIdx.x >= p.plan->ctas) return;
    at = p.plan->cut[blockIdx.x];
    end = p.plan->cut[blockIdx.x + 1];
    row = p.plan->first_row[blockIdx.x];
  }

#pragma unroll 1
  for (bool first = true; at < end; first = false) {
    // the segment: columns c0 .. c1 - 1 of the row for the head group hg
    int hg = (int)(blockIdx.x % hgroups), c0 = 0, slot_out = -1;
    int64_t req = p.t2r ? __ldg(p.t2r + row) : row;
    int c1 = 0;
    const int row_now = row;
    if (p.plan) {
      const int64_t row_at = p.prefix[row] * hgroups;
      const int row_units = (int)(p.prefix[row + 1] - p.prefix[row]);
      const int in_row = (int)(at - row_at);
      hg = in_row / row_units;
      const int from = in_row - hg * row_units;
      const int to = (int)min((int64_t)row_units, from + (end - at));
      c0 = from * kUnit;
      c1 = (int)min((int64_t)to * kUnit, (int64_t)p.lengths[row]);
      if (from > 0 || to < row_units) slot_out = 2 * blockIdx.x + (from > 0 ? 0 : 1);
      at += to - from;
      if (to == row_units && hg == hgroups - 1) ++row;
    } else {
      c1 = p.counts ? min(__ldg(p.counts + row), p.topk) : p.topk;
      if (req < 0 || req >= p.num_reqs) req = 0, c1 = 0;
      at = end;
    }
    const int g0 = hg * kCh;                                               // the CTA's first cache head
    const int in_group = head_in % kParts * p.part_heads;                  // this warp's first query head in its group
    const int h0 = (g0 + head_in / kParts) * p.group + in_group;
    const int heads = min(p.part_heads, p.group - in_group);

    // the queries as loaded: head r of a set, 16 dims of either half; converted
    // below, when the first tiles are under way
    uint4 q_raw[4];
    auto load_q = [&](int u) {
#pragma unroll
      for (int i = 0; i < 4; ++i) q_raw[i] = make_uint4(0u, 0u, 0u, 0u);
      if (u * 8 + r < heads) {
        const uint4* src = reinterpret_cast<const uint4*>(p.q + ((int64_t)row_now * p.num_q_heads + h0 + u * 8 + r) * kHeadDim);
        q_raw[0] = __ldg(src + 2 * c), q_raw[1] = __ldg(src + 2 * c + 1);
        q_raw[2] = __ldg(src + 8 + 2 * c), q_raw[3] = __ldg(src + 8 + 2 * c + 1);
      }
    };
    load_q(0);
    // Q fragments: f16 of q 2^e, in the order of dims of the K fragments. One
    // set of heads has them in registers, two leave them in shared memory
    uint32_t qf[kSets == 1 ? 8 : 1][2];
    uint4* q_here = reinterpret_cast<uint4*>(smem + C::kQ) + head_in * 8 * 32 + lane;
    float qs[kSets][2];   // of heads 2c, 2c + 1 of the set: 2^-e softmax_scale log2(e)
    float o[kSets][8][4]; // [set][dims 16r + 2i, + 1][head 2c, 2c + 1 of either dim]
    float m[kSets][2], l[kSets][2], W[kSets][2], inv_w[kSets][2];  // of heads 2c, 2c + 1
#pragma unroll
    for (int u = 0; u < kSets; ++u) {
#pragma unroll
      for (int h = 0; h < 2; ++h) m[u][h] = kLowest, l[u][h] = 0.f, W[u][h] = 0.f, inv_w[u][h] = 0.f;  // the first score passes
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[u][i][j] = 0.f;
    }

    // this thread's part of a fetch: 16 bytes of the rows 4i + lane / 8 of its
    // warp's, and a scale of row tid % 128 (K's in the first warps, V's in the
    // others). Row (token, head) lies at token * kCh + head; a token's chunks
    // are stored permuted, K's by (t & 1) << 2, V's by t & 6, so that the 8
    // threads of a 16-byte read phase meet no bank twice.
    const int row0 = warp * (kBdTile / kParts) + lane / 8;
    const int token0 = row0 / kCh;
    const int token_bytes = p.num_kv_heads * kHeadDim;
    const uint8_t* k_src = p.k + (g0 + row0 % kCh) * kHeadDim + lane % 8 * 16;
    const uint8_t* v_src = p.v + (g0 + row0 % kCh) * kHeadDim + lane % 8 * 16;
    const int scale_row = tid % 128;
    const float* s_src = (tid < 128 ? p.k_scales : p.v_scales) + g0 + scale_row % kCh;
    const uint32_t k_dst = smem_s + row0 * kHeadDim + ((lane % 8 ^ ((token0 & 1) << 2)) << 4);
    const uint32_t v_dst = smem_s + (C::kRows + row0) * kHeadDim + ((lane % 8 ^ (token0 & 6)) << 4);
    const uint32_t s_dst = smem_s + C::kScales + (tid / 128 * C::kRows + scale_row) * 4;
    // where this warp's fragments and scales lie in a stage
    const int own = part * kBdTile * kCh + head_in / kParts;
    const uint32_t k_at = own * kHeadDim + r * kRowStep + ((c ^ ((r & 1) << 2)) << 4);
    const uint32_t v_at = (C::kRows + own) * kHeadDim + 2 * c * kRowStep + ((r ^ (2 * c)) << 4);
    const int s_at = own + r * kCh;

#pragma unroll 1
    for (int base = c0; base < c1; base += kBdTable) {
      const int n = min(kBdTable, c1 - base);
      const int tiles = (n + kUnit - 1) / kUnit;
      if (base > c0 || !first) __syncthreads();  // the table's readers are done
      bool valid = true;
      // several columns a thread at once: an index, then its page, wait on
      // memory. Steps past the last column are left by the whole CTA.
#pragma unroll 1
      for (int i0 = 0; i0 < tiles * kUnit; i0 += kBdColumns * C::kThreads) {
        int t[kBdColumns], off[kBdColumns], page[kBdColumns];
#pragma unroll
        for (int i = 0; i < kBdColumns; ++i) {
          const int col = i0 + i * C::kThreads + tid;
          t[i] = base + col;
          if (p.indices && i0 + i * C::kThreads < n) t[i] = col < n ? __ldg(p.indices + (int64_t)row_now * p.indices_stride + t[i]) : -1;
        }
#pragma unroll
        for (int i = 0; i < kBdColumns; ++i) {
          if (i0 + i * C::kThreads >= n) break;
          const int col = i0 + i * C::kThreads + tid;
          const uint32_t lp = __umulhi(2u * (uint32_t)max(t[i], 0), p.page_mul) >> p.page_shift;
          off[i] = t[i] - (int)lp * p.page_size;
          page[i] = col < n && t[i] >= 0 && (int)lp < p.pages_per_req ? __ldg(p.btable + req * p.btable_stride + lp) : -1;
        }
#pragma unroll
        for (int i = 0; i < kBdColumns; ++i) {
          const int col = i0 + i * C::kThreads + tid;
          if (i0 + i * C::kThreads >= tiles * kUnit) break;
          const bool in = i0 + i * C::kThreads < n && page[i] >= 0 && page[i] < p.num_pages;
          if (col < tiles * kUnit) table[col] = in ? page[i] * p.page_size + off[i] : -1;
          valid = valid && (in || col >= n);
        }
      }
      const bool clean = __syncthreads_and(valid);  // only the last tile may have masked places
      const int whole = clean ? n / kUnit : 0;      // leading tiles without one

      // Row row0 + 4i of a stage: with 8 heads the token's other four or the
      // next token's first, else the same heads 4 / kCh tokens on. The bits that
      // step adds to the token are none that token0 has, so the chunk
      // permutation splits into token0's and a constant.
      auto fetch = [&](int k, int st) {
        const int* ahead = table + k * kUnit;
        if (__builtin_expect(k < whole, 1)) {
#pragma unroll
          for (int i = 0; i < 4 / kParts; ++i) {
            const int step = 4 * i / kCh;
            const int64_t from = (int64_t)ahead[token0 + step] * token_bytes;
            const int to_head = kCh == 8 ? i % 2 * 4 * kHeadDim : 0;
            cp_async_16_all((k_dst ^ ((step & 1) << 6)) + st * C::kStageBytes + i * 4 * kHeadDim, k_src + from + to_head);
            cp_async_16_all((v_dst ^ ((step & 6) << 4)) + st * C::kStageBytes + i * 4 * kHeadDim, v_src + from + to_head);
          }
          if (kParts == 1 || scale_row < C::kRows) {
            const uint32_t block = __umulhi(2u * (uint32_t)ahead[scale_row / kCh], p.block_mul) >> p.block_shift;
            cp_async_4_or_zero(s_dst + st * 2 * C::kRows * 4, s_src + (int64_t)(int)block * p.num_kv_heads, 4u);
          }
        } else if (k < tiles) {  // masked places read as zeros, whatever the cache holds
#pragma unroll 1
          for (int i = 0; i < 4 / kParts; ++i) {
            const int step = 4 * i / kCh;
            const int slot = ahead[token0 + step];
            const int64_t from = (int64_t)max(slot, 0) * token_bytes + (kCh == 8 ? i % 2 * 4 * kHeadDim : 0);
            const uint32_t bytes = slot < 0 ? 0u : 16u;
            cp_async_16((k_dst ^ ((step & 1) << 6)) + st * C::kStageBytes + i * 4 * kHeadDim, k_src + from, bytes);
            cp_async_16((v_dst ^ ((step & 6) << 4)) + st * C::kStageBytes + i * 4 * kHeadDim, v_src + from, bytes);
          }
          if (kParts == 1 || scale_row < C::kRows) {
            const int slot = ahead[scale_row / kCh];
            const uint32_t block = __umulhi(2u * (uint32_t)max(slot, 0), p.block_mul) >> p.block_shift;
            cp_async_4_or_zero(s_dst + st * 2 * C::kRows * 4, s_src + (int64_t)(int)block * p.num_kv_heads, slot < 0 ? 0u : 4u);
          }
        }
        cp_async_commit();
      };
#pragma unroll
      for (int st = 0; st < kStages - 1; ++st) fetch(st, st);

      if (base == c0) {
#pragma unroll
        for (int u = 0; u < kSets; ++u) {
          if (u > 0) load_q(u);
          float top = 0.f;
          float2 x[16];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t b[4] = {q_raw[i].x, q_raw[i].y, q_raw[i].z, q_raw[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              x[4 * i + j] = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&b[j]));
              top = fmaxf(top, fmaxf(fabsf(x[4 * i + j].x), fabsf(x[4 * i + j].y)));
            }
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          int e = 0;  // 2^e maps the largest |q| into [2^14, 2^15)
          if (top > 0.f && top <= -kLowest) e = min(max(14 + 127 - (int)(__float_as_uint(top) >> 23), -120), 120);
          const float up = __uint_as_float((uint32_t)(127 + e) << 23);
          const float down = __uint_as_float((uint32_t)(127 - e) << 23) * p.score_scale_log2;
          qs[u][0] = __shfl_sync(0xffffffffu, down, 8 * c);
          qs[u][1] = __shfl_sync(0xffffffffu, down, 8 * c + 4);
#pragma unroll
          for (int s = 0; s < 8; ++s) {  // k-step s: word s of the thread's chunks c and c + 4
            const uint32_t f0 = pack_f16(x[2 * s].x * up, x[2 * s].y * up);
            const uint32_t f1 = pack_f16(x[2 * s + 1].x * up, x[2 * s + 1].y * up);
            if constexpr (kSets == 1) {
              qf[s][0] = f0, qf[s][1] = f1;
            } else {  // the same for every part; the loop's first barrier is between this and its reading
              if (part == 0) reinterpret_cast<uint2*>(q_here + s * 32)[u] = make_uint2(f0, f1);
            }
          }
        }
      }

#pragma unroll 1
      for (int k0 = 0; k0 < tiles; k0 += kStages) {
#pragma unroll
        for (int st = 0; st < kStages; ++st) {
          if (k0 + st >= tiles) break;
          cp_async_wait<kStages - 2>();
          __syncthreads();  // the tile is there, and every warp has read the one before
          fetch(k0 + st + kStages - 1, (st + kStages - 1) % kStages);
          const uint8_t* stage = smem + st * C::kStageBytes;
          const float* sc = scales + st * 2 * C::kRows + s_at;

          // [set][token r: heads 2c, 2c+1; token r + 8: the same], of one set in
          // two chains
          float s[2][4] = {};
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint4 a4 = *reinterpret_cast<const uint4*>(stage + (k_at ^ (64 * j)));
            const uint4 b4 = *reinterpret_cast<const uint4*>(stage + (k_at ^ (64 * j)) + 8 * kRowStep);
            const uint32_t wa[4] = {a4.x, a4.y, a4.z, a4.w}, wb[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t a[4] = {f16_of(wa[i]), f16_of(wb[i]), f16_of(wa[i] >> 16), f16_of(wb[i] >> 16)};
              if constexpr (kSets == 1) {
                mma16816(s[j], a, qf[4 * j + i][0], qf[4 * j + i][1]);
              } else {
                const uint4 q4 = q_here[(4 * j + i) * 32];
                mma16816(s[0], a, q4.x, q4.y);
                mma16816(s[1], a, q4.z, q4.w);
              }
            }
          }
          if constexpr (kSets == 1) {
#pragma unroll
            for (int j = 0; j < 4; ++j) s[0][j] += s[1][j];
          }
          const float ks[2] = {sc[0], sc[8 * kCh]}, vs[2] = {sc[C::kRows], sc[C::kRows + 8 * kCh]};
          bool masked[2] = {false, false};
          if (k0 + st >= whole) {
            const int* slots = table + (k0 + st) * kUnit + part * kBdTile;
            masked[0] = slots[r] < 0, masked[1] = slots[8 + r] < 0;
          }

          // scores over the reference, probabilities, weights over theirs
          uint32_t pf[kSets][2];
#pragma unroll
          for (int u = 0; u < kSets; ++u) {
            float pr[4], w[4], x_top = -INFINITY, w_abs = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int t = j / 2, h = j % 2;
              float x = fmaf(s[u][j], ks[t] * qs[u][h], -m[u][h]);
              x = masked[t] ? -INFINITY : x;
              pr[j] = ex2(x);
              // a scale over a far smaller reference may pass fp32's range; of a
              // probability of 0 it must not
              w[j] = (pr[j] * vs[t]) * inv_w[u][h];
              x_top = fmaxf(x_top, x);
              w_abs = fmaxf(w_abs, fabsf(w[j]));
            }
            if (__any_sync(0xffffffffu, x_top > kLazy || w_abs > kLazyW * kOneW)) {
              // move the references, and what was summed against them
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float x0 = masked[0] ? -INFINITY : s[u][h] * (ks[0] * qs[u][h]);
                const float x1 = masked[1] ? -INFINITY : s[u][2 + h] * (ks[1] * qs[u][h]);
                float top = fmaxf(x0, x1);
#pragma unroll
                for (int d = 4; d <= 16; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                const float m_new = fmaxf(m[u][h], top);
                const float alpha = ex2(m[u][h] - m_new);
                pr[h] = ex2(x0 - m_new), pr[2 + h] = ex2(x1 - m_new);
                const float w0 = pr[h] * vs[0], w1 = pr[2 + h] * vs[1];
                float w_top = fmaxf(fabsf(w0), fabsf(w1));
#pragma unroll
                for (int d = 4; d <= 16; d *= 2) w_top = fmaxf(w_top, __shfl_xor_sync(0xffffffffu, w_top, d));
                const float was = W[u][h] * alpha;
                W[u][h] = fmaxf(fmaxf(was, w_top), kLeastW);
                inv_w[u][h] = kOneW / W[u][h];
                const float f = was > 0.f ? was / W[u][h] : 0.f;
                m[u][h] = m_new;
                l[u][h] *= alpha;
                w[h] = w0 * inv_w[u][h], w[2 + h] = w1 * inv_w[u][h];
#pragma unroll
                for (int i = 0; i < 8; ++i) o[u][i][h] *= f, o[u][i][2 + h] *= f;
              }
            }
            l[u][0] += pr[0] + pr[2];
            l[u][1] += pr[1] + pr[3];
            pf[u][0] = transpose8x8(pack_f16(w[0], w[1])), pf[u][1] = transpose8x8(pack_f16(w[2], w[3]));
          }
          // V: chunk r of tokens 2c, 2c+1, 8+2c, 9+2c
          uint32_t vw[4][4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4 q4 = *reinterpret_cast<const uint4*>(stage + v_at + ((j / 2) * 8 + j % 2) * kRowStep);
            vw[j][0] = q4.x, vw[j][1] = q4.y, vw[j][2] = q4.z, vw[j][3] = q4.w;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            // a dim's codes of two tokens side by side in the low half
            const uint32_t sel = i % 2 ? 0x0062 : 0x0040, sel1 = i % 2 ? 0x0073 : 0x0051;
            const uint32_t a[4] = {f16_of(__byte_perm(vw[0][i / 2], vw[1][i / 2], sel)),
                                   f16_of(__byte_perm(vw[0][i / 2], vw[1][i / 2], sel1)),
                                   f16_of(__byte_perm(vw[2][i / 2], vw[3][i / 2], sel)),
                                   f16_of(__byte_perm(vw[2][i / 2], vw[3][i / 2], sel1))};
#pragma unroll
            for (int u = 0; u < kSets; ++u) mma16816(o[u][i], a, pf[u][0], pf[u][1]);
          }
        }
      }
      cp_async_wait<0>();
    }

#pragma unroll
    for (int u = 0; u < kSets; ++u) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        W[u][h] *= 1.0f / kOneW;
#pragma unroll
        for (int d = 4; d <= 16; d *= 2) l[u][h] += __shfl_xor_sync(0xffffffffu, l[u][h], d);
      }
    }
    if (C::kSplit > 1) {
      // the warps of a head join in shared memory: each leaves its result, part
      // 0 gathers (m and l by head, values by head and dim)
      __syncthreads();
      float* left = reinterpret_cast<float*>(smem + warp * C::kLeft);  // [heads][2], then [heads][128]
#pragma unroll
      for (int u = 0; u < kSets; ++u) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int hh = u * 8 + 2 * c + h;
          if (r == 0) left[2 * hh] = m[u][h], left[2 * hh + 1] = l[u][h];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            *reinterpret_cast<float2*>(left + 16 * kSets + hh * kHeadDim + 16 * r + 2 * i) =
                make_float2(o[u][i][h] * W[u][h], o[u][i][2 + h] * W[u][h]);
        }
      }
      __syncthreads();
      if (part > 0) continue;  // the next segment's barriers hold until part 0 has read
#pragma unroll
      for (int u = 0; u < kSets; ++u) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int hh = u * 8 + 2 * c + h;
          float sum = 0.f, top = kLowest;
#pragma unroll
          for (int w = 0; w < C::kSplit; ++w)
            top = fmaxf(top, reinterpret_cast<const float*>(smem + (warp + w * C::kHeads) * C::kLeft)[2 * hh]);
#pragma unroll
          for (int i = 0; i < 8; ++i) o[u][i][h] = o[u][i][2 + h] = 0.f;
#pragma unroll 2
          for (int w = 0; w < C::kSplit; ++w) {
            const float* from = reinterpret_cast<const float*>(smem + (warp + w * C::kHeads) * C::kLeft);
            const float f = ex2(from[2 * hh] - top);
            sum = fmaf(from[2 * hh + 1], f, sum);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float2 v = *reinterpret_cast<const float2*>(from + 16 * kSets + hh * kHeadDim + 16 * r + 2 * i);
              o[u][i][h] = fmaf(f, v.x, o[u][i][h]), o[u][i][2 + h] = fmaf(f, v.y, o[u][i][2 + h]);
            }
          }
          m[u][h] = top, l[u][h] = sum, W[u][h] = 1.f;
        }
      }
    }

#pragma unroll
    for (int u = 0; u < kSets; ++u) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int hh = u * 8 + 2 * c + h;
        if (hh >= heads) continue;
        const float f = l[u][h] == 0.f ? 0.f : W[u][h] / l[u][h];  // a NaN sum stays one
        float x[16];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[2 * i] = o[u][i][h] * f, x[2 * i + 1] = o[u][i][2 + h] * f;
        if (slot_out >= 0) {
          const int64_t to = ((int64_t)slot_out * C::kHeads + head_in) * p.part_heads + hh;
          float4* dst = reinterpret_cast<float4*>(p.part_o + to * kHeadDim + 16 * r);
#pragma unroll
          for (int i = 0; i < 4; ++i) dst[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
          if (r == 0) p.part_lse[to] = l[u][h] == 0.f ? -INFINITY : m[u][h] + log2f(l[u][h]);
          continue;
        }
        const int64_t hr = (int64_t)row_now * p.num_q_heads + h0 + hh;
        if (p.gate) {
          const uint4* src = reinterpret_cast<const uint4*>(p.gate + hr * kHeadDim + 16 * r);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint4 w4 = __ldg(src + i);
            const uint32_t b[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 gt = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&b[j]));
              x[8 * i + 2 * j] *= sigmoid(gt.x), x[8 * i + 2 * j + 1] *= sigmoid(gt.y);
            }
          }
        }
        uint32_t b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
          b[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
        uint4* dst = reinterpret_cast<uint4*>(p.out + hr * kHeadDim + 16 * r);
        dst[0] = make_uint4(b[0], b[1], b[2], b[3]);
        dst[1] = make_uint4(b[4], b[5], b[6], b[7]);
      }
    }
  }
}

// Valid length of each row for the plan: its count, or the place past its last
// index that is not negative. A CTA a row, from the row's end.
constexpr int kLenThreads = 256;
__global__ void __launch_bounds__(kLenThreads) qsa_block_lengths_kernel(const __grid_constant__ BlockDecodeParams p) {
  launch_dependents();
  const int row = blockIdx.x;
  const int count = p.counts ? min(max(__ldg(p.counts + row), 0), p.topk) : p.topk;
  const int32_t* list = p.indices + (int64_t)row * p.indices_stride;
  int len = 0;
  for (int hi = count; hi > 0 && len == 0; hi -= 4 * kLenThreads) {
    int last = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int col = hi - 1 - (int)threadIdx.x - i * kLenThreads;
      if (col >= 0 && __ldg(list + col) >= 0) last = max(last, col + 1);
    }
    len = __reduce_max_sync(0xffffffffu, last);
    __shared__ int top[kLenThreads / 32];
    if (threadIdx.x % 32 == 0) top[threadIdx.x / 32] = len;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kLenThreads / 32; ++w) len = max(len, top[w]);
    __syncthreads();
  }
  if (threadIdx.x == 0) p.lengths[row] = len;
}

// Plans the segments: prefix sums of the rows' units (a row without a valid
// place has one: its zeros), the number of CTAs that share them, and the row
// that each begins in. One CTA; a thread takes consecutive rows.
constexpr int kPlanThreads = 1024;
constexpr int kJoinFew = 8;      // pieces that a warp joins
constexpr int kPlanTokens = 128;  // columns a CTA gets at least (and two units), so that small work has few pieces
__global__ void __launch_bounds__(kPlanThreads) qsa_block_plan_kernel(const __grid_constant__ BlockDecodeParams p, int max_ctas) {
  launch_dependents();
  wait_for_prerequisites();
  const int t = threadIdx.x;
  const int unit = kBdWarps / p.cta_heads * kBdTile;
  const int hgroups = p.virtual_heads / p.cta_heads;
  const int each = (p.rows + kPlanThreads - 1) / kPlanThreads;
  const int r0 = min(t * each, p.rows), r1 = min(r0 + each, p.rows);
  int64_t mine = 0;
  for (int r = r0; r < r1; ++r) {
    const int req = p.t2r ? __ldg(p.t2r + r) : r;
    int len = p.indices ? p.lengths[r] : p.counts ? min(max(__ldg(p.counts + r), 0), p.topk) : p.topk;
    if (req < 0 || req >= p.num_reqs) len = 0;
    p.lengths[r] = len;
    mine += max(1, (int)(((int64_t)len + unit - 1) / unit));
  }
  __shared__ int64_t sums[kPlanThreads / 32];
  __shared__ int listed[2];
  if (t < 2) listed[t] = 0;
  int64_t run = mine;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int64_t below = __shfl_up_sync(0xffffffffu, run, d);
    if (t % 32 >= d) run += below;
  }
  if (t % 32 == 31) sums[t / 32] = run;
  __syncthreads();
  if (t < 32) {
    int64_t s = sums[t];
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int64_t below = __shfl_up_sync(0xffffffffu, s, d);
      if (t >= d) s += below;
    }
    sums[t] = s;
  }
  __syncthreads();
  const int64_t total = sums[kPlanThreads / 32 - 1];
  const int64_t units = total * hgroups;
  const int least = max(kPlanTokens / unit, 2);
  const int ctas = (int)min((int64_t)max_ctas, (units + least - 1) / least);
  int64_t before = run - mine + (t >= 32 ? sums[t / 32 - 1] : 0);
  for (int r = r0; r < r1; ++r) {
    p.prefix[r] = before;
    before += max(1, (int)(((int64_t)p.lengths[r] + unit - 1) / unit));
  }
  if (t == 0) p.plan->ctas = ctas, p.prefix[p.rows] = total;
  __syncthreads();
  // CTA b begins at unit b units / ctas, in the last row that begins before it
  for (int b = t; b <= ctas; b += kPlanThreads) {
    const int64_t x = b * units / ctas;
    int lo = 0, hi = p.rows - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (p.prefix[mid] * hgroups <= x) lo = mid;
      else hi = mid - 1;
    }
    p.plan->cut[b] = x;
    p.plan->first_row[b] = lo;
    // a row and head group that this cut is the first to cut is joined: its last
    // piece is of the last CTA that begins before its end
    const int64_t row_at = p.prefix[lo] * hgroups, row_units = p.prefix[lo + 1] - p.prefix[lo];
    const int hg = (int)(x - row_at) / (int)row_units;
    const int64_t begin = row_at + hg * row_units;
    if (b > 0 && b < ctas && x > begin && (b - 1) * units / ctas <= begin) {
      const int last = (int)(((begin + row_units) * ctas - 1) / units);
      const bool many = last - b + 2 > kJoinFew;
      const int at = atomicAdd(&listed[many], 1);  // the order of the list does not matter
      p.plan->joins[many ? kPlanMaxCtas - 1 - at : at] = make_int4(lo, hg, b, last);
    }
  }
  __syncthreads();
  if (t < 2) p.plan->num_joins[t] = listed[t];
}

// Joins the pieces of the rows that the plan cut, in the plan's order: a warp a
// query head where they are few, a CTA a query head where a long row was cut
// into many (256 pieces one after the other took a warp 40 us).
constexpr int kJoinThreads = 256, kJoinCtas = 6;  // CTAs an SM
__global__ void __launch_bounds__(kJoinThreads, kJoinCtas) qsa_block_join_kernel(const __grid_constant__ BlockDecodeParams p) {
  __shared__ float tops[8], sums[8];
  __shared__ float4 accs[8][32];
  wait_for_prerequisites();
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int heads = p.cta_heads * p.part_heads;  // of a head group, with those that a part lacks
  // One query head: `pieces` of the CTAs from what.z - 1 on, every `step`-th from `first`
  struct Sum {
    float top, sum;
    float4 acc;
  };
  auto locate = [&](const int4& what, int head, int& in_group) {
    const int gv = what.y * p.cta_heads + head / p.part_heads;
    in_group = gv % p.head_parts * p.part_heads + head % p.part_heads;
    return ((int64_t)what.x * p.num_q_heads + gv / p.head_parts * p.group + in_group) * kHeadDim + lane * 4;
  };
  auto gather = [&](const int4& what, int head, int first, int step) {
    auto piece = [&](int at) -> int64_t {  // the first piece is its CTA's second kind
      return (int64_t)(2 * at + (at == what.z - 1 ? 1 : 0)) * heads + head;
    };
    Sum s = {-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
    for (int at = what.z - 1 + first + lane * step; at <= what.w; at += 32 * step) s.top = fmaxf(s.top, p.part_lse[piece(at)]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s.top = fmaxf(s.top, __shfl_xor_sync(0xffffffffu, s.top, d));
#pragma unroll 4
    for (int at = what.z - 1 + first; at <= what.w; at += step) {
      const int64_t from = piece(at);
      const float lse = p.part_lse[from];
      const float4 v = *reinterpret_cast<const float4*>(p.part_o + from * kHeadDim + lane * 4);
      const float w = lse == -INFINITY ? 0.f : exp2f(lse - s.top);
      s.sum += w;
      s.acc.x = fmaf(w, v.x, s.acc.x), s.acc.y = fmaf(w, v.y, s.acc.y);
      s.acc.z = fmaf(w, v.z, s.acc.z), s.acc.w = fmaf(w, v.w, s.acc.w);
    }
    return s;
  };
  auto finish = [&](const Sum& s, int64_t off) {
    const float inv = s.sum == 0.f ? 0.f : 1.0f / s.sum;
    float x[4] = {s.acc.x * inv, s.acc.y * inv, s.acc.z * inv, s.acc.w * inv};
    if (p.gate) {
#pragma unroll
      for (int d = 0; d < 4; ++d) x[d] *= sigmoid(__bfloat162float(p.gate[off + d]));
    }
    const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
    *reinterpret_cast<uint2*>(p.out + off) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  };
  int in_group;
  const int few = p.plan->num_joins[0] * heads, many = p.plan->num_joins[1] * heads;
  for (int item = blockIdx.x * 8 + warp; item < few; item += gridDim.x * 8) {
    const int4 what = p.plan->joins[item / heads];
    const int64_t off = locate(what, item % heads, in_group);
    if (in_group < p.group) finish(gather(what, item % heads, 0, 1), off);
  }
  for (int item = blockIdx.x; item < many; item += gridDim.x) {
    const int4 what = p.plan->joins[kPlanMaxCtas - 1 - item / heads];
    const int64_t off = locate(what, item % heads, in_group);
    if (in_group >= p.group) continue;
    const Sum mine = gather(what, item % heads, warp, 8);
    if (lane == 0) tops[warp] = mine.top, sums[warp] = mine.sum;
    accs[warp][lane] = mine.acc;
    __syncthreads();
    if (warp == 0) {
      Sum all = {-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll
      for (int i = 0; i < 8; ++i) all.top = fmaxf(all.top, tops[i]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float w = tops[i] == -INFINITY ? 0.f : exp2f(tops[i] - all.top);
        all.sum = fmaf(w, sums[i], all.sum);
        const float4 v = accs[i][lane];
        all.acc.x = fmaf(w, v.x, all.acc.x), all.acc.y = fmaf(w, v.y, all.acc.y);
        all.acc.z = fmaf(w, v.z, all.acc.z), all.acc.w = fmaf(w, v.w, all.acc.w);
      }
      finish(all, off);
    }
    __syncthreads();
  }
}

int sm_count() {
  static std::atomic<int> known[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  int n = known[dev & 63].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) n = 148;
    known[dev & 63].store(n, std::memory_order_relaxed);
  }
  return n;
}

int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }
int planned_ctas() { return min(2 * sm_count(), kPlanMaxCtas); }

// Launches a kernel that waits for its prerequisites itself (early = true: it
// may start before the stream's last kernel has ended).
template <typename Kernel, typename... Args>
cudaError_t start(Kernel kernel, dim3 grid, int threads, int smem, bool early, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = early ? 1 : 0;
  return cudaLaunchKernelEx(&config, kernel, args...);
}

template <int kSets, int kParts, int kCh>
cudaError_t launch(const BlockDecodeParams& p, cudaStream_t stream) {
  using C = BdCfg<kSets, kParts, kCh>;
  // the shared memory beyond the default limit, once per device
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(ready.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(qsa_block_decode_kernel<kSets, kParts, kCh>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return e;
    ready.fetch_or(bit, std::memory_order_acq_rel);
  }
  const int64_t grid = p.plan ? planned_ctas() : (int64_t)p.rows * (p.num_kv_heads / kCh);
  if (grid > 0x7fffffffll) return cudaErrorInvalidValue;
  return start(qsa_block_decode_kernel<kSets, kParts, kCh>, dim3((unsigned)grid), C::kThreads, C::kSmem, p.plan != nullptr, stream, p);
}

cudaError_t launch_main(const BlockDecodeParams& p, cudaStream_t stream) {
  const int ch = p.cta_heads / p.head_parts;
  switch ((p.part_heads > 8 ? 64 : 0) + p.head_parts * 8 + ch) {
    case 8 + 1: return launch<1, 1, 1>(p, stream);
    case 8 + 2: return launch<1, 1, 2>(p, stream);
    case 8 + 4: return launch<1, 1, 4>(p, stream);
    case 8 + 8: return launch<1, 1, 8>(p, stream);
    case 16 + 1: return launch<1, 2, 1>(p, stream);
    case 16 + 2: return launch<1, 2, 2>(p, stream);
    case 16 + 4: return launch<1, 2, 4>(p, stream);
    case 32 + 1: return launch<1, 4, 1>(p, stream);
    case 32 + 2: return launch<1, 4, 2>(p, stream);
    case 72 + 1: return launch<2, 1, 1>(p, stream);
    case 72 + 2: return launch<2, 1, 2>(p, stream);
    case 72 + 4: return launch<2, 1, 4>(p, stream);
    case 72 + 8: return launch<2, 1, 8>(p, stream);
    case 80 + 1: return launch<2, 2, 1>(p, stream);
    case 80 + 2: return launch<2, 2, 2>(p, stream);
    case 80 + 4: return launch<2, 2, 4>(p, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace

int64_t block_decode_plan(BlockDecodeParams& p) {
  // A group above 8: two sets of heads a warp share the conversions (128 rows of
  // 2000 tokens, 16 heads for each of 8 KV heads: 138 us against 170), but make a
  // tile's work longer, which shows where a CTA has few tiles (61 rows of 3000
  // tokens on average, 20 heads for one KV head: 61 us against 52)
  const bool large = (int64_t)p.rows * p.num_kv_heads * p.topk >= kBdTwoSets;
  p.head_parts = p.group <= 8 ? 1 : p.group <= 16 ? (large ? 1 : 2) : (large ? 2 : 4);
  p.part_heads = (p.group + p.head_parts - 1) / p.head_parts;
  p.virtual_heads = p.num_kv_heads * p.head_parts;
  p.cta_heads = p.head_parts;
  while (p.cta_heads < kBdWarps && p.virtual_heads % (2 * p.cta_heads) == 0) p.cta_heads *= 2;
  // mul = ceil(2^(31 + shift) / d) with d <= 2^shift: n mul exceeds
  // n 2^(31 + shift) / d by less than n, so n / d is exact for n < 2^31
  auto reciprocal = [](uint32_t d, uint32_t& mul, uint32_t& shift) {
    shift = 0;
    while ((1ll << shift) < d) ++shift;
    mul = (uint32_t)((((uint64_t)1 << (31 + shift)) + d - 1) / d);
  };
  reciprocal(p.block_size, p.block_mul, p.block_shift);
  reciprocal(p.page_size, p.page_mul, p.page_shift);
  p.planned = p.topk > kBdDirect;
  if (!p.planned) return 0;
  const int64_t pieces = 2ll * planned_ctas() * p.cta_heads * p.part_heads;
  return align256(pieces * kHeadDim * 4) + align256(pieces * 4) + align256((int64_t)sizeof(BlockDecodePlan)) +
         align256(8ll * (p.rows + 1)) + align256(4ll * p.rows);
}

void block_decode_place(BlockDecodeParams& p, void* workspace) {
  char* at = static_cast<char*>(workspace);
  const int64_t pieces = 2ll * planned_ctas() * p.cta_heads * p.part_heads;
  auto take = [&](int64_t bytes) {
    char* here = at;
    at += align256(bytes);
    return here;
  };
  p.part_o = reinterpret_cast<float*>(take(pieces * kHeadDim * 4));
  p.part_lse = reinterpret_cast<float*>(take(pieces * 4));
  p.plan = reinterpret_cast<BlockDecodePlan*>(take(sizeof(BlockDecodePlan)));
  p.prefix = reinterpret_cast<int64_t*>(take(8ll * (p.rows + 1)));
  p.lengths = reinterpret_cast<int*>(take(4ll * p.rows));
}

cudaError_t launch_block_decode(const BlockDecodeParams& p, cudaStream_t stream) {
  if (!p.plan) return launch_main(p, stream);
  cudaError_t e = cudaSuccess;
  if (p.indices) e = start(qsa_block_lengths_kernel, dim3(p.rows), kLenThreads, 0, false, stream, p);
  if (e == cudaSuccess) e = start(qsa_block_plan_kernel, dim3(1), kPlanThreads, 0, p.indices != nullptr, stream, p, planned_ctas());
  if (e == cudaSuccess) e = launch_main(p, stream);
  if (e == cudaSuccess) e = start(qsa_block_join_kernel, dim3(kJoinCtas * sm_count()), kJoinThreads, 0, true, stream, p);
  return e;
}

}  // namespace qsa
