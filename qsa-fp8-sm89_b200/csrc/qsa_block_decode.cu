// Attention over the block-scaled caches.
//
//   out[r,h] = softmax_t(q . K[t] ks[t] scale) . V[t] vs[t]  (*) sigmoid(gate)
//
// A CTA of 8 warps takes a range of one row's columns for up to 8 KV heads (a
// segment): it first turns its columns into physical slots (a table in shared
// memory), then brings them through a ring of stages by cp.async, 128 (token,
// KV head) rows of K and of V at a time: 16 tokens of 8 heads, or more tokens
// of fewer heads. A token's heads are neighbours in the cache, so a warp's loads
// run along 1 KiB. Each warp multiplies 16 tokens of one head; with fewer than
// 8 heads the warps of a head join their results in shared memory.
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
// range. The usual tile needs one vote and no reduction.
#include <atomic>

#include "qsa_common.cuh"

namespace qsa {
namespace {

constexpr int kBdWarps = 8;
constexpr int kBdTile = 16;                         // tokens a warp takes at a time
constexpr int kBdTable = 2048;                      // slots of a CTA's table
constexpr int kBdDirect = 512;                      // columns of a row that are not planned
constexpr int kBdRows = kBdTile * kBdWarps;          // K rows of a stage, and V rows
constexpr int kStageBytes = 2 * kBdRows * kHeadDim;
constexpr float kLazy = 8.f;                        // log2 by which a score may pass its reference
constexpr float kLazyW = 128.f;                     // factor by which a weight may pass its reference
constexpr float kOneW = 256.f;                      // what stands for W in f16
constexpr float kLowest = -3.402823466e38f;

__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + expf(-x)); }
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

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Logical tokens (negative: masked) to physical slots, -1 where masked.
template <int N>
__device__ __forceinline__ void column_slots(const BlockDecodeParams& p, int64_t req, int (&t)[N]) {
  int page[N], off[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int lp = t[i] / p.page_size;
    off[i] = t[i] - lp * p.page_size;
    page[i] = t[i] >= 0 && lp < p.pages_per_req ? __ldg(p.btable + req * p.btable_stride + lp) : -1;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) t[i] = page[i] < 0 || page[i] >= p.num_pages ? -1 : page[i] * p.page_size + off[i];
}

// kHeads: query heads of a warp's tile, 8 or 16 (which need the registers of
// both CTAs). kCh: cache heads of a CTA.
template <int kHeads, int kCh>
struct BdCfg {
  static constexpr int kSets = kHeads / 8;
  static constexpr int kStages = kHeads == 8 ? 3 : 6;
  static constexpr int kThreads = 32 * kBdWarps;
  static constexpr int kCtas = kHeads == 8 ? 2 : 1;  // per SM
  static constexpr int kScales = kStages * kStageBytes;              // float [stages][K, V][kBdRows]
  static constexpr int kTable = kScales + kStages * 2 * kBdRows * 4;  // int [kBdTable]
  static constexpr int kSmem = kTable + kBdTable * 4;
  static constexpr int kLeft = (kHeads * (kHeadDim + 2) * 4 + 127) / 128 * 128;  // a warp's result
  static_assert(kBdWarps * kLeft <= kScales, "the warps' results fit the ring");
};

template <int kHeads, int kCh>
__global__ void __launch_bounds__(32 * kBdWarps, BdCfg<kHeads, kCh>::kCtas)
    qsa_block_decode_kernel(const __grid_constant__ BlockDecodeParams p) {
  using C = BdCfg<kHeads, kCh>;
  constexpr int kSets = C::kSets, kStages = C::kStages;
  constexpr int kRowStep = kCh * kHeadDim;  // from a token of a stage to the next
  extern __shared__ __align__(128) uint8_t smem[];
  int* table = reinterpret_cast<int*>(smem + C::kTable);
  float* scales = reinterpret_cast<float*>(smem + C::kScales);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int r = lane / 4, c = lane % 4;
  const uint32_t smem_s = smem_u32(smem);

  const int hgroups = p.virtual_heads / p.cta_heads;
  const int split = kBdWarps / p.cta_heads;  // warps of a head
  const int part = warp / p.cta_heads;       // this warp's share of the tiles
  const int unit = split * kBdTile;          // tokens of a stage; the plan counts in them

  // the CTA's range of the plan's units, and its first row
  int64_t at = 0, end = 1;
  int row = (int)(blockIdx.x / hgroups);
  if (p.plan) {
    const int64_t units = p.plan->units;
    const int ctas = p.plan->ctas;
    if ((int)blockIdx.x >= ctas) return;
    at = blockIdx.x * units / ctas;
    end = (blockIdx.x + 1) * units / ctas;
    row = p.first_row[blockIdx.x];
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
    c0 = from * unit;
    c1 = min((int64_t)to * unit, (int64_t)p.lengths[row]);
    if (from > 0 || to < row_units) slot_out = 2 * blockIdx.x + (from > 0 ? 0 : 1);
    at += to - from;
    if (to == row_units && hg == hgroups - 1) ++row;
  } else {
    c1 = p.counts ? min(__ldg(p.counts + row), p.topk) : p.topk;
    if (req < 0 || req >= p.num_reqs) req = 0, c1 = 0;
    at = end;
  }
  const int gv = hg * p.cta_heads + warp % p.cta_heads;             // (virtual) KV head
  const int g = gv / p.head_parts;                                  // cache head
  const int h0 = g * p.group + (gv % p.head_parts) * p.part_heads;  // first query head
  const int heads = min(p.part_heads, (g + 1) * p.group - h0);

  // Q fragments: f16 of q 2^e for head r, the order of dims is that of the K
  // fragments (k-step s: word s of the thread's chunks c and c + 4)
  uint32_t qf[kSets][8][2];
  float qs[kSets][2];  // of heads 2c, 2c + 1: 2^-e softmax_scale log2(e)
#pragma unroll
  for (int u = 0; u < kSets; ++u) {
    uint4 w[4] = {};
    if (u * 8 + r < heads) {
      const uint4* src = reinterpret_cast<const uint4*>(p.q + ((int64_t)row_now * p.num_q_heads + h0 + u * 8 + r) * kHeadDim);
      w[0] = src[2 * c], w[1] = src[2 * c + 1], w[2] = src[8 + 2 * c], w[3] = src[8 + 2 * c + 1];
    }
    float top = 0.f;
    float2 x[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t b[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
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
    for (int s = 0; s < 8; ++s) {
      qf[u][s][0] = pack_f16(x[2 * s].x * up, x[2 * s].y * up);
      qf[u][s][1] = pack_f16(x[2 * s + 1].x * up, x[2 * s + 1].y * up);
    }
  }

  float o[kSets][8][4];  // [head set][dims 16r + 2i, + 1][head 2c, 2c + 1 of either dim]
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
  // others). Row (token, head) lies at token * kCh + head; a token's chunks are
  // stored permuted, K's by (t & 1) << 2, V's by t & 6, so that the 8 threads
  // of a 16-byte read phase meet no bank twice.
  const int warp_rows = kBdTile / p.head_parts;  // of the stage's rows
  const int row0 = warp * warp_rows + lane / 8;
  const int g0 = hg * p.cta_heads / p.head_parts;  // the CTA's first cache head
  const int token_bytes = p.num_kv_heads * kHeadDim;
  const uint8_t* k_src = p.k + (g0 + row0 % kCh) * kHeadDim + lane % 8 * 16;
  const uint8_t* v_src = p.v + (g0 + row0 % kCh) * kHeadDim + lane % 8 * 16;
  const int scale_row = tid % kBdRows;
  const float* s_src = (tid < kBdRows ? p.k_scales : p.v_scales) + g0 + scale_row % kCh;
  const int token0 = row0 / kCh;
  const uint32_t k_dst = smem_s + row0 * kHeadDim + ((lane % 8 ^ ((token0 & 1) << 2)) << 4);
  const uint32_t v_dst = smem_s + (kBdRows + row0) * kHeadDim + ((lane % 8 ^ (token0 & 6)) << 4);
  const uint32_t s_dst = smem_s + C::kScales + tid * 4;
  // where this warp's fragments lie in a stage
  const uint32_t own = (part * kBdTile * kCh + (warp % p.cta_heads) / p.head_parts) * kHeadDim;
  const uint32_t k_at = own + r * kRowStep + ((c ^ ((r & 1) << 2)) << 4);
  const uint32_t v_at = own + kBdRows * kHeadDim + 2 * c * kRowStep + ((r ^ (2 * c)) << 4);
  const uint32_t s_at = part * kBdTile * kCh + (warp % p.cta_heads) / p.head_parts;

  for (int base = c0; base < c1; base += kBdTable) {
    const int n = min(kBdTable, c1 - base);
    if (base > c0 || !first) __syncthreads();  // the table's readers are done
    bool valid = true;
    // several columns a thread at once: an index, then its page, wait on memory
#pragma unroll 1
    for (int i0 = tid; i0 < (n + unit - 1) / unit * unit; i0 += 4 * C::kThreads) {
      int slot[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int col = i0 + i * C::kThreads;
        slot[i] = col < n ? (p.indices ? __ldg(p.indices + (int64_t)row_now * p.indices_stride + base + col) : base + col) : -1;
      }
      column_slots(p, req, slot);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int col = i0 + i * C::kThreads;
        if (col < (n + unit - 1) / unit * unit) table[col] = slot[i];
        valid = valid && (slot[i] >= 0 || col >= n);
      }
    }
    const bool clean = __syncthreads_and(valid);  // only the last tile may have masked places
    const int tiles = (n + unit - 1) / unit;
    const int whole = clean ? n / unit : 0;  // leading tiles without a masked place

    auto fetch = [&](int k, int st) {
      if (k < tiles) {
        const int* ahead = table + k * unit;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (i >= 2 && p.head_parts == 2) break;
          // Row row0 + 4i: with 8 heads the token's other four or the next
          // token's first, else the same heads 4 / kCh tokens on. The bits that
          // step adds to the token are none that token0 has, so the chunk
          // permutation splits into token0's and a constant.
          const int step = 4 * i / kCh;
          const int64_t at = kCh == 8 ? i % 2 * 4 * kHeadDim : 0;
          const int slot = ahead[token0 + step];
          const uint32_t kd = (k_dst ^ ((step & 1) << 6)) + st * kStageBytes + i * 4 * kHeadDim;
          const uint32_t vd = (v_dst ^ ((step & 6) << 4)) + st * kStageBytes + i * 4 * kHeadDim;
          if (k < whole) {
            cp_async_16_all(kd, k_src + (int64_t)slot * token_bytes + at);
            cp_async_16_all(vd, v_src + (int64_t)slot * token_bytes + at);
          } else {  // masked places read as zeros, whatever the cache holds
            const int64_t from = (int64_t)max(slot, 0) * token_bytes + at;
            cp_async_16(kd, k_src + from, slot < 0 ? 0u : 16u);
            cp_async_16(vd, v_src + from, slot < 0 ? 0u : 16u);
          }
        }
        if (scale_row < unit * kCh) {
          const int slot = ahead[scale_row / kCh];
          const uint32_t block = __umulhi(2u * (uint32_t)max(slot, 0), p.block_mul) >> p.block_shift;
          cp_async_4_or_zero(s_dst + st * 2 * kBdRows * 4, s_src + (int64_t)(int)block * p.num_kv_heads,
                             slot < 0 ? 0u : 4u);
        }
      }
      cp_async_commit();
    };
#pragma unroll
    for (int st = 0; st < kStages - 1; ++st) fetch(st, st);

#pragma unroll 1
    for (int k0 = 0; k0 < tiles; k0 += kStages) {
#pragma unroll
      for (int st = 0; st < kStages; ++st) {
        if (k0 + st >= tiles) break;
        cp_async_wait<kStages - 2>();
        __syncthreads();  // the tile is there, and every warp has read the one before
        fetch(k0 + st + kStages - 1, (st + kStages - 1) % kStages);
        const uint8_t* stage = smem + st * kStageBytes;
        const float* sc = scales + st * 2 * kBdRows + s_at;

        // [head set][token r: heads 2c, 2c+1; token r + 8: the same], in two chains
        float s[kSets][4] = {}, s1[kSets][4] = {};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint4 a4 = *reinterpret_cast<const uint4*>(stage + (k_at ^ (64 * j)));
          const uint4 b4 = *reinterpret_cast<const uint4*>(stage + (k_at ^ (64 * j)) + 8 * kRowStep);
          const uint32_t wa[4] = {a4.x, a4.y, a4.z, a4.w}, wb[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t a[4] = {f16_of(wa[i]), f16_of(wb[i]), f16_of(wa[i] >> 16), f16_of(wb[i] >> 16)};
#pragma unroll
            for (int u = 0; u < kSets; ++u) mma16816(j ? s1[u] : s[u], a, qf[u][4 * j + i][0], qf[u][4 * j + i][1]);
          }
        }
#pragma unroll
        for (int u = 0; u < kSets; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[u][j] += s1[u][j];
        const float ks[2] = {sc[r * kCh], sc[(8 + r) * kCh]};
        const float vs[2] = {sc[kBdRows + r * kCh], sc[kBdRows + (8 + r) * kCh]};
        bool masked[2] = {false, false};
        if (k0 + st >= whole) {
          const int* slots = table + (k0 + st) * unit + part * kBdTile;
          masked[0] = slots[r] < 0, masked[1] = slots[8 + r] < 0;
        }

        // scores over the reference, probabilities, weights over theirs
        float pr[kSets][4], w[kSets][4];
        bool pass = false;
#pragma unroll
        for (int u = 0; u < kSets; ++u) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int t = j / 2, h = j % 2;
            float x = fmaf(s[u][j], ks[t] * qs[u][h], -m[u][h]);
            x = masked[t] ? -INFINITY : x;
            pr[u][j] = ex2(x);
            w[u][j] = pr[u][j] * (vs[t] * inv_w[u][h]);
            pass = pass || x > kLazy || fabsf(w[u][j]) > kLazyW * kOneW;
          }
        }
        if (__any_sync(0xffffffffu, pass)) {
          // move the references, and what was summed against them
#pragma unroll
          for (int u = 0; u < kSets; ++u) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float x0 = masked[0] ? -INFINITY : s[u][h] * (ks[0] * qs[u][h]);
              const float x1 = masked[1] ? -INFINITY : s[u][2 + h] * (ks[1] * qs[u][h]);
              float top = fmaxf(x0, x1);
#pragma unroll
              for (int d = 4; d <= 16; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
              const float m_new = fmaxf(m[u][h], top);
              const float alpha = ex2(m[u][h] - m_new);
              pr[u][h] = ex2(x0 - m_new), pr[u][2 + h] = ex2(x1 - m_new);
              const float w0 = pr[u][h] * vs[0], w1 = pr[u][2 + h] * vs[1];
              float w_top = fmaxf(fabsf(w0), fabsf(w1));
#pragma unroll
              for (int d = 4; d <= 16; d *= 2) w_top = fmaxf(w_top, __shfl_xor_sync(0xffffffffu, w_top, d));
              const float was = W[u][h] * alpha;
              W[u][h] = fmaxf(was, w_top);
              // without a weight yet, any that matters passes
              inv_w[u][h] = W[u][h] > 0.f ? kOneW / W[u][h] : 1e38f;
              const float f = was > 0.f ? was / W[u][h] : 0.f;
              m[u][h] = m_new;
              l[u][h] *= alpha;
              w[u][h] = w0 * inv_w[u][h], w[u][2 + h] = w1 * inv_w[u][h];
#pragma unroll
              for (int i = 0; i < 8; ++i) o[u][i][h] *= f, o[u][i][2 + h] *= f;
            }
          }
        }
        uint32_t pf[kSets][2];
#pragma unroll
        for (int u = 0; u < kSets; ++u) {
          l[u][0] += pr[u][0] + pr[u][2];
          l[u][1] += pr[u][1] + pr[u][3];
          pf[u][0] = transpose8x8(pack_f16(w[u][0], w[u][1]));
          pf[u][1] = transpose8x8(pack_f16(w[u][2], w[u][3]));
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
  if (split > 1) {
    // the warps of a head join in shared memory: each leaves its result, part
    // 0 gathers (m and l by head, values by head and dim)
    __syncthreads();
    float* left = reinterpret_cast<float*>(smem + warp * C::kLeft);  // [kHeads][2], then [kHeads][128]
#pragma unroll
    for (int u = 0; u < kSets; ++u) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int hh = u * 8 + 2 * c + h;
        if (r == 0) left[2 * hh] = m[u][h], left[2 * hh + 1] = l[u][h];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          *reinterpret_cast<float2*>(left + 2 * kHeads + hh * kHeadDim + 16 * r + 2 * i) =
              make_float2(o[u][i][h] * W[u][h], o[u][i][2 + h] * W[u][h]);
      }
    }
    __syncthreads();
    if (part > 0) continue;  // the next table's barrier holds until part 0 has read
#pragma unroll
    for (int u = 0; u < kSets; ++u) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int hh = u * 8 + 2 * c + h;
        float sum = 0.f, top = kLowest;
        for (int w = 0; w < split; ++w)
          top = fmaxf(top, reinterpret_cast<const float*>(smem + (warp + w * p.cta_heads) * C::kLeft)[2 * hh]);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[u][i][h] = o[u][i][2 + h] = 0.f;
        for (int w = 0; w < split; ++w) {
          const float* from = reinterpret_cast<const float*>(smem + (warp + w * p.cta_heads) * C::kLeft);
          const float f = ex2(from[2 * hh] - top);
          sum = fmaf(from[2 * hh + 1], f, sum);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 v = *reinterpret_cast<const float2*>(from + 2 * kHeads + hh * kHeadDim + 16 * r + 2 * i);
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
      const int64_t hr = (int64_t)row_now * p.num_q_heads + h0 + hh;
      if (slot_out >= 0) {
        const int64_t to = ((int64_t)slot_out * p.cta_heads + warp) * p.part_heads + hh;
        float4* dst = reinterpret_cast<float4*>(p.part_o + to * kHeadDim + 16 * r);
#pragma unroll
        for (int i = 0; i < 4; ++i) dst[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
        if (r == 0) p.part_lse[to] = l[u][h] == 0.f ? -INFINITY : m[u][h] + log2f(l[u][h]);
        continue;
      }
      if (p.gate) {
        const uint4* src = reinterpret_cast<const uint4*>(p.gate + hr * kHeadDim + 16 * r);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint4 w4 = src[i];
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
  }  // segments
}

// Valid length of each row for the plan: its count, or the place past its last
// index that is not negative. A CTA a row, from the row's end.
constexpr int kLenThreads = 256;
__global__ void __launch_bounds__(kLenThreads) qsa_block_lengths_kernel(const __grid_constant__ BlockDecodeParams p) {
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
constexpr int kPlanUnits = 8;  // units a CTA gets at least, so that small work has few pieces
__global__ void __launch_bounds__(kPlanThreads) qsa_block_plan_kernel(const __grid_constant__ BlockDecodeParams p, int max_ctas) {
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
  const int ctas = (int)min((int64_t)max_ctas, (units + kPlanUnits - 1) / kPlanUnits);
  int64_t before = run - mine + (t >= 32 ? sums[t / 32 - 1] : 0);
  if (t == 0) p.plan->units = units, p.plan->ctas = ctas, p.prefix[0] = 0;
  for (int r = r0; r < r1; ++r) {
    const int64_t n = max(1, (int)(((int64_t)p.lengths[r] + unit - 1) / unit));
    // CTAs whose first unit, b units / ctas, lies in this row
    const int64_t lo = before * hgroups, hi = (before + n) * hgroups;
    for (int64_t b = (lo * ctas + units - 1) / units; b < ctas && b * units / ctas < hi; ++b)
      if (b * units / ctas >= lo) p.first_row[b] = r;
    before += n;
    p.prefix[r + 1] = before;
  }
}

// Joins the pieces of one (row, query head) a warp, in the plan's order; a row
// that one CTA took whole is done.
__global__ void __launch_bounds__(256) qsa_block_join_kernel(const __grid_constant__ BlockDecodeParams p) {
  const int lane = threadIdx.x % 32;
  const int64_t hr = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  if (hr >= (int64_t)p.rows * p.num_q_heads) return;
  const int row = (int)(hr / p.num_q_heads), h = (int)(hr % p.num_q_heads);
  const int in_group = h % p.group;
  const int gv = h / p.group * p.head_parts + in_group / p.part_heads;
  const int hgroups = p.virtual_heads / p.cta_heads;
  const int64_t units = p.plan->units, ctas = p.plan->ctas;
  const int64_t n = p.prefix[row + 1] - p.prefix[row];
  const int64_t x0 = p.prefix[row] * hgroups + gv / p.cta_heads * n;
  // unit x is CTA b's where b units / ctas <= x < (b + 1) units / ctas
  const int b0 = (int)(((x0 + 1) * ctas - 1) / units), b1 = (int)(((x0 + n) * ctas - 1) / units);
  if (b0 == b1) return;
  auto piece = [&](int b) -> int64_t {  // the first piece is its CTA's second kind
    return ((int64_t)(2 * b + (b == b0 ? 1 : 0)) * p.cta_heads + gv % p.cta_heads) * p.part_heads + in_group % p.part_heads;
  };
  float top = -INFINITY;
  for (int b = b0 + lane; b <= b1; b += 32) top = fmaxf(top, p.part_lse[piece(b)]);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
#pragma unroll 4
  for (int b = b0; b <= b1; ++b) {
    const int64_t from = piece(b);
    const float lse = p.part_lse[from];
    const float4 v = *reinterpret_cast<const float4*>(p.part_o + from * kHeadDim + lane * 4);
    const float w = lse == -INFINITY ? 0.f : exp2f(lse - top);
    sum += w;
    acc[0] = fmaf(w, v.x, acc[0]), acc[1] = fmaf(w, v.y, acc[1]);
    acc[2] = fmaf(w, v.z, acc[2]), acc[3] = fmaf(w, v.w, acc[3]);
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  const int64_t off = hr * kHeadDim + lane * 4;
#pragma unroll
  for (int d = 0; d < 4; ++d) acc[d] *= inv * (p.gate ? sigmoid(__bfloat162float(p.gate[off + d])) : 1.f);
  const __nv_bfloat162 a = __floats2bfloat162_rn(acc[0], acc[1]), b = __floats2bfloat162_rn(acc[2], acc[3]);
  *reinterpret_cast<uint2*>(p.out + off) =
      make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
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
int planned_ctas(const BlockDecodeParams& p) { return sm_count() * (p.part_heads > 8 ? BdCfg<16, 1>::kCtas : BdCfg<8, 1>::kCtas); }

template <int kHeads, int kCh>
cudaError_t launch(const BlockDecodeParams& p, cudaStream_t stream) {
  using C = BdCfg<kHeads, kCh>;
  // the shared memory beyond the default limit, once per device
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(ready.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(qsa_block_decode_kernel<kHeads, kCh>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return e;
    ready.fetch_or(bit, std::memory_order_acq_rel);
  }
  const int64_t grid = p.plan ? planned_ctas(p) : (int64_t)p.rows * (p.virtual_heads / p.cta_heads);
  if (grid > 0x7fffffffll) return cudaErrorInvalidValue;
  qsa_block_decode_kernel<kHeads, kCh><<<(unsigned)grid, C::kThreads, C::kSmem, stream>>>(p);
  return cudaGetLastError();
}

template <int kHeads>
cudaError_t launch(const BlockDecodeParams& p, cudaStream_t stream) {
  switch (p.cta_heads / p.head_parts) {
    case 1: return launch<kHeads, 1>(p, stream);
    case 2: return launch<kHeads, 2>(p, stream);
    case 4: return launch<kHeads, 4>(p, stream);
    default: return launch<kHeads, 8>(p, stream);
  }
}

}  // namespace

int64_t block_decode_plan(BlockDecodeParams& p) {
  // a group above 16 goes as two virtual KV heads
  p.head_parts = p.group > 16 ? 2 : 1;
  p.part_heads = (p.group + p.head_parts - 1) / p.head_parts;
  p.virtual_heads = p.num_kv_heads * p.head_parts;
  p.cta_heads = 1;
  while (p.cta_heads < 8 && p.virtual_heads % (2 * p.cta_heads) == 0) p.cta_heads *= 2;
  // mul = ceil(2^(31 + shift) / block) with block <= 2^shift: n mul exceeds
  // n 2^(31 + shift) / block by less than n, so n / block is exact for n < 2^31
  uint32_t shift = 0;
  while ((1ll << shift) < p.block_size) ++shift;
  p.block_shift = shift;
  p.block_mul = (uint32_t)((((uint64_t)1 << (31 + shift)) + p.block_size - 1) / p.block_size);
  p.planned = p.topk > kBdDirect;
  if (!p.planned) return 0;
  const int64_t pieces = 2ll * planned_ctas(p) * p.cta_heads * p.part_heads;
  return align256(pieces * kHeadDim * 4) + align256(pieces * 4) + align256((int64_t)sizeof(BlockDecodePlan)) +
         align256(8ll * (p.rows + 1)) + align256(4ll * p.rows) + align256(4ll * planned_ctas(p));
}

void block_decode_place(BlockDecodeParams& p, void* workspace) {
  char* at = static_cast<char*>(workspace);
  const int64_t pieces = 2ll * planned_ctas(p) * p.cta_heads * p.part_heads;
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
  p.first_row = reinterpret_cast<int*>(take(4ll * planned_ctas(p)));
}

cudaError_t launch_block_decode(const BlockDecodeParams& p, cudaStream_t stream) {
  if (p.plan) {
    if (p.indices) qsa_block_lengths_kernel<<<p.rows, kLenThreads, 0, stream>>>(p);
    qsa_block_plan_kernel<<<1, kPlanThreads, 0, stream>>>(p, planned_ctas(p));
  }
  cudaError_t e = p.part_heads > 8 ? launch<16>(p, stream) : launch<8>(p, stream);
  if (e != cudaSuccess || !p.plan) return e;
  const int64_t warps = (int64_t)p.rows * p.num_q_heads;
  qsa_block_join_kernel<<<(unsigned)((warps + 7) / 8), 256, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace qsa
