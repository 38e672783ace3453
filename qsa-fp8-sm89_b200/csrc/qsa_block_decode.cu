// Attention over the block-scaled caches.
//
//   out[r,h] = softmax_t(q . K[t] ks[t] scale) . V[t] vs[t]  (*) sigmoid(gate)
//
// A CTA of 8 warps takes a range of one row's columns for up to 8 KV heads: it
// first turns its columns into physical slots (a table in shared memory), then
// every warp streams on its own, without CTA barriers: 16 tokens at a time of
// one KV head, K and V rows brought by cp.async into a ring of the warp. With
// fewer than 8 heads several warps share a head, every n-th tile each, and
// join their results in shared memory. The 8 heads' rows of a token, 1 KiB in
// a row, are so fetched at about the same time.
//
// The bytes bound it: 256 per token and head for 4 x 128 x group flops, so
// the tensor work is small against the rate that mma.sync reaches (a tile of
// 16 tokens is 24 or 32 instructions), while its register fragments let the
// codes go from shared memory through one conversion (E4M3 -> f16, exact) into
// the product, with no operand written back to shared memory:
//   S = Q K^T    m16n8k16: 16 query heads, 8 tokens. A thread's fragments of K
//                are 32 of a row's 128 bytes; the order of the dims in the
//                product is theirs, and Q's fragments follow it.
//   O^T = V^T P^T  16 dims, 8 heads, 16 tokens. S's accumulator layout is P's
//                operand layout. A thread's V fragments are 16 bytes of four
//                tokens, interleaved by byte permutes.
// Queries are scaled by a power of two to below 2^15 and held in f16: exact
// for a bf16 element down to 2^-28 of the head's largest. A probability times
// its token's V scale is rounded to f16 (2^-11), relative to a running
// reference W: the reference is held as 2^11 in f16's range, so a weight keeps
// its 11 bits down to 2^-25 W and is off by 2^-36 W at most below that. Sums,
// maxima and accumulators are fp32.
//
// Softmax with lazy references: scores are taken against a reference m that
// moves only when one passes it by 8, weights p vs against a reference W that
// moves when one passes 16 W (2^15 in f16), so that scales may spread over any
// range. The usual tile needs one vote and no reduction.
#include <atomic>

#include "qsa_common.cuh"

namespace qsa {
namespace {

constexpr int kBdWarps = 8;
constexpr int kBdTile = 16;                         // tokens a warp takes at a time
constexpr int kBdTable = 2048;                      // slots of a CTA's table
constexpr int kStageBytes = 2 * kBdTile * kHeadDim;  // K and V of a tile
constexpr float kLazy = 8.f;                        // log2 by which a score may pass its reference
constexpr float kLazyW = 16.f;                      // factor by which a weight may pass its reference
constexpr float kOneW = 2048.f;                     // what stands for W in f16
constexpr float kLowest = -3.402823466e38f;

__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + expf(-x)); }
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ void cp_async_4_or_zero(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two E4M3 codes (the low or high half of a word) as f16, exactly.
__device__ __forceinline__ uint32_t f16_of_lo(uint32_t w) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
  return (uint32_t)h.x | ((uint32_t)h.y << 16);
}
__device__ __forceinline__ uint32_t f16_of_hi(uint32_t w) { return f16_of_lo(w >> 16); }

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Physical slot of column `col` of a row, -1 where it is masked.
__device__ __forceinline__ int column_slot(const BlockDecodeParams& p, int row, int64_t req, int col) {
  const int t = p.indices ? __ldg(p.indices + (int64_t)row * p.indices_stride + col) : col;
  if (t < 0) return -1;
  const int lp = t / p.page_size;
  if (lp >= p.pages_per_req) return -1;
  const int page = __ldg(p.btable + req * p.btable_stride + lp);
  return page < 0 || page >= p.num_pages ? -1 : page * p.page_size + (t - lp * p.page_size);
}

// kHeads: query heads of a warp's tile, 8 or 16. kStages: tiles in flight.
template <int kHeads>
struct BdCfg {
  static constexpr int kSets = kHeads / 8;
  static constexpr int kStages = kHeads == 8 ? 3 : 6;
  static constexpr int kCtas = kHeads == 8 ? 2 : 1;  // per SM
  static constexpr int kRing = kStages * kStageBytes;
  static constexpr int kScales = kBdWarps * kRing;                              // float [warps][stages][32]
  static constexpr int kTable = kScales + kBdWarps * kStages * 32 * 4;          // int [kBdTable]
  static constexpr int kSmem = kTable + kBdTable * 4;
  static_assert(kHeads * (kHeadDim + 2) * 4 <= kRing, "a warp's result fits its ring");
};

template <int kHeads>
__global__ void __launch_bounds__(32 * kBdWarps, BdCfg<kHeads>::kCtas)
    qsa_block_decode_kernel(const __grid_constant__ BlockDecodeParams p) {
  using C = BdCfg<kHeads>;
  constexpr int kSets = C::kSets, kStages = C::kStages;
  extern __shared__ __align__(128) uint8_t smem[];
  int* table = reinterpret_cast<int*>(smem + C::kTable);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int r = lane / 4, c = lane % 4;
  uint8_t* ring = smem + warp * C::kRing;
  const uint32_t ring_s = smem_u32(ring);
  float* scales = reinterpret_cast<float*>(smem + C::kScales) + warp * kStages * 32;
  const uint32_t scales_s = smem_u32(scales);

  // this warp's (virtual) KV head and its share of the tiles
  const int hgroups = p.virtual_heads / p.cta_heads;
  const int row = blockIdx.x / hgroups;
  const int split = kBdWarps / p.cta_heads;
  const int gv = (blockIdx.x % hgroups) * p.cta_heads + warp % p.cta_heads;
  const int part = warp / p.cta_heads;
  const int g = gv / p.head_parts;                                  // cache head
  const int h0 = g * p.group + (gv % p.head_parts) * p.part_heads;  // first query head
  const int heads = min(p.part_heads, (g + 1) * p.group - h0);

  int64_t req = p.t2r ? __ldg(p.t2r + row) : row;
  int count = p.counts ? min(__ldg(p.counts + row), p.topk) : p.topk;
  if (req < 0 || req >= p.num_reqs) req = 0, count = 0;
  const int c0 = blockIdx.y * p.chunk_tokens;
  const int c1 = (int)min((int64_t)c0 + p.chunk_tokens, (int64_t)count);

  // Q fragments: f16 of q 2^e, the order of dims is that of the K fragments
  // (k-step s: bytes 4s .. 4s+3 of the thread's chunks c and c + 4)
  uint32_t qf[8][4];
  float qs[kSets];  // of head r (and r + 8): 2^-e softmax_scale log2(e)
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const bool in = u < kSets && u * 8 + r < heads;
    uint4 w[4] = {};
    if (in) {
      const uint4* src = reinterpret_cast<const uint4*>(p.q + ((int64_t)row * p.num_q_heads + h0 + u * 8 + r) * kHeadDim);
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
    if (top > 0.f && top <= 3.0e38f) e = min(max(14 + 127 - (int)(__float_as_uint(top) >> 23), -120), 120);
    const float up = __uint_as_float((uint32_t)(127 + e) << 23);
    if (u < kSets) qs[u] = __uint_as_float((uint32_t)(127 - e) << 23) * p.score_scale_log2;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      qf[s][u] = pack_f16(x[2 * s].x * up, x[2 * s].y * up);
      qf[s][2 + u] = pack_f16(x[2 * s + 1].x * up, x[2 * s + 1].y * up);
    }
  }

  float o[kSets][8][4];  // [head set][dims 16r + 2i, + 1][head 2c, 2c + 1 of either dim]
  float m[kSets], l[kSets], W[kSets], inv_w[kSets];
#pragma unroll
  for (int u = 0; u < kSets; ++u) {
    m[u] = kLowest, l[u] = 0.f, W[u] = 0.f, inv_w[u] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[u][i][j] = 0.f;
  }

  const int64_t token_bytes = (int64_t)p.num_kv_heads * kHeadDim;
  for (int base = c0; base < c1; base += kBdTable) {
    const int n = min(kBdTable, c1 - base);
    if (base > c0) __syncthreads();  // the table's readers are done
    for (int i = tid; i < (n + kBdTile - 1) / kBdTile * kBdTile; i += 32 * kBdWarps)
      table[i] = i < n ? column_slot(p, row, req, base + i) : -1;
    __syncthreads();
    const int tiles = (n + kBdTile - 1) / kBdTile;
    const int mine = tiles > part ? (tiles - part + split - 1) / split : 0;

    // tile k of this warp into its ring slot: lane l copies 16 bytes of rows
    // l/8, 4 + l/8, ...; scales of K by lanes 0-15, of V by lanes 16-31
    auto fetch = [&](int k) {
      if (k < mine) {
        const int* slots = table + (part + k * split) * kBdTile;
        const int st = k % kStages;
        const uint32_t dst = ring_s + st * kStageBytes;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int t = i * 4 + lane / 8, chunk = lane % 8;
          const int slot = slots[t];
          const int64_t off = slot < 0 ? 0 : slot * token_bytes + g * kHeadDim + chunk * 16;
          const uint32_t bytes = slot < 0 ? 0u : 16u;
          cp_async_16(dst + t * kHeadDim + ((chunk ^ ((t & 1) << 2)) << 4), p.k + off, bytes);
          cp_async_16(dst + (kBdTile + t) * kHeadDim + ((chunk ^ (t & 6)) << 4), p.v + off, bytes);
        }
        const int slot = slots[lane % 16];
        const int64_t at = slot < 0 ? 0 : (int64_t)(__umulhi(2u * (uint32_t)slot, p.block_mul) >> p.block_shift) * p.num_kv_heads + g;
        cp_async_4_or_zero(scales_s + (st * 32 + lane) * 4, (lane < 16 ? p.k_scales : p.v_scales) + at, slot < 0 ? 0u : 4u);
      }
      cp_async_commit();
    };
#pragma unroll
    for (int k = 0; k < kStages; ++k) fetch(k);

#pragma unroll 1
    for (int k = 0; k < mine; ++k) {
      cp_async_wait<kStages - 1>();
      __syncwarp();
      const int st = k % kStages;
      const uint8_t* kt = ring + st * kStageBytes;
      const uint8_t* vt = kt + kBdTile * kHeadDim;
      const float* sc = scales + st * 32;
      const int* slots = table + (part + k * split) * kBdTile;

      float s[2][4];  // [tokens 2c, 2c+1 / 8+2c, 9+2c][head r: 0, 1; head r + 8: 2, 3]
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint8_t* krow = kt + (j * 8 + r) * kHeadDim;
        const uint4 w0 = *reinterpret_cast<const uint4*>(krow + ((c ^ ((r & 1) << 2)) << 4));
        const uint4 w1 = *reinterpret_cast<const uint4*>(krow + (((c + 4) ^ ((r & 1) << 2)) << 4));
        const uint32_t w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
        s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) mma16816(s[j], qf[i], f16_of_lo(w[i]), f16_of_hi(w[i]));
      }
      const float2 ks[2] = {*reinterpret_cast<const float2*>(sc + 2 * c), *reinterpret_cast<const float2*>(sc + 8 + 2 * c)};
      const float2 vs[2] = {*reinterpret_cast<const float2*>(sc + 16 + 2 * c), *reinterpret_cast<const float2*>(sc + 24 + 2 * c)};
      const int2 sl[2] = {*reinterpret_cast<const int2*>(slots + 2 * c), *reinterpret_cast<const int2*>(slots + 8 + 2 * c)};

      float x[kSets][4], pr[kSets][4], w[kSets][4];  // scores, probabilities, weights of tokens 2c, 2c+1, 8+2c, 9+2c
      bool pass = false;
#pragma unroll
      for (int u = 0; u < kSets; ++u) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          x[u][2 * j] = sl[j].x < 0 ? -INFINITY : s[j][2 * u] * (ks[j].x * qs[u]);
          x[u][2 * j + 1] = sl[j].y < 0 ? -INFINITY : s[j][2 * u + 1] * (ks[j].y * qs[u]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          pr[u][j] = ex2(x[u][j] - m[u]);
          w[u][j] = pr[u][j] * (j % 2 ? vs[j / 2].y : vs[j / 2].x);
          pass = pass || x[u][j] > m[u] + kLazy || fabsf(w[u][j]) > W[u] * kLazyW;
        }
      }
      if (__any_sync(0xffffffffu, pass)) {
        // move the references, and what was summed against them
#pragma unroll
        for (int u = 0; u < kSets; ++u) {
          float top = fmaxf(fmaxf(x[u][0], x[u][1]), fmaxf(x[u][2], x[u][3]));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const float m_new = fmaxf(m[u], top);
          const float alpha = ex2(m[u] - m_new);
          float w_top = 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            pr[u][j] = ex2(x[u][j] - m_new);
            w[u][j] = pr[u][j] * (j % 2 ? vs[j / 2].y : vs[j / 2].x);
            w_top = fmaxf(w_top, fabsf(w[u][j]));
          }
          w_top = fmaxf(w_top, __shfl_xor_sync(0xffffffffu, w_top, 1));
          w_top = fmaxf(w_top, __shfl_xor_sync(0xffffffffu, w_top, 2));
          const float was = W[u] * alpha;
          W[u] = fmaxf(was, w_top);
          inv_w[u] = W[u] > 0.f ? kOneW / W[u] : 0.f;
          const float f = was > 0.f ? was / W[u] : 0.f;
          m[u] = m_new;
          l[u] *= alpha;
          // head r's factor is on lanes 4r .. 4r+3
          const float f0 = __shfl_sync(0xffffffffu, f, 8 * c), f1 = __shfl_sync(0xffffffffu, f, 8 * c + 4);
#pragma unroll
          for (int i = 0; i < 8; ++i) o[u][i][0] *= f0, o[u][i][1] *= f1, o[u][i][2] *= f0, o[u][i][3] *= f1;
        }
      }
      uint32_t pf[kSets][2];
#pragma unroll
      for (int u = 0; u < kSets; ++u) {
        l[u] += (pr[u][0] + pr[u][1]) + (pr[u][2] + pr[u][3]);
        pf[u][0] = pack_f16(w[u][0] * inv_w[u], w[u][1] * inv_w[u]);
        pf[u][1] = pack_f16(w[u][2] * inv_w[u], w[u][3] * inv_w[u]);
      }
      // V: chunk r of tokens 2c, 2c+1, 8+2c, 9+2c
      uint32_t vw[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = (j / 2) * 8 + 2 * c + j % 2;
        const uint4 q4 = *reinterpret_cast<const uint4*>(vt + t * kHeadDim + ((r ^ (t & 6)) << 4));
        vw[j][0] = q4.x, vw[j][1] = q4.y, vw[j][2] = q4.z, vw[j][3] = q4.w;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t sel = i % 2 ? 0x7362 : 0x5140;  // a dim's codes of two tokens side by side
        const uint32_t lo = __byte_perm(vw[0][i / 2], vw[1][i / 2], sel), hi = __byte_perm(vw[2][i / 2], vw[3][i / 2], sel);
        const uint32_t a[4] = {f16_of_lo(lo), f16_of_hi(lo), f16_of_lo(hi), f16_of_hi(hi)};
#pragma unroll
        for (int u = 0; u < kSets; ++u) mma16816(o[u][i], a, pf[u][0], pf[u][1]);
      }
      __syncwarp();  // every lane has read the slot
      fetch(k + kStages);
    }
    cp_async_wait<0>();
  }

  // to heads 2c, 2c + 1: the sums and references
#pragma unroll
  for (int u = 0; u < kSets; ++u) {
    W[u] *= 1.0f / kOneW;
    l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
    l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
  }
  if (split > 1) {
    // the warps of a head join in shared memory: each leaves its result, part
    // 0 gathers (m and l by head, values by head and dim)
    __syncthreads();
    float* left = reinterpret_cast<float*>(ring);  // [kHeads][2], then [kHeads][128]
#pragma unroll
    for (int u = 0; u < kSets; ++u) {
      if (c == 0) left[2 * (u * 8 + r)] = m[u], left[2 * (u * 8 + r) + 1] = l[u];
      const float W0 = __shfl_sync(0xffffffffu, W[u], 8 * c), W1 = __shfl_sync(0xffffffffu, W[u], 8 * c + 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float* at = left + 2 * kHeads + (u * 8 + 2 * c) * kHeadDim + 16 * r + 2 * i;
        *reinterpret_cast<float2*>(at) = make_float2(o[u][i][0] * W0, o[u][i][2] * W0);
        *reinterpret_cast<float2*>(at + kHeadDim) = make_float2(o[u][i][1] * W1, o[u][i][3] * W1);
      }
    }
    __syncthreads();
    if (part > 0) return;
#pragma unroll
    for (int u = 0; u < kSets; ++u) {
      float sum = 0.f, top = kLowest;
      for (int w = 0; w < split; ++w)
        top = fmaxf(top, reinterpret_cast<const float*>(smem + (warp + w * p.cta_heads) * C::kRing)[2 * (u * 8 + r)]);
      const float top0 = __shfl_sync(0xffffffffu, top, 8 * c), top1 = __shfl_sync(0xffffffffu, top, 8 * c + 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) o[u][i][0] = o[u][i][1] = o[u][i][2] = o[u][i][3] = 0.f;
      for (int w = 0; w < split; ++w) {
        const float* from = reinterpret_cast<const float*>(smem + (warp + w * p.cta_heads) * C::kRing);
        sum += from[2 * (u * 8 + r) + 1] * ex2(from[2 * (u * 8 + r)] - top);
        const float f0 = ex2(from[2 * (u * 8 + 2 * c)] - top0), f1 = ex2(from[2 * (u * 8 + 2 * c + 1)] - top1);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float* at = from + 2 * kHeads + (u * 8 + 2 * c) * kHeadDim + 16 * r + 2 * i;
          const float2 a = *reinterpret_cast<const float2*>(at), b = *reinterpret_cast<const float2*>(at + kHeadDim);
          o[u][i][0] = fmaf(f0, a.x, o[u][i][0]), o[u][i][2] = fmaf(f0, a.y, o[u][i][2]);
          o[u][i][1] = fmaf(f1, b.x, o[u][i][1]), o[u][i][3] = fmaf(f1, b.y, o[u][i][3]);
        }
      }
      m[u] = top, l[u] = sum, W[u] = 1.f;
    }
  }

#pragma unroll
  for (int u = 0; u < kSets; ++u) {
    const float inv = l[u] == 0.f ? 0.f : W[u] / l[u];  // a NaN sum stays one
    const float lse = l[u] == 0.f ? -INFINITY : m[u] + log2f(l[u]);
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const float f = __shfl_sync(0xffffffffu, inv, 8 * c + 4 * side);
      const float head_lse = __shfl_sync(0xffffffffu, lse, 8 * c + 4 * side);
      const int hh = u * 8 + 2 * c + side;
      if (hh >= heads) continue;
      float x[16];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[2 * i] = o[u][i][side] * f, x[2 * i + 1] = o[u][i][2 + side] * f;
      const int64_t hr = (int64_t)row * p.num_q_heads + h0 + hh;
      if (p.num_chunks > 1) {
        const int64_t at = hr * p.num_chunks + blockIdx.y;
        float4* dst = reinterpret_cast<float4*>(p.part_o + at * kHeadDim + 16 * r);
#pragma unroll
        for (int i = 0; i < 4; ++i) dst[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
        if (r == 0) p.part_lse[at] = head_lse;
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
}

// Joins the chunks of one (row, query head) a warp.
__global__ void __launch_bounds__(256) qsa_block_join_kernel(const __grid_constant__ BlockDecodeParams p) {
  const int lane = threadIdx.x % 32;
  const int64_t hr = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  if (hr >= (int64_t)p.rows * p.num_q_heads) return;
  const int64_t base = hr * p.num_chunks;
  float top = -INFINITY;
  for (int c = 0; c < p.num_chunks; ++c) top = fmaxf(top, p.part_lse[base + c]);
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
  for (int c = 0; c < p.num_chunks; ++c) {
    const float lse = p.part_lse[base + c];
    if (lse == -INFINITY) continue;
    const float w = exp2f(lse - top);
    const float4 v = *reinterpret_cast<const float4*>(p.part_o + (base + c) * kHeadDim + lane * 4);
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

template <int kHeads>
cudaError_t launch(const BlockDecodeParams& p, cudaStream_t stream) {
  using C = BdCfg<kHeads>;
  // the shared memory beyond the default limit, once per device
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(ready.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(qsa_block_decode_kernel<kHeads>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return e;
    ready.fetch_or(bit, std::memory_order_acq_rel);
  }
  const dim3 grid((unsigned)(p.rows * (p.virtual_heads / p.cta_heads)), (unsigned)p.num_chunks);
  qsa_block_decode_kernel<kHeads><<<grid, 32 * kBdWarps, C::kSmem, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

int64_t block_decode_plan(BlockDecodeParams& p) {
  // a group above 16 goes as two virtual KV heads
  p.head_parts = p.group > 16 ? 2 : 1;
  p.part_heads = (p.group + p.head_parts - 1) / p.head_parts;
  p.virtual_heads = p.num_kv_heads * p.head_parts;
  p.cta_heads = 1;
  while (p.cta_heads < kBdWarps && p.virtual_heads % (2 * p.cta_heads) == 0) p.cta_heads *= 2;
  // mul = ceil(2^(31 + shift) / block) with block <= 2^shift: n mul exceeds
  // n 2^(31 + shift) / block by less than n, so n / block is exact for n < 2^31
  uint32_t shift = 0;
  while ((1ll << shift) < p.block_size) ++shift;
  p.block_shift = shift;
  p.block_mul = (uint32_t)((((uint64_t)1 << (31 + shift)) + p.block_size - 1) / p.block_size);
  const int64_t ctas = (int64_t)p.rows * (p.virtual_heads / p.cta_heads);
  int64_t chunk = ((int64_t)p.topk * ctas / (2 * 148 * 2) + 255) / 256 * 256;
  if (chunk < 256) chunk = 256;
  if (chunk > kBdTable) chunk = kBdTable;
  p.chunk_tokens = (int)chunk;
  p.num_chunks = p.topk <= chunk ? 1 : (int)((p.topk + chunk - 1) / chunk);
  if (p.num_chunks == 1) return 0;
  const int64_t n = (int64_t)p.rows * p.num_q_heads * p.num_chunks;
  return (n * kHeadDim * 4 + 255) / 256 * 256 + (n * 4 + 255) / 256 * 256;
}

cudaError_t launch_block_decode(const BlockDecodeParams& p, cudaStream_t stream) {
  if (p.num_chunks > 65535) return cudaErrorInvalidValue;
  cudaError_t e = p.part_heads <= 8 ? launch<8>(p, stream) : launch<16>(p, stream);
  if (e != cudaSuccess || p.num_chunks == 1) return e;
  const int64_t warps = (int64_t)p.rows * p.num_q_heads;
  qsa_block_join_kernel<<<(unsigned)((warps + 7) / 8), 256, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace qsa
