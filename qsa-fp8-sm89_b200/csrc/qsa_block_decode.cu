// Attention over the block-scaled caches.
//
//   out[r,h] = softmax_t(q . K[t] ks[t] scale) . V[t] vs[t]  (*) sigmoid(gate)
//
// One warp takes a query head over a chunk of the row's columns, 32 tokens at
// a time: lane j finds token j's slot and scales, lane l owns dims 4l .. 4l+3
// of every product, a transposing reduction leaves token j's score on lane j,
// and the softmax keeps a running maximum and sum in fp32. Chunks are joined
// by their log-sums in a second kernel.
#include "qsa_common.cuh"

namespace qsa {
namespace {

constexpr int kBdHeads = 8;  // query heads (warps) of a CTA
constexpr int kBdChunk = 512;

__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + expf(-x)); }

__device__ __forceinline__ void fp8x4(uint32_t w, float (&f)[4]) {
  const float2 lo = e4m3x2_to_f32x2((uint16_t)(w & 0xffffu));
  const float2 hi = e4m3x2_to_f32x2((uint16_t)(w >> 16));
  f[0] = lo.x, f[1] = lo.y, f[2] = hi.x, f[3] = hi.y;
}

__device__ __forceinline__ void bf16x4(const __nv_bfloat16* src, float (&f)[4]) {
  const uint2 raw = *reinterpret_cast<const uint2*>(src);
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.x));
  const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.y));
  f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
}

__device__ __forceinline__ void store_bf16x4(__nv_bfloat16* dst, const float (&f)[4]) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
  *reinterpret_cast<uint2*>(dst) =
      make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// Physical slot of column `col` of a row, -1 where it is masked.
__device__ __forceinline__ int64_t column_slot(const BlockDecodeParams& p, int row, int64_t req, int count, int col) {
  if (req < 0 || col >= count) return -1;
  const int t = p.indices ? __ldg(p.indices + (int64_t)row * p.indices_stride + col) : col;
  if (t < 0) return -1;
  const int lp = t / p.page_size;
  if (lp >= p.pages_per_req) return -1;
  const int64_t page = __ldg(p.btable + req * p.btable_stride + lp);
  return page < 0 || page >= p.num_pages ? -1 : page * p.page_size + (t - lp * p.page_size);
}

__global__ void __launch_bounds__(32 * kBdHeads) qsa_block_decode_kernel(const __grid_constant__ BlockDecodeParams p) {
  const int g = blockIdx.x % p.num_kv_heads;
  const int row = blockIdx.x / p.num_kv_heads;
  const int lane = threadIdx.x % 32;
  const int hg = blockIdx.z * kBdHeads + threadIdx.x / 32;
  if (hg >= p.group) return;
  const int h = g * p.group + hg;
  int64_t req = p.t2r ? __ldg(p.t2r + row) : row;
  if (req < 0 || req >= p.num_reqs) req = -1;
  const int count = p.counts ? min(__ldg(p.counts + row), p.topk) : p.topk;
  const int c0 = blockIdx.y * p.chunk_tokens;
  const int c1 = (int)min((int64_t)c0 + p.chunk_tokens, (int64_t)count);
  const int64_t qoff = ((int64_t)row * p.num_q_heads + h) * kHeadDim + lane * 4;
  float q[4];
  bf16x4(p.q + qoff, q);
  float m = -INFINITY, sum = 0.f;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int base = c0; base < c1; base += 32) {
    const int64_t slot = column_slot(p, row, req, c1, base + lane);
    const bool valid = slot >= 0;
    float ks = 0.f, vs = 0.f;
    if (valid) {
      const int64_t at = slot / p.block_size * p.num_kv_heads + g;
      ks = __ldg(p.k_scales + at) * p.score_scale_log2;
      vs = __ldg(p.v_scales + at);
    }
    const long long off = valid ? (long long)(slot * p.num_kv_heads + g) * kHeadDim : -1ll;
    float part[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const long long o = __shfl_sync(0xffffffffu, off, i);
      part[i] = 0.f;
      if (o >= 0) {
        float f[4];
        fp8x4(__ldg(reinterpret_cast<const uint32_t*>(p.k + o + lane * 4)), f);
        part[i] = q[0] * f[0] + q[1] * f[1] + q[2] * f[2] + q[3] * f[3];
      }
    }
#pragma unroll
    for (int s = 16; s >= 1; s >>= 1) {
      const bool upper = (lane & s) != 0;
#pragma unroll
      for (int k = 0; k < s; ++k) {
        const float send = upper ? part[k] : part[k + s];
        const float keep = upper ? part[k + s] : part[k];
        part[k] = keep + __shfl_xor_sync(0xffffffffu, send, s);
      }
    }
    const float score = valid ? part[0] * ks : -INFINITY;
    float top = score;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (!__any_sync(0xffffffffu, valid)) continue;
    const float m_new = fmaxf(m, top);
    const float ref = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = exp2f(m - ref);
    const float pj = valid ? exp2f(score - ref) : 0.f;
    float s = pj;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    sum = sum * alpha + s;
#pragma unroll
    for (int d = 0; d < 4; ++d) acc[d] *= alpha;
#pragma unroll 8
    for (int i = 0; i < 32; ++i) {
      const long long o = __shfl_sync(0xffffffffu, off, i);
      const float pi = __shfl_sync(0xffffffffu, pj * vs, i);
      if (o >= 0) {
        float f[4];
        fp8x4(__ldg(reinterpret_cast<const uint32_t*>(p.v + o + lane * 4)), f);
#pragma unroll
        for (int d = 0; d < 4; ++d) acc[d] = fmaf(pi, f[d], acc[d]);
      }
    }
    m = m_new;
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;  // a NaN sum stays one
#pragma unroll
  for (int d = 0; d < 4; ++d) acc[d] *= inv;
  if (p.num_chunks == 1) {
    if (p.gate) {
      float gt[4];
      bf16x4(p.gate + qoff, gt);
#pragma unroll
      for (int d = 0; d < 4; ++d) acc[d] *= sigmoid(gt[d]);
    }
    store_bf16x4(p.out + qoff, acc);
  } else {
    const int64_t at = ((int64_t)row * p.num_q_heads + h) * p.num_chunks + blockIdx.y;
    *reinterpret_cast<float4*>(p.part_o + at * kHeadDim + lane * 4) = make_float4(acc[0], acc[1], acc[2], acc[3]);
    if (lane == 0) p.part_lse[at] = sum == 0.f ? -INFINITY : m + log2f(sum);
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
  float gt[4] = {INFINITY, INFINITY, INFINITY, INFINITY};
  if (p.gate) bf16x4(p.gate + off, gt);
#pragma unroll
  for (int d = 0; d < 4; ++d) acc[d] *= inv * (p.gate ? sigmoid(gt[d]) : 1.f);
  store_bf16x4(p.out + off, acc);
}

}  // namespace

int64_t block_decode_plan(BlockDecodeParams& p) {
  p.chunk_tokens = kBdChunk;
  p.num_chunks = p.topk <= kBdChunk ? 1 : (int)(((int64_t)p.topk + kBdChunk - 1) / kBdChunk);
  if (p.num_chunks == 1) return 0;
  const int64_t n = (int64_t)p.rows * p.num_q_heads * p.num_chunks;
  return (n * kHeadDim * 4 + 255) / 256 * 256 + (n * 4 + 255) / 256 * 256;
}

cudaError_t launch_block_decode(const BlockDecodeParams& p, cudaStream_t stream) {
  if (p.num_chunks > 65535) return cudaErrorInvalidValue;
  const dim3 grid((unsigned)(p.rows * p.num_kv_heads), (unsigned)p.num_chunks, (unsigned)((p.group + kBdHeads - 1) / kBdHeads));
  qsa_block_decode_kernel<<<grid, 32 * (p.group < kBdHeads ? p.group : kBdHeads), 0, stream>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || p.num_chunks == 1) return e;
  const int64_t warps = (int64_t)p.rows * p.num_q_heads;
  qsa_block_join_kernel<<<(unsigned)((warps + 7) / 8), 256, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace qsa
