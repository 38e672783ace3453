// Attention in the latent's space over the latent cache (the absorbed form).
//
// A warp takes one query head of one node and goes through its columns, a token
// at a time: lane l holds elements 4l .. 4l+3 of each 128 of the latent and two
// rotated ones. Softmax by a running maximum and sum, all in fp32.
#include "qsa_latent.cuh"

namespace qsa {
namespace {

constexpr int kLdWarps = 4;

template <int kChunks>
__global__ void __launch_bounds__(32 * kLdWarps) qsa_latent_decode_kernel(const __grid_constant__ LatentDecodeParams p) {
  constexpr int kRank = 128 * kChunks;
  const int lane = threadIdx.x % 32;
  const int64_t at = (int64_t)blockIdx.x * kLdWarps + threadIdx.x / 32;  // (row, node, head)
  if (at >= (int64_t)p.rows * p.nodes * p.heads) return;
  const int row = (int)(at / (p.nodes * p.heads));
  const int node = (int)(at / p.heads) % p.nodes;
  const __nv_bfloat16* q = p.q + at * (kRank + kLatentRope);
  float x[kChunks][4], o[kChunks][4] = {};
#pragma unroll
  for (int i = 0; i < kChunks; ++i) latent_load4(q + 128 * i + 4 * lane, x[i]);
  const uint32_t qr = __ldg(reinterpret_cast<const uint32_t*>(q + kRank) + lane);
  const float q0 = __uint_as_float(qr << 16), q1 = __uint_as_float(qr & 0xffff0000u);

  const int64_t req = p.t2r ? (int64_t)__ldg(p.t2r + row) : (int64_t)row;
  const int capacity = p.indices ? p.topk : p.cache.pages_per_req * p.cache.page_size;
  const int count = p.counts ? max(__ldg(p.counts + row), 0) : capacity;
  const int columns = req >= 0 && req < p.cache.num_reqs ? min(count, capacity) : 0;
  const int own = p.nodes > 1 ? count - p.nodes : 0x7fffffff;  // the first node's place
  float m = -INFINITY, l = 0.f;
  for (int col = 0; col < columns; ++col) {
    if (p.nodes > 1 && col >= own) {
      const int d = col - own;
      const bool seen = p.tree ? (__ldg(p.tree + ((int64_t)row * p.nodes + node) * p.tree_words + d / 32) >> (d % 32)) & 1 : d <= node;
      if (!seen) continue;
    }
    const int t = p.indices ? __ldg(p.indices + (int64_t)row * p.indices_stride + col) : col;
    const int slot = latent_slot(p.cache, req, t);
    if (slot < 0) continue;
    float v[kChunks][4];
    float s = __ldg(p.cache.scales + slot);
    s = s != s ? s : fminf(fmaxf(s, kLatentLeastScale), kLatentMostScale);
    const uint32_t kr = __ldg(reinterpret_cast<const uint32_t*>(p.cache.rope + (int64_t)slot * kLatentRope) + lane);
    float sum = q0 * __uint_as_float(kr << 16) + q1 * __uint_as_float(kr & 0xffff0000u);
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const uint32_t c = __ldg(reinterpret_cast<const uint32_t*>(p.cache.codes + (int64_t)slot * kRank + 128 * i) + lane);
      const float2 lo = e4m3x2_to_f32x2((uint16_t)c), hi = e4m3x2_to_f32x2((uint16_t)(c >> 16));
      v[i][0] = lo.x, v[i][1] = lo.y, v[i][2] = hi.x, v[i][3] = hi.y;
#pragma unroll
      for (int j = 0; j < 4; ++j) sum = fmaf(x[i][j], v[i][j], sum);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const float score = sum * s * p.score_scale_log2;
    const float next = fmaxf(m, score);
    const float back = exp2f(m - next), w = exp2f(score - next);
    m = next;
    l = l * back + w;
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = o[i][j] * back + w * s * v[i][j];
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  __nv_bfloat16* out = p.out + at * kRank + 4 * lane;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(o[i][0] * inv, o[i][1] * inv);
    const __nv_bfloat162 b = __floats2bfloat162_rn(o[i][2] * inv, o[i][3] * inv);
    *reinterpret_cast<__nv_bfloat162*>(out + 128 * i) = a;
    *reinterpret_cast<__nv_bfloat162*>(out + 128 * i + 2) = b;
  }
}

}  // namespace

cudaError_t launch_latent_decode(const LatentDecodeParams& p, cudaStream_t stream) {
  const int64_t grid = ((int64_t)p.rows * p.nodes * p.heads + kLdWarps - 1) / kLdWarps;
  if (grid > 0x7fffffffll) return cudaErrorInvalidValue;
  switch (p.cache.rank / 128) {
    case 1: qsa_latent_decode_kernel<1><<<(unsigned)grid, 32 * kLdWarps, 0, stream>>>(p); break;
    case 2: qsa_latent_decode_kernel<2><<<(unsigned)grid, 32 * kLdWarps, 0, stream>>>(p); break;
    case 3: qsa_latent_decode_kernel<3><<<(unsigned)grid, 32 * kLdWarps, 0, stream>>>(p); break;
    default: qsa_latent_decode_kernel<4><<<(unsigned)grid, 32 * kLdWarps, 0, stream>>>(p); break;
  }
  return cudaGetLastError();
}

}  // namespace qsa
