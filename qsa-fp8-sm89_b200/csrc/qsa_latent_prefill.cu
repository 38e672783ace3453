// Attention of prompts in the expanded form: keys of 128 values a head and 64
// for all heads, values of 128.
//
// A warp takes one head of one query token and goes through its keys, one at a
// time: lane l holds elements 4l .. 4l+3 of the 128 and two rotated ones.
// Softmax by a running maximum and sum, all in fp32.
#include "../../include/qsa_b200.h"
#include "qsa_latent.cuh"

namespace qsa {
namespace {

constexpr int kLpWarps = 4;

__device__ __forceinline__ void load2(const __nv_bfloat16* at, float& a, float& b) {
  const uint32_t v = __ldg(reinterpret_cast<const uint32_t*>(at));
  a = __uint_as_float(v << 16), b = __uint_as_float(v & 0xffff0000u);
}
__device__ __forceinline__ void load2(const __half* at, float& a, float& b) {
  const uint32_t v = __ldg(reinterpret_cast<const uint32_t*>(at));
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
  a = f.x, b = f.y;
}

template <typename T>
__global__ void __launch_bounds__(32 * kLpWarps) qsa_latent_prefill_kernel(const __grid_constant__ LatentPrefillParams p) {
  const int lane = threadIdx.x % 32;
  const int64_t at = (int64_t)blockIdx.x * kLpWarps + threadIdx.x / 32;  // (token, head)
  if (at >= (int64_t)p.q_tokens * p.heads) return;
  const int token = (int)(at / p.heads), head = (int)(at % p.heads);
  int lo = 0, hi = p.entries;  // the last entry that begins at or before the token
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (__ldg(p.cu_q + mid) <= token) lo = mid; else hi = mid;
  }
  const int q0 = __ldg(p.cu_q + lo), q1 = __ldg(p.cu_q + lo + 1);
  if (token < q0 || token >= q1) return;
  const int k0 = max(__ldg(p.cu_k + lo), 0), k1 = min(__ldg(p.cu_k + lo + 1), p.k_tokens);
  const int last = p.causal ? min(k1, k0 + (token - q0) + (k1 - k0) - (q1 - q0) + 1) : k1;
  const T* q = static_cast<const T*>(p.q) + token * p.q_stride + head * p.q_head_stride;
  float x[4], o[4] = {}, r0, r1;
  latent_load4(q + 4 * lane, x);
  load2(q + 128 + 2 * lane, r0, r1);
  float m = -INFINITY, l = 0.f;
  for (int j = k0; j < last; ++j) {
    float k[4], v[4], kr0, kr1;
    latent_load4(static_cast<const T*>(p.k) + j * p.k_stride + head * p.k_head_stride + 4 * lane, k);
    load2(static_cast<const T*>(p.k_rope) + j * p.k_rope_stride + 2 * lane, kr0, kr1);
    latent_load4(static_cast<const T*>(p.v) + j * p.v_stride + head * p.v_head_stride + 4 * lane, v);
    float sum = r0 * kr0 + r1 * kr1;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum = fmaf(x[i], k[i], sum);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const float score = sum * p.score_scale_log2;
    const float next = fmaxf(m, score);
    const float back = exp2f(m - next), w = exp2f(score - next);
    m = next;
    l = l * back + w;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = o[i] * back + w * v[i];
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* out = static_cast<T*>(p.out) + at * 128 + 4 * lane;
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = (T)(o[i] * inv);
}

}  // namespace

cudaError_t launch_latent_prefill(const LatentPrefillParams& p, cudaStream_t stream) {
  const int64_t grid = ((int64_t)p.q_tokens * p.heads + kLpWarps - 1) / kLpWarps;
  if (grid > 0x7fffffffll) return cudaErrorInvalidValue;
  if (p.dtype == QSA_B200_DTYPE_BF16)
    qsa_latent_prefill_kernel<__nv_bfloat16><<<(unsigned)grid, 32 * kLpWarps, 0, stream>>>(p);
  else
    qsa_latent_prefill_kernel<__half><<<(unsigned)grid, 32 * kLpWarps, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace qsa
