// RMS norm of every query and key head and the position rotation, one pass.
//
//   y = rotate(x * rsqrt(mean(x^2) + eps) * weight)   per 128-element head
//
// Bound by HBM: 2 x 128 elements a head. A half warp takes up to 8 heads of one
// token (qsa_rope.cuh), so that the token's cosines and sines are read and held
// once for them, and loads kQrBatch heads before it works on the first. With
// less than a full GPU of half warps each takes fewer heads, down to one.
#include "qsa_rope.cuh"

namespace qsa {
namespace {

constexpr int kQrThreads = 256;
constexpr int kQrHeads = 8;  // heads of a half warp, at most

template <typename T>
__global__ void __launch_bounds__(kQrThreads) qsa_qk_rope_kernel(const __grid_constant__ QkRopeParams p, int per) {
  constexpr int kQrBatch = 4;
  const int l = threadIdx.x % kRowLanes;
  const int q_parts = (p.heads[0] + per - 1) / per;
  const int parts = q_parts + (p.heads[1] + per - 1) / per;
  const int64_t at = (int64_t)blockIdx.x * (kQrThreads / kRowLanes) + threadIdx.x / kRowLanes;
  const bool live = at < (int64_t)p.tokens * parts;  // every lane goes through the norm's exchanges
  const int64_t token = live ? (at <= 0xffffffffll ? (uint32_t)at / (uint32_t)parts : at / parts) : 0;
  const int part = live ? (int)(at - token * parts) : 0;
  const int which = part >= q_parts ? 1 : 0;
  const int h0 = (part - which * q_parts) * per;
  const int n = live ? min(per, p.heads[which] - h0) : 0;
  const Pieces pieces = lane_pieces(p.rope, l);
  const T* src = static_cast<const T*>(p.x[which]) + token * p.stride[which] + h0 * 128;
  T* dst = static_cast<T*>(p.out[which]) + token * p.out_stride[which] + h0 * 128;
  const void* weight = p.weight[which];
  float w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = 1.f;
  if (weight) load_weight8(weight, p.weight_dtype, pieces, w);
  Turn4 t;
  if (p.rope.table) load_turn4(p.rope, token, 0, l, t);
  const bool norms = p.weight[0] || p.weight[1];
  for (int b = 0; b < per; b += kQrBatch) {
    Raw8<T> raw[kQrBatch];
#pragma unroll
    for (int i = 0; i < kQrBatch; ++i) {
      raw[i] = {};
      if (b + i < n) load8(src + (b + i) * 128, pieces, raw[i]);
    }
#pragma unroll
    for (int i = 0; i < kQrBatch; ++i) {
      if (b + i >= per) break;  // the same for the whole warp
      float x[8];
      widen8(raw[i], x);
      if (norms) {
        float y[8];
#pragma unroll
        for (int d = 0; d < 8; ++d) y[d] = x[d];
        rms_norm8(y, w, p.eps);
#pragma unroll
        for (int d = 0; d < 8; ++d) x[d] = weight ? y[d] : x[d];
      }
      if (p.rope.table) rotate8(p.rope, t, x);
      if (b + i < n) store8(dst + (b + i) * 128, pieces, x);
    }
  }
}

}  // namespace

cudaError_t launch_qk_rope(const QkRopeParams& p, cudaStream_t stream) {
  const int64_t rows = (int64_t)p.tokens * (p.heads[0] + p.heads[1]);
  // 148 SMs hold 148 x 128 half warps
  int per = 1;
  while (per < kQrHeads && rows / (2 * per) >= 148 * 128) per *= 2;
  const int64_t parts = (p.heads[0] + per - 1) / per + (p.heads[1] + per - 1) / per;
  const int64_t grid = (p.tokens * parts * kRowLanes + kQrThreads - 1) / kQrThreads;
  if (grid > 0x7fffffffll) return cudaErrorInvalidValue;
  switch (p.dtype) {
    case QSA_B200_DTYPE_BF16: qsa_qk_rope_kernel<__nv_bfloat16><<<(unsigned)grid, kQrThreads, 0, stream>>>(p, per); break;
    case QSA_B200_DTYPE_F16: qsa_qk_rope_kernel<__half><<<(unsigned)grid, kQrThreads, 0, stream>>>(p, per); break;
    default: qsa_qk_rope_kernel<float><<<(unsigned)grid, kQrThreads, 0, stream>>>(p, per); break;
  }
  return cudaGetLastError();
}

}  // namespace qsa
