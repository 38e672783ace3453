// RMS norm of every query and key head and the position rotation, one pass.
//
//   y = rotate(x * rsqrt(mean(x^2) + eps) * weight)   per 128-element head
//
// One half warp takes one head of one token (qsa_rope.cuh).
#include "qsa_rope.cuh"

namespace qsa {
namespace {

constexpr int kQrThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kQrThreads) qsa_qk_rope_kernel(const __grid_constant__ QkRopeParams p) {
  const int l = threadIdx.x % kRowLanes;
  const int heads = p.heads[0] + p.heads[1];
  const int64_t total = (int64_t)p.tokens * heads;
  const int64_t at = ((int64_t)blockIdx.x * kQrThreads + threadIdx.x) / kRowLanes;
  const bool live = at < total;  // every lane goes through the exchanges
  const int64_t token = live ? at / heads : 0;
  const int hh = live ? (int)(at % heads) : 0;
  const int which = hh >= p.heads[0] ? 1 : 0;
  const int h = which ? hh - p.heads[0] : hh;
  Raw8<T> raw;
  load8(static_cast<const T*>(p.x[which]) + token * p.stride[which] + h * 128 + 8 * l, raw);
  float x[8];
  widen8(raw, x);
  if (p.weight[0] || p.weight[1]) {
    float w[8], y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x[i], w[i] = 1.f;
    if (p.weight[which]) load_weight8(p.weight[which], p.weight_dtype, l, w);
    rms_norm8(y, w, p.eps);
    if (p.weight[which]) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = y[i];
    }
  }
  if (p.rope.table) {
    Turn8 t;
    load_turn8(p.rope, token, 0, l, t);
    rotate8(p.rope, t, l, x);
  }
  if (live) store8(static_cast<T*>(p.out[which]) + token * p.out_stride[which] + h * 128 + 8 * l, x);
}

}  // namespace

cudaError_t launch_qk_rope(const QkRopeParams& p, cudaStream_t stream) {
  const int64_t rows = (int64_t)p.tokens * (p.heads[0] + p.heads[1]);
  const int64_t grid = (rows * kRowLanes + kQrThreads - 1) / kQrThreads;
  if (grid > 0x7fffffffll) return cudaErrorInvalidValue;
  switch (p.dtype) {
    case QSA_B200_DTYPE_BF16: qsa_qk_rope_kernel<__nv_bfloat16><<<(unsigned)grid, kQrThreads, 0, stream>>>(p); break;
    case QSA_B200_DTYPE_F16: qsa_qk_rope_kernel<__half><<<(unsigned)grid, kQrThreads, 0, stream>>>(p); break;
    default: qsa_qk_rope_kernel<float><<<(unsigned)grid, kQrThreads, 0, stream>>>(p); break;
  }
  return cudaGetLastError();
}

}  // namespace qsa
