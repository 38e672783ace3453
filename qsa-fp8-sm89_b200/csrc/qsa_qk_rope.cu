// RMS norm of every query and key head and the position rotation, one pass.
//
//   y = rotate(x * rsqrt(mean(x^2) + eps) * weight)   per 128-element head
//
// Bound by HBM: 2 x 128 elements a head. A half warp takes up to 8 heads of one
// token (qsa_rope.cuh), so that the token's cosines and sines are read and held
// once for them, and loads 2 heads before it works on the first. With less than
// a full GPU of half warps each takes fewer heads, down to one. The pairing and
// the norm are template parameters: 43 M instead of 55 M instructions at the size
// below. 9 CTAs of 128 threads an SM (56 registers).
//
// 16384 tokens of 32 + 8 heads of bf16, 2 x 168 MB and the table's 8 MB: 67.8 us,
// 5.1 TB/s (a plain copy: 6.5). 4 heads at a time and 256 threads: 71.7; 8 CTAs
// an SM: 70; 10: 68.1, with spills; loads ahead of the table's rows and a batch
// ahead: 73 to 86. Warps wait for memory most of the time (56 % of DRAM, 62 % of
// the issue slots). 256 tokens of 64 + 8 heads of f16: 6.2 us one after the other
// in a graph, 12.3 with a cold L2: a half warp's heads are loaded after its position
// and its table row, three rounds to memory. 1531 tokens of 24 + 4 heads of fp32 with
// three axes: 8.1 us and 14 to 16 (from Python back to back 10.2; 4 heads at a
// time: 14.6).
#include "qsa_rope.cuh"

namespace qsa {
namespace {

constexpr int kQrThreads = 128;
constexpr int kQrHeads = 8;  // heads of a half warp, at most

// kTurn: the rotation's pairs, or none. kNorm: some heads are normed.
template <typename T, int kTurn, bool kNorm>
__global__ void __launch_bounds__(kQrThreads, sizeof(T) == 4 ? 8 : 9) qsa_qk_rope_kernel(const __grid_constant__ QkRopeParams p, int per) {
  constexpr int kBatch = 2;
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
  const int turning = kTurn == kPlain ? 0 : p.rope.rotary >> 3;  // lanes that hold rotated elements
  const Pieces pieces = lane_pieces<kTurn>(l, p.rope.rotary);
  const T* src = static_cast<const T*>(p.x[which]) + token * p.stride[which] + h0 * 128;
  T* dst = static_cast<T*>(p.out[which]) + token * p.out_stride[which] + h0 * 128;
  const void* weight = p.weight[which];
  float w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = 1.f;
  if (kNorm && weight) load_weight8(weight, p.weight_dtype, pieces, w);
  float4 c = {}, sn = {};
  const bool in = kTurn == kPlain || load_turn(p.rope, token, 0, l, turning, c, sn);

  // heads b .. b + kBatch - 1; kFull: every lane of the warp has all of them
  auto batch = [&](int b, auto full) {
    constexpr bool kFull = decltype(full)::value;
    Raw8<T> raw[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (!kFull) raw[i] = {};
      if (kFull || b + i < n) load8(src + (b + i) * 128, pieces, raw[i]);
    }
    float x[kBatch][8];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) widen8(raw[i], x[i]);
    if constexpr (kNorm) rms_norm8(x, w, p.eps, weight != nullptr);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      turn_row<kTurn>(c, sn, in, l < turning, x[i]);
      if (kFull || b + i < n) store8(dst + (b + i) * 128, pieces, x[i]);
    }
  };
  int b = 0;
  for (; b + kBatch <= per && __all_sync(0xffffffffu, b + kBatch <= n); b += kBatch) batch(b, std::true_type());
  for (; b < per; b += kBatch) batch(b, std::false_type());
}

template <typename T, int kTurn>
void launch(const QkRopeParams& p, unsigned grid, int per, cudaStream_t stream) {
  if (p.weight[0] || p.weight[1])
    qsa_qk_rope_kernel<T, kTurn, true><<<grid, kQrThreads, 0, stream>>>(p, per);
  else
    qsa_qk_rope_kernel<T, kTurn, false><<<grid, kQrThreads, 0, stream>>>(p, per);
}

template <typename T>
void launch(const QkRopeParams& p, unsigned grid, int per, cudaStream_t stream) {
  if (!p.rope.table)
    launch<T, kPlain>(p, grid, per, stream);
  else if (!p.rope.interleaved)
    launch<T, kHalves>(p, grid, per, stream);
  else
    launch<T, kNeighbours>(p, grid, per, stream);
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
    case QSA_B200_DTYPE_BF16: launch<__nv_bfloat16>(p, (unsigned)grid, per, stream); break;
    case QSA_B200_DTYPE_F16: launch<__half>(p, (unsigned)grid, per, stream); break;
    default: launch<float>(p, (unsigned)grid, per, stream); break;
  }
  return cudaGetLastError();
}

}  // namespace qsa
