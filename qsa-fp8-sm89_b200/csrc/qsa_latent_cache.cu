// The latent cache's writer and reader.
//
// Append, a warp a token:
//   y     = c * rsqrt(mean(c^2) + eps) * weight
//   scale = 2^e, the least power of two with max|y| <= 448 scale
//   codes = e4m3fn(y / scale),  rope = bf16(rotated r / scale)
// Read: scale * codes and scale * rope.
//
// The scale is a power of two: a division by it rounds nothing (E4M3 has an
// exponent of its own, so that a finer scale would gain only where the smallest
// codes are subnormal), and attention can take it through exponents.
#include "qsa_latent.cuh"
#include "qsa_rope.cuh"

namespace qsa {
namespace {

constexpr int kLcWarps = 4;

// The exponent of the least power of two s with top <= 448 s, for a finite top >= 0.
__device__ __forceinline__ int latent_exponent(float top) {
  const uint32_t bits = __float_as_uint(top);
  // 448 = 1.75 * 2^8
  const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, -60), 60);
}

// A lane holds elements 128 i + 4 lane .. + 3 of the latent, and of the rotated
// part one pair, or two neighbours past the rotated elements.
template <typename T, int kChunks>
__global__ void __launch_bounds__(32 * kLcWarps) qsa_latent_append_kernel(const __grid_constant__ LatentAppendParams p) {
  constexpr int kRank = 128 * kChunks;
  const int lane = threadIdx.x % 32;
  const int token = blockIdx.x * kLcWarps + threadIdx.x / 32;
  if (token >= p.list.tokens) return;
  const T* src = static_cast<const T*>(p.c) + (int64_t)token * p.c_stride;
  float y[kChunks][4];
#pragma unroll
  for (int i = 0; i < kChunks; ++i) latent_load4(src + 128 * i + 4 * lane, y[i]);
  const int half = p.rope.rotary >> 1;
  int a = 2 * lane, b = 2 * lane + 1;  // the lane's two rotated elements
  if (lane < half && !p.rope.interleaved) a = lane, b = half + lane;
  const T* rsrc = static_cast<const T*>(p.r) + (int64_t)token * p.r_stride;
  float u = latent_to_float(rsrc[a]), v = latent_to_float(rsrc[b]);
  int slot, pos;
  if (!latent_place(p.cache, p.list, token, lane, slot, pos) || slot < 0) return;

  if (p.c_weight) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum = fmaf(y[i][j], y[i][j], sum);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    // one Newton step from the 2 ulp of rsqrtf to nearly the nearest value: what
    // a token is off by shifts all its codes
    const float m = fmaf(sum, 1.0f / kRank, p.eps);
    float r = rsqrtf(m);
    const float t = m * r, e = fmaf(-fmaf(m, r, -t), r, fmaf(-t, r, 1.0f));  // 1 - m r r
    if (r > 0.f && r <= 3.4e38f) r = fmaf(0.5f * r, e, r);
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      float w[4];
      if (p.weight_dtype == QSA_B200_DTYPE_F32)
        latent_load4(static_cast<const float*>(p.c_weight) + 128 * i + 4 * lane, w);
      else if (p.weight_dtype == QSA_B200_DTYPE_F16)
        latent_load4(static_cast<const __half*>(p.c_weight) + 128 * i + 4 * lane, w);
      else
        latent_load4(static_cast<const __nv_bfloat16*>(p.c_weight) + 128 * i + 4 * lane, w);
#pragma unroll
      for (int j = 0; j < 4; ++j) y[i][j] = y[i][j] * r * w[j];
    }
  }
  float top = 0.f;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < kChunks; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float m = fabsf(y[i][j]);
      if (m <= 3.402823466e38f) top = fmaxf(top, m);
      nan = nan || m != m;
    }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  nan = __any_sync(0xffffffffu, nan);
  const int e = latent_exponent(top);
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);  // 1 / scale

  uint8_t* dst = p.cache.codes + (int64_t)slot * kRank + 4 * lane;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[i][0] * inv, y[i][1] * inv), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[i][2] * inv, y[i][3] * inv), __NV_SATFINITE, __NV_E4M3);
    *reinterpret_cast<uint32_t*>(dst + 128 * i) = nan ? 0u : lo | hi << 16;
  }
  if (lane < half) {
    const int at = p.rope.positions ? __ldg(p.rope.positions + token) : pos;
    if (at >= 0 && at < p.rope.table_len) {
      const float* row = p.rope.table + (int64_t)at * p.rope.rotary + lane;
      const float cs = __ldg(row), sn = __ldg(row + half);
      const float x = u * cs - v * sn;
      v = v * cs + u * sn;
      u = x;
    } else {
      u = v = 0.f;
    }
  } else if (half > 0) {
    const int at = p.rope.positions ? __ldg(p.rope.positions + token) : pos;
    if (at < 0 || at >= p.rope.table_len) u = v = 0.f;
  }
  __nv_bfloat16* rdst = p.cache.rope + (int64_t)slot * kLatentRope;
  rdst[a] = __float2bfloat16_rn(u * inv);
  rdst[b] = __float2bfloat16_rn(v * inv);
  if (lane == 0) p.cache.scales[slot] = nan ? __int_as_float(0x7fffffff) : __uint_as_float((uint32_t)(127 + e) << 23);
}

__device__ __forceinline__ float latent_scale(float s) {
  return s != s ? s : fminf(fmaxf(s, kLatentLeastScale), kLatentMostScale);
}

template <typename T, int kChunks>
__global__ void __launch_bounds__(32 * kLcWarps) qsa_latent_read_kernel(const __grid_constant__ LatentReadParams p) {
  constexpr int kRank = 128 * kChunks;
  const int lane = threadIdx.x % 32;
  const int token = blockIdx.x * kLcWarps + threadIdx.x / 32;
  if (token >= p.list.tokens) return;
  int slot, pos;
  if (!latent_place(p.cache, p.list, token, lane, slot, pos)) return;
  uint32_t codes[kChunks] = {};
  uint32_t rope = 0;
  float s = 0.f;
  if (slot >= 0) {
    const uint8_t* src = p.cache.codes + (int64_t)slot * kRank + 4 * lane;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) codes[i] = __ldg(reinterpret_cast<const uint32_t*>(src + 128 * i));
    rope = __ldg(reinterpret_cast<const uint32_t*>(p.cache.rope + (int64_t)slot * kLatentRope) + lane);
    s = latent_scale(__ldg(p.cache.scales + slot));
  }
  T* dst = static_cast<T*>(p.c) + (int64_t)token * kRank + 4 * lane;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    const float2 lo = e4m3x2_to_f32x2((uint16_t)codes[i]), hi = e4m3x2_to_f32x2((uint16_t)(codes[i] >> 16));
    const float x[4] = {lo.x * s, lo.y * s, hi.x * s, hi.y * s};
    store4(dst + 128 * i, x);
  }
  T* rdst = static_cast<T*>(p.r) + (int64_t)token * kLatentRope + 2 * lane;
  const float a = __uint_as_float(rope << 16) * s, b = __uint_as_float(rope & 0xffff0000u) * s;
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float2*>(rdst) = make_float2(a, b);
  } else if constexpr (std::is_same<T, __half>::value) {
    *reinterpret_cast<__half2*>(rdst) = __floats2half2_rn(a, b);
  } else {
    *reinterpret_cast<__nv_bfloat162*>(rdst) = __floats2bfloat162_rn(a, b);
  }
}

template <typename T>
void append(const LatentAppendParams& p, unsigned grid, cudaStream_t stream) {
  switch (p.cache.rank / 128) {
    case 1: qsa_latent_append_kernel<T, 1><<<grid, 32 * kLcWarps, 0, stream>>>(p); break;
    case 2: qsa_latent_append_kernel<T, 2><<<grid, 32 * kLcWarps, 0, stream>>>(p); break;
    case 3: qsa_latent_append_kernel<T, 3><<<grid, 32 * kLcWarps, 0, stream>>>(p); break;
    default: qsa_latent_append_kernel<T, 4><<<grid, 32 * kLcWarps, 0, stream>>>(p); break;
  }
}

template <typename T>
void read(const LatentReadParams& p, unsigned grid, cudaStream_t stream) {
  switch (p.cache.rank / 128) {
    case 1: qsa_latent_read_kernel<T, 1><<<grid, 32 * kLcWarps, 0, stream>>>(p); break;
    case 2: qsa_latent_read_kernel<T, 2><<<grid, 32 * kLcWarps, 0, stream>>>(p); break;
    case 3: qsa_latent_read_kernel<T, 3><<<grid, 32 * kLcWarps, 0, stream>>>(p); break;
    default: qsa_latent_read_kernel<T, 4><<<grid, 32 * kLcWarps, 0, stream>>>(p); break;
  }
}

}  // namespace

cudaError_t launch_latent_append(const LatentAppendParams& p, cudaStream_t stream) {
  const unsigned grid = ((unsigned)p.list.tokens + kLcWarps - 1) / kLcWarps;
  switch (p.dtype) {
    case QSA_B200_DTYPE_BF16: append<__nv_bfloat16>(p, grid, stream); break;
    case QSA_B200_DTYPE_F16: append<__half>(p, grid, stream); break;
    default: append<float>(p, grid, stream); break;
  }
  return cudaGetLastError();
}

cudaError_t launch_latent_read(const LatentReadParams& p, cudaStream_t stream) {
  const unsigned grid = ((unsigned)p.list.tokens + kLcWarps - 1) / kLcWarps;
  switch (p.dtype) {
    case QSA_B200_DTYPE_BF16: read<__nv_bfloat16>(p, grid, stream); break;
    case QSA_B200_DTYPE_F16: read<__half>(p, grid, stream); break;
    default: read<float>(p, grid, stream); break;
  }
  return cudaGetLastError();
}

}  // namespace qsa
