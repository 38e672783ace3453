// The latent cache's writer and reader.
//
// Append:
//   y     = c * rsqrt(mean(c^2) + eps) * weight
//   scale = 2^e, the least power of two with max|y| <= 448 scale
//   codes = e4m3fn(y / scale),  rope = bf16(rotated r / scale)
// Read: scale * codes and scale * rope.
//
// The scale is a power of two: a division by it rounds nothing (E4M3 has an
// exponent of its own, so that a finer scale would gain only where the smallest
// codes are subnormal), and attention can take it through exponents.
//
// A warp takes two tokens, whose loads are under way together: with one, 24 prompts of
// up to 4097 f16 tokens (rank 512, norm and rotation, 52000 tokens, 107 MB) take 35.6 us,
// with two 30.9, with four 32.6 (80 registers a thread); 24 whole contexts of up to 8192
// tokens (104000, 187 MB) are read in 36.9, 34.7 (5.4 TB/s) and 34.9. The reader is bound
// by its traffic; the writer by instructions as much (issue slots 60 % busy), so two
// elements go through one where they can. 256 single tokens take 5.8 us, a launch's time.
#include "qsa_latent.cuh"
#include "qsa_rope.cuh"

namespace qsa {
namespace {

constexpr int kLcWarps = 4;
constexpr int kLcTokens = 2;  // of a warp

// The exponent of the least power of two s with top <= 448 s, for a finite top >= 0.
__device__ __forceinline__ int latent_exponent(float top) {
  const uint32_t bits = __float_as_uint(top);
  // 448 = 1.75 * 2^8
  const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, -60), 60);
}

// A lane holds elements 128 i + 4 lane .. + 3 of the latent, and of the rotated
// part one pair, or two neighbours past the rotated elements. The warp's kLcTokens
// tokens are loaded, and their places found, before the first is worked on.
template <typename T, int kChunks>
__global__ void __launch_bounds__(32 * kLcWarps) qsa_latent_append_kernel(const __grid_constant__ LatentAppendParams p) {
  constexpr int kRank = 128 * kChunks;
  using Word = typename std::conditional<sizeof(T) == 4, uint4, uint2>::type;  // of 4 elements
  const int lane = threadIdx.x % 32;
  const int first = (blockIdx.x * kLcWarps + threadIdx.x / 32) * kLcTokens;
  if (first >= p.list.tokens) return;
  const int half = p.rope.rotary >> 1;
  int a = 2 * lane, b = 2 * lane + 1;  // the lane's two rotated elements
  if (lane < half && !p.rope.interleaved) a = lane, b = half + lane;
  Word words[kLcTokens][kChunks] = {};
  T us[kLcTokens] = {}, vs[kLcTokens] = {};
#pragma unroll
  for (int k = 0; k < kLcTokens; ++k)
    if (first + k < p.list.tokens) {
      const T* src = static_cast<const T*>(p.c) + (int64_t)(first + k) * p.c_stride + 4 * lane;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) words[k][i] = __ldg(reinterpret_cast<const Word*>(src + 128 * i));
      const T* rsrc = static_cast<const T*>(p.r) + (int64_t)(first + k) * p.r_stride;
      us[k] = rsrc[a], vs[k] = rsrc[b];
    }
  int its_slot, its_pos;
  latent_place(p.cache, p.list, first, kLcTokens, lane, its_slot, its_pos);
  if (p.rope.positions && lane < kLcTokens && first + lane < p.list.tokens) its_pos = __ldg(p.rope.positions + first + lane);
  if (its_pos >= p.rope.table_len) its_pos = -1;
  const uint32_t turned = __ballot_sync(0xffffffffu, its_pos >= 0);  // whose position the table holds
  uint64_t weight[kChunks][2] = {};
  if (p.c_weight) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      float w[4];
      if (p.weight_dtype == QSA_B200_DTYPE_F32)
        latent_load4(static_cast<const float*>(p.c_weight) + 128 * i + 4 * lane, w);
      else if (p.weight_dtype == QSA_B200_DTYPE_F16)
        latent_load4(static_cast<const __half*>(p.c_weight) + 128 * i + 4 * lane, w);
      else
        latent_load4(static_cast<const __nv_bfloat16*>(p.c_weight) + 128 * i + 4 * lane, w);
      weight[i][0] = pair2(w[0], w[1]), weight[i][1] = pair2(w[2], w[3]);
    }
  }
  float cs[kLcTokens], sn[kLcTokens];
#pragma unroll
  for (int k = 0; k < kLcTokens; ++k) {
    const int at = __shfl_sync(0xffffffffu, its_pos, k);
    cs[k] = sn[k] = 0.f;
    if (lane < half && at >= 0) {
      const float* row = p.rope.table + (int64_t)at * p.rope.rotary + lane;
      cs[k] = __ldg(row), sn[k] = __ldg(row + half);
    }
  }
#pragma unroll
  for (int k = 0; k < kLcTokens; ++k) {
    const int slot = __shfl_sync(0xffffffffu, its_slot, k);
    if (slot < 0) continue;
    uint64_t y[kChunks][2];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      float x[4];
      latent_widen(words[k][i], x, T());
      y[i][0] = pair2(x[0], x[1]), y[i][1] = pair2(x[2], x[3]);
    }
    float u = latent_to_float(us[k]), v = latent_to_float(vs[k]);

    if (p.c_weight) {
      uint64_t sums = 0;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) sums = fma2(y[i][1], y[i][1], fma2(y[i][0], y[i][0], sums));
      float sum, odd;
      unpair2(sums, sum, odd);
      sum += odd;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      // one Newton step from the 2 ulp of rsqrtf to nearly the nearest value: what
      // a token is off by shifts all its codes
      const float m = fmaf(sum, 1.0f / kRank, p.eps);
      float r = rsqrtf(m);
      const float t = m * r, e = fmaf(-fmaf(m, r, -t), r, fmaf(-t, r, 1.0f));  // 1 - m r r
      if (r > 0.f && r <= 3.4e38f) r = fmaf(0.5f * r, e, r);
#pragma unroll
      for (int i = 0; i < kChunks; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) y[i][j] = mul2(mul2(y[i][j], pair2(r, r)), weight[i][j]);
    }
    float part[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float a, d;
        unpair2(y[i][j], a, d);
        part[j] = max3_nan(part[j], fabsf(a), fabsf(d));
      }
    // bits of values without a sign are in the values' order, those of a NaN above all
    uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(max3_nan(part[0], part[1], part[1])));
    const bool nan = top > 0x7f800000u;
    if (top >= 0x7f800000u) {  // the largest finite one; what is infinite becomes the largest code
      float of = 0.f;
#pragma unroll
      for (int i = 0; i < kChunks; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float a, d;
          unpair2(y[i][j], a, d);
          if (fabsf(a) <= 3.402823466e38f) of = fmaxf(of, fabsf(a));
          if (fabsf(d) <= 3.402823466e38f) of = fmaxf(of, fabsf(d));
        }
      top = __reduce_max_sync(0xffffffffu, __float_as_uint(of));
    }
    const int e = latent_exponent(__uint_as_float(top));
    const float inv = __uint_as_float((uint32_t)(127 - e) << 23);  // 1 / scale

    uint8_t* dst = p.cache.codes + (int64_t)slot * kRank + 4 * lane;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      float2 lo, hi;
      unpair2(mul2(y[i][0], pair2(inv, inv)), lo.x, lo.y);
      unpair2(mul2(y[i][1], pair2(inv, inv)), hi.x, hi.y);
      const uint32_t codes = (uint32_t)__nv_cvt_float2_to_fp8x2(lo, __NV_SATFINITE, __NV_E4M3) |
                             (uint32_t)__nv_cvt_float2_to_fp8x2(hi, __NV_SATFINITE, __NV_E4M3) << 16;
      *reinterpret_cast<uint32_t*>(dst + 128 * i) = nan ? 0u : codes;
    }
    if (half > 0 && !(turned >> k & 1u)) {
      u = v = 0.f;
    } else if (lane < half) {
      const float x = u * cs[k] - v * sn[k];
      v = v * cs[k] + u * sn[k];
      u = x;
    }
    __nv_bfloat16* rdst = p.cache.rope + (int64_t)slot * kLatentRope;
    const __nv_bfloat162 uv = __floats2bfloat162_rn(u * inv, v * inv);
    if (b == a + 1) {
      *reinterpret_cast<__nv_bfloat162*>(rdst + a) = uv;
    } else {
      rdst[a] = uv.x;
      rdst[b] = uv.y;
    }
    if (lane == 0) p.cache.scales[slot] = nan ? __int_as_float(0x7fffffff) : __uint_as_float((uint32_t)(127 + e) << 23);
  }
}

__device__ __forceinline__ float latent_scale(float s) {
  return s != s ? s : fminf(fmaxf(s, kLatentLeastScale), kLatentMostScale);
}

template <typename T, int kChunks>
__global__ void __launch_bounds__(32 * kLcWarps) qsa_latent_read_kernel(const __grid_constant__ LatentReadParams p) {
  constexpr int kRank = 128 * kChunks;
  const int lane = threadIdx.x % 32;
  const int first = (blockIdx.x * kLcWarps + threadIdx.x / 32) * kLcTokens;
  if (first >= p.list.tokens) return;
  int its_slot, its_pos;
  const uint32_t named = __ballot_sync(0xffffffffu, latent_place(p.cache, p.list, first, kLcTokens, lane, its_slot, its_pos));
  float its_scale = 0.f;
  if (its_slot >= 0) its_scale = latent_scale(__ldg(p.cache.scales + its_slot));
  uint32_t codes[kLcTokens][kChunks] = {}, rope[kLcTokens] = {};
#pragma unroll
  for (int k = 0; k < kLcTokens; ++k) {
    const int slot = __shfl_sync(0xffffffffu, its_slot, k);
    if (slot < 0) continue;
    const uint8_t* src = p.cache.codes + (int64_t)slot * kRank + 4 * lane;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) codes[k][i] = __ldg(reinterpret_cast<const uint32_t*>(src + 128 * i));
    rope[k] = __ldg(reinterpret_cast<const uint32_t*>(p.cache.rope + (int64_t)slot * kLatentRope) + lane);
  }
#pragma unroll
  for (int k = 0; k < kLcTokens; ++k) {
    const float s = __shfl_sync(0xffffffffu, its_scale, k);
    if (!(named >> k & 1u)) continue;
    T* dst = static_cast<T*>(p.c) + (int64_t)(first + k) * kRank + 4 * lane;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const float2 lo = e4m3x2_to_f32x2((uint16_t)codes[k][i]), hi = e4m3x2_to_f32x2((uint16_t)(codes[k][i] >> 16));
      const float x[4] = {lo.x * s, lo.y * s, hi.x * s, hi.y * s};
      store4(dst + 128 * i, x);
    }
    T* rdst = static_cast<T*>(p.r) + (int64_t)(first + k) * kLatentRope + 2 * lane;
    const float a = __uint_as_float(rope[k] << 16) * s, b = __uint_as_float(rope[k] & 0xffff0000u) * s;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float2*>(rdst) = make_float2(a, b);
    } else if constexpr (std::is_same<T, __half>::value) {
      *reinterpret_cast<__half2*>(rdst) = __floats2half2_rn(a, b);
    } else {
      *reinterpret_cast<__nv_bfloat162*>(rdst) = __floats2bfloat162_rn(a, b);
    }
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

unsigned grid_of(int tokens) { return ((unsigned)tokens + kLcWarps * kLcTokens - 1) / (kLcWarps * kLcTokens); }

}  // namespace

cudaError_t launch_latent_append(const LatentAppendParams& p, cudaStream_t stream) {
  switch (p.dtype) {
    case QSA_B200_DTYPE_BF16: append<__nv_bfloat16>(p, grid_of(p.list.tokens), stream); break;
    case QSA_B200_DTYPE_F16: append<__half>(p, grid_of(p.list.tokens), stream); break;
    default: append<float>(p, grid_of(p.list.tokens), stream); break;
  }
  return cudaGetLastError();
}

cudaError_t launch_latent_read(const LatentReadParams& p, cudaStream_t stream) {
  switch (p.dtype) {
    case QSA_B200_DTYPE_BF16: read<__nv_bfloat16>(p, grid_of(p.list.tokens), stream); break;
    case QSA_B200_DTYPE_F16: read<__half>(p, grid_of(p.list.tokens), stream); break;
    default: read<float>(p, grid_of(p.list.tokens), stream); break;
  }
  return cudaGetLastError();
}

}  // namespace qsa
