// One 128-element head by a half warp: load, RMS norm, position rotation.
//
// Lane l of the 16 holds two pieces of 4 elements. Where pairs are (j, j + R/2)
// of R rotated elements, lanes below R/8 hold elements 4l .. 4l+3 and R/2 + 4l
// .. + 3, which are the two sides of pairs 4l .. 4l+3; the others, and all lanes
// where pairs are neighbours, hold elements 8l .. 8l+7. A rotation then needs
// no exchange between lanes, and four cosines and sines a lane in either form.
// A norm takes 4 shuffles. Everything is fp32; the caller rounds.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "../../include/qsa_b200.h"
#include "qsa_common.cuh"
#include "qsa_internal.h"

namespace qsa {

constexpr int kRowLanes = 16;  // lanes of a row, 8 elements each

enum { kPlain = 0, kHalves = 1, kNeighbours = 2 };  // no rotation; its pairs

// First elements of a lane's two pieces.
struct Pieces {
  int a, b;
};
template <int kTurn>
__device__ __forceinline__ Pieces lane_pieces(int l, int rotary) {
  if (kTurn == kHalves && l < (rotary >> 3)) return {4 * l, (rotary >> 1) + 4 * l};
  return {8 * l, 8 * l + 4};
}

// A lane's 8 elements as loaded, widened later so that several rows' loads can
// be in flight together.
template <typename T>
struct Raw8 {
  typename std::conditional<sizeof(T) == 4, uint4, uint2>::type a, b;
};

template <typename T>
__device__ __forceinline__ void load8(const T* row, Pieces at, Raw8<T>& r) {
  using W = decltype(r.a);
  r.a = *reinterpret_cast<const W*>(row + at.a);
  r.b = *reinterpret_cast<const W*>(row + at.b);
}

__device__ __forceinline__ void widen4(const uint4& w, float* x, float) {
  x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y), x[2] = __uint_as_float(w.z), x[3] = __uint_as_float(w.w);
}
__device__ __forceinline__ void widen4(const uint2& w, float* x, __nv_bfloat16) {
  const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w.x));
  const float2 g = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w.y));
  x[0] = f.x, x[1] = f.y, x[2] = g.x, x[3] = g.y;
}
__device__ __forceinline__ void widen4(const uint2& w, float* x, __half) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
  const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
  x[0] = f.x, x[1] = f.y, x[2] = g.x, x[3] = g.y;
}

template <typename T>
__device__ __forceinline__ void widen8(const Raw8<T>& r, float (&x)[8]) {
  widen4(r.a, x, T());
  widen4(r.b, x + 4, T());
}

__device__ __forceinline__ void store4(float* dst, const float* x) {
  *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void store4(__nv_bfloat16* dst, const float* x) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
  *reinterpret_cast<uint2*>(dst) =
      make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}
__device__ __forceinline__ void store4(__half* dst, const float* x) {
  const __half2 a = __floats2half2_rn(x[0], x[1]), b = __floats2half2_rn(x[2], x[3]);
  *reinterpret_cast<uint2*>(dst) =
      make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

template <typename T>
__device__ __forceinline__ void store8(T* row, Pieces at, const float (&x)[8]) {
  store4(row + at.a, x);
  store4(row + at.b, x + 4);
}

// A lane's elements of a norm weight.
__device__ __forceinline__ void load_weight8(const void* weight, int dtype, Pieces at, float (&w)[8]) {
  if (dtype == QSA_B200_DTYPE_F32) {
    Raw8<float> r;
    load8(static_cast<const float*>(weight), at, r);
    widen8(r, w);
  } else if (dtype == QSA_B200_DTYPE_F16) {
    Raw8<__half> r;
    load8(static_cast<const __half*>(weight), at, r);
    widen8(r, w);
  } else {
    Raw8<__nv_bfloat16> r;
    load8(static_cast<const __nv_bfloat16*>(weight), at, r);
    widen8(r, w);
  }
}

// x *= rsqrt(mean(x^2) + eps) * w over the half warp's 128 elements, for N rows
// whose exchanges run side by side. Every lane goes through them; where `norms` is
// false it keeps its rows.
template <int N>
__device__ __forceinline__ void rms_norm8(float (&x)[N][8], const float (&w)[8], float eps, bool norms = true) {
  float s[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    uint64_t sum = 0;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const uint64_t v = pair2(x[n][i], x[n][i + 1]);
      sum = fma2(v, v, sum);
    }
    float even, odd;
    unpair2(sum, even, odd);
    s[n] = even + odd;
  }
#pragma unroll
  for (int o = kRowLanes / 2; o > 0; o >>= 1)
#pragma unroll
    for (int n = 0; n < N; ++n) s[n] += __shfl_xor_sync(0xffffffffu, s[n], o);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    // one Newton step from the 2 ulp of rsqrtf to nearly the nearest value: what a
    // row is off by shifts all its codes where it is quantised
    const float v = fmaf(s[n], 1.0f / 128.0f, eps);
    float r = rsqrtf(v);
    const float t = v * r, e = fmaf(-fmaf(v, r, -t), r, fmaf(-t, r, 1.0f));  // 1 - v r r
    if (r > 0.f && r <= 3.4e38f) r = fmaf(0.5f * r, e, r);
    if (!norms) r = 1.f;
#pragma unroll
    for (int i = 0; i < 8; i += 2)
      unpair2(mul2(mul2(pair2(x[n][i], x[n][i + 1]), pair2(r, r)), pair2(w[i], w[i + 1])), x[n][i], x[n][i + 1]);
  }
}

// Axis of pair j.
__device__ __forceinline__ int rope_axis(const RopeParams& p, int j) {
  int axis = 0;
#pragma unroll
  for (int a = 0; a < kRopeMaxAxes - 1; ++a) axis += (a + 1 < p.axes && j >= p.ends[a]) ? 1 : 0;
  return axis;
}

// The token's position on an axis; `own` where the rotation has no list.
__device__ __forceinline__ int rope_position(const RopeParams& p, int64_t token, uint32_t own, int axis) {
  if (!p.positions) return (int)min(own, 0x7fffffffu);
  return __ldg(p.positions + axis * p.axis_stride + token);
}

// The cosines and sines of a lane's pairs 4l .. 4l+3; false where a position
// lies outside the table (nothing is read there). turning: lanes that hold
// rotated elements.
__device__ __forceinline__ bool load_turn(const RopeParams& p, int64_t token, uint32_t own, int l, int turning, float4& c,
                                          float4& s) {
  bool in = true;
  for (int a = 0; a < p.axes; ++a) {
    const int pos = rope_position(p, token, own, a);
    in = in && pos >= 0 && pos < p.table_len;
  }
  if (!in || l >= turning) return in;
  const int half = p.rotary >> 1;
  if (p.quads) {
    const float* at = p.table + (int64_t)rope_position(p, token, own, rope_axis(p, 4 * l)) * p.rotary + 4 * l;
    c = __ldg(reinterpret_cast<const float4*>(at));
    s = __ldg(reinterpret_cast<const float4*>(at + half));
  } else {
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float* at = p.table + (int64_t)rope_position(p, token, own, rope_axis(p, 4 * l + i)) * p.rotary + 4 * l + i;
      v[i] = __ldg(at), v[4 + i] = __ldg(at + half);
    }
    c = make_float4(v[0], v[1], v[2], v[3]), s = make_float4(v[4], v[5], v[6], v[7]);
  }
  return in;
}

// A row outside the table becomes zeros. turns: the lane holds rotated elements.
template <int kTurn>
__device__ __forceinline__ void turn_row(const float4& c, const float4& s, bool in, bool turns, float (&x)[8]) {
  if constexpr (kTurn != kPlain) {
    const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
    if (turns && kTurn == kHalves) {
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const uint64_t u = pair2(x[i], x[i + 1]), v = pair2(x[4 + i], x[5 + i]);
        const uint64_t co = pair2(cc[i], cc[i + 1]);
        unpair2(fma2(u, co, mul2(v, pair2(-ss[i], -ss[i + 1]))), x[i], x[i + 1]);
        unpair2(fma2(v, co, mul2(u, pair2(ss[i], ss[i + 1]))), x[4 + i], x[5 + i]);
      }
    } else if (turns) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float &u = x[2 * i], &v = x[2 * i + 1];
        const float y = u * cc[i] - v * ss[i];
        v = v * cc[i] + u * ss[i];
        u = y;
      }
    }
    if (!in) {
#pragma unroll
      for (int d = 0; d < 8; ++d) x[d] = 0.f;
    }
  }
}

}  // namespace qsa
