// One 128-element head by a half warp: load, RMS norm, position rotation.
//
// Lane l of the 16 holds elements 8l .. 8l+7. A norm is then 8 products and
// 4 shuffles; the partner of element d in a rotation of half h = rotary / 2
// is element d + h, 8 | h, so whole lanes exchange: lane l and lane l + h/8
// (adjacent pairs stay inside a lane). Everything is fp32; the caller rounds.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "../../include/qsa_b200.h"
#include "qsa_internal.h"

namespace qsa {

constexpr int kRowLanes = 16;  // lanes of a row, 8 elements each

// 8 consecutive elements as loaded (16 bytes, or 32 in fp32), widened later
// so that several rows' loads can be in flight together
template <typename T>
struct Raw8 {
  uint4 w[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ void load8(const T* src, Raw8<T>& r) {
  const uint4* p = reinterpret_cast<const uint4*>(src);
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 2); ++i) r.w[i] = p[i];
}

template <typename T>
__device__ __forceinline__ void widen8(const Raw8<T>& r, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    const uint32_t w[8] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w, r.w[1].x, r.w[1].y, r.w[1].z, r.w[1].w};
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
  } else {
    const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 f;
      if constexpr (std::is_same<T, __nv_bfloat16>::value)
        f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
      else
        f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* dst, const float (&x)[8]) {
  uint4* p = reinterpret_cast<uint4*>(dst);
  if constexpr (sizeof(T) == 4) {
    p[0] = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    p[1] = make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    *p = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Elements 8l .. 8l+7 of a norm weight.
__device__ __forceinline__ void load_weight8(const void* weight, int dtype, int l, float (&w)[8]) {
  if (dtype == QSA_B200_DTYPE_F32) {
    Raw8<float> r;
    load8(static_cast<const float*>(weight) + 8 * l, r);
    widen8(r, w);
  } else if (dtype == QSA_B200_DTYPE_F16) {
    Raw8<__half> r;
    load8(static_cast<const __half*>(weight) + 8 * l, r);
    widen8(r, w);
  } else {
    Raw8<__nv_bfloat16> r;
    load8(static_cast<const __nv_bfloat16*>(weight) + 8 * l, r);
    widen8(r, w);
  }
}

// x *= rsqrt(mean(x^2) + eps) * w over the half warp's 128 elements.
__device__ __forceinline__ void rms_norm8(float (&x)[8], const float (&w)[8], float eps) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s = fmaf(x[i], x[i], s);
#pragma unroll
  for (int o = kRowLanes / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const float r = rsqrtf(fmaf(s, 1.0f / 128.0f, eps));
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = x[i] * r * w[i];
}

// A lane's cosines and sines: for adjacent pairs the first four are its four
// pairs', for split halves element i's pair (8 (l mod h/8) + i).
struct Turn8 {
  float c[8], s[8];
  bool in;  // the token's positions lie inside the table
};

// Position of the token on the axis of pair j. `own`: the position where the
// rotation has no list of positions.
__device__ __forceinline__ int rope_position(const RopeParams& p, int64_t token, int64_t own, int j) {
  if (!p.positions) return own > 0x7fffffffll ? 0x7fffffff : (int)own;
  int axis = 0;
  if (p.axes > 1) {
#pragma unroll
    for (int a = 0; a < kRopeMaxAxes - 1; ++a) axis += (a + 1 < p.axes && j >= p.ends[a]) ? 1 : 0;
  }
  return __ldg(p.positions + axis * p.axis_stride + token);
}

// Must run in every lane of the half warp (lanes past the rotated elements
// get the identity). Reads nothing outside the table.
__device__ __forceinline__ void load_turn8(const RopeParams& p, int64_t token, int64_t own, int l, Turn8& t) {
#pragma unroll
  for (int i = 0; i < 8; ++i) t.c[i] = 1.f, t.s[i] = 0.f;
  t.in = true;
  const int half = p.rotary >> 1;
  const int lanes = p.rotary >> 3;  // lanes that hold rotated elements
  if (p.axes == 1) {
    const int pos = rope_position(p, token, own, 0);
    t.in = pos >= 0 && pos < p.table_len;
  } else {
    for (int a = 0; a < p.axes; ++a) {
      const int pos = __ldg(p.positions + a * p.axis_stride + token);
      t.in = t.in && pos >= 0 && pos < p.table_len;
    }
  }
  if (!t.in || l >= lanes) return;
  const int n = p.interleaved ? 4 : 8;                          // pairs of this lane
  const int j0 = p.interleaved ? 4 * l : 8 * (l % (lanes >> 1));  // the first of them
  if (p.quads) {
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      if (i >= n) break;
      const float* row = p.table + (int64_t)rope_position(p, token, own, j0 + i) * p.rotary + j0 + i;
      const float4 c = __ldg(reinterpret_cast<const float4*>(row));
      const float4 s = __ldg(reinterpret_cast<const float4*>(row + half));
      t.c[i] = c.x, t.c[i + 1] = c.y, t.c[i + 2] = c.z, t.c[i + 3] = c.w;
      t.s[i] = s.x, t.s[i + 1] = s.y, t.s[i + 2] = s.z, t.s[i + 3] = s.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i >= n) break;
      const float* row = p.table + (int64_t)rope_position(p, token, own, j0 + i) * p.rotary + j0 + i;
      t.c[i] = __ldg(row);
      t.s[i] = __ldg(row + half);
    }
  }
}

// Rotates the half warp's row. Every lane of the warp takes part in the
// exchange.
__device__ __forceinline__ void rotate8(const RopeParams& p, const Turn8& t, int l, float (&x)[8]) {
  if (p.interleaved) {
    if (l < (p.rotary >> 3)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = x[2 * i], b = x[2 * i + 1];
        x[2 * i] = a * t.c[i] - b * t.s[i];
        x[2 * i + 1] = b * t.c[i] + a * t.s[i];
      }
    }
  } else {
    const int hl = p.rotary >> 4;  // lanes of one half
    const int partner = l < hl ? l + hl : l < 2 * hl ? l - hl : l;
    const float sign = l < hl ? -1.f : 1.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float other = __shfl_sync(0xffffffffu, x[i], partner, kRowLanes);
      // past the rotated elements 0 * infinity would be NaN
      x[i] = l < 2 * hl ? x[i] * t.c[i] + sign * other * t.s[i] : x[i];
    }
  }
  if (!t.in) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.f;
  }
}

}  // namespace qsa
