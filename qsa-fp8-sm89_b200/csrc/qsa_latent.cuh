// Device helpers of the latent cache's kernels: the tokens that a call's entries
// name, and their places in the cache.
#pragma once
#include <atomic>

#include "qsa_common.cuh"
#include "qsa_internal.h"

namespace qsa {

// Slot of a request's logical position, -1 outside the block table or the cache.
__device__ __forceinline__ int latent_slot(const LatentCache& c, int64_t req, int t) {
  if (t < 0) return -1;
  const uint32_t lp = __umulhi(2u * (uint32_t)t, c.page_mul) >> c.page_shift;
  if ((int)lp >= c.pages_per_req) return -1;
  const int page = __ldg(c.btable + req * c.btable_stride + lp);
  return page >= 0 && page < c.num_pages ? page * c.page_size + (t - (int)lp * c.page_size) : -1;
}

// The places of `count` tokens from `first_token`, a lane each, found by the whole warp:
// slot (-1: none) and logical position; false where no entry names the token.
__device__ __forceinline__ bool latent_place(const LatentCache& c, const LatentTokens& list, int first_token, int count, int lane,
                                             int& slot, int& pos) {
  slot = -1, pos = -1;
  const int token = first_token + lane;
  int e = token, first = token, lo = 0;
  if (list.cu_tokens) {
    // the last entry that begins at or before the first token, by 32 probes at a time
    int hi = list.entries;
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32;
      const int at = lo + lane * step;
      const int begun = __popc(__ballot_sync(0xffffffffu, at < hi && __ldg(list.cu_tokens + at) <= first_token));
      hi = min(hi, lo + max(begun, 1) * step);
      lo += max(begun - 1, 0) * step;
    }
  }
  if (lane >= count || token >= list.tokens) return false;
  if (list.cu_tokens) {
    e = lo;
    while (e + 1 < list.entries && __ldg(list.cu_tokens + e + 1) <= token) ++e;
    first = __ldg(list.cu_tokens + e);
    if (token < first || token >= __ldg(list.cu_tokens + e + 1)) return false;
  }
  const int start = __ldg(list.starts + e);
  const int64_t req = list.reqs ? (int64_t)__ldg(list.reqs + e) : (int64_t)e;
  const int64_t at = (int64_t)start + (token - first);
  if (start >= 0 && req >= 0 && req < c.num_reqs && at <= 0x7fffffffll) {
    pos = (int)at;
    slot = latent_slot(c, req, pos);
  }
  return true;
}

// Four elements of a type, as they were loaded, widened to fp32.
__device__ __forceinline__ void latent_widen(const uint4& v, float (&x)[4], float) {
  x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void latent_widen(const uint2& v, float (&x)[4], __nv_bfloat16) {
  x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xffff0000u);
  x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xffff0000u);
}
__device__ __forceinline__ void latent_widen(const uint2& v, float (&x)[4], __half) {
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}
template <typename T>
__device__ __forceinline__ void latent_load4(const T* at, float (&x)[4]) {
  using Word = typename std::conditional<sizeof(T) == 4, uint4, uint2>::type;
  latent_widen(__ldg(reinterpret_cast<const Word*>(at)), x, T());
}
__device__ __forceinline__ float latent_to_float(float x) { return x; }
__device__ __forceinline__ float latent_to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float latent_to_float(__half x) { return __half2float(x); }

// The largest of three, NaN where one is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// SMs of the current device.
inline int latent_sm_count() {
  static std::atomic<int> known[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  int n = known[dev & 63].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) n = 148;
    known[dev & 63].store(n, std::memory_order_relaxed);
  }
  return n;
}

}  // namespace qsa
