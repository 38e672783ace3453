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

// A token's place, found by the whole warp: its slot (-1: none) and logical
// position; false where no entry names it.
__device__ __forceinline__ bool latent_place(const LatentCache& c, const LatentTokens& list, int token, int lane, int& slot,
                                             int& pos) {
  int e = token, first = token;
  if (list.cu_tokens) {
    // the last entry that begins at or before the token, by 32 probes at a time
    int lo = 0, hi = list.entries;
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32;
      const int at = lo + lane * step;
      const int begun = __popc(__ballot_sync(0xffffffffu, at < hi && __ldg(list.cu_tokens + at) <= token));
      hi = min(hi, lo + max(begun, 1) * step);
      lo += max(begun - 1, 0) * step;
    }
    e = lo;
    first = __ldg(list.cu_tokens + e);
    if (token < first || token >= __ldg(list.cu_tokens + e + 1)) return false;
  }
  slot = -1, pos = -1;
  const int start = __ldg(list.starts + e);
  const int64_t req = list.reqs ? (int64_t)__ldg(list.reqs + e) : (int64_t)e;
  const int64_t at = (int64_t)start + (token - first);
  if (start >= 0 && req >= 0 && req < c.num_reqs && at <= 0x7fffffffll) {
    pos = (int)at;
    slot = latent_slot(c, req, pos);
  }
  return true;
}

// Elements of `T` in the words of a load, widened to fp32.
__device__ __forceinline__ void latent_load4(const float* at, float (&x)[4]) {
  const float4 v = __ldg(reinterpret_cast<const float4*>(at));
  x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}
__device__ __forceinline__ void latent_load4(const __nv_bfloat16* at, float (&x)[4]) {
  const uint2 v = __ldg(reinterpret_cast<const uint2*>(at));
  x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xffff0000u);
  x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xffff0000u);
}
__device__ __forceinline__ void latent_load4(const __half* at, float (&x)[4]) {
  const uint2 v = __ldg(reinterpret_cast<const uint2*>(at));
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}
__device__ __forceinline__ float latent_to_float(float x) { return x; }
__device__ __forceinline__ float latent_to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float latent_to_float(__half x) { return __half2float(x); }

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
