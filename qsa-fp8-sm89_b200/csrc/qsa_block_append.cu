// Appends new keys and values to the block-scaled paged caches; the keys are
// normed and rotated on the way.
//
//   s = max(s_old if the block keeps earlier tokens, max|x| / 448, 2^-126)
//   new rows: e4m3fn(x / s)      kept rows: e4m3fn(code * (s_old / s))
//
// A block belongs to one request, so one warp owns a (block, KV head, K or V)
// and needs no atomics: it reads the block's new rows, two at a time (a half
// warp each, qsa_rope.cuh), for their maximum, and a second time to store
// them.
//
// Entry e has at most floor(n_e / B) + 2 blocks of B tokens, so its blocks get
// the slots floor(cu[e] / B) + 2e + j, which never overlap and end below
// tokens / B + 2 entries: the grid is known without reading the device, and a
// slot finds its entry by bisection.
#include <cfloat>

#include "qsa_common.cuh"
#include "qsa_rope.cuh"

namespace qsa {
namespace {

constexpr int kApWarps = 8;
constexpr float kMinScale = 1.17549435e-38f;  // 2^-126: 1 / scale stays finite

// x / s rounded to nearest: one product with the reciprocal and one residual
// step (an IEEE division per element would cost several times as much).
__device__ __forceinline__ float divide(float x, float s, float inv) {
  const float q = x * inv;
  const float r = fmaf(-q, s, x);
  return fabsf(q) < FLT_MAX ? fmaf(r, inv, q) : q;
}

__device__ __forceinline__ uint2 to_e4m3(const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[2 * i], x[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

struct ApBlock {
  int64_t token;  // first new token of the block
  int64_t pos;    // its logical position
  int kept;       // rows of the block before it that stay
  int count;      // new rows
  int64_t slot;   // physical slot of the block's row 0
};

// The block of a slot; false when there is none.
__device__ __forceinline__ bool find_block(const BlockAppendParams& p, int64_t slot, ApBlock& b) {
  const int B = p.block_size;
  int e;
  int64_t j, first, count;
  if (p.cu_tokens) {
    int lo = 0, hi = p.entries - 1;  // the last entry whose first slot is <= slot
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((int64_t)(__ldg(p.cu_tokens + mid) / B) + 2 * (int64_t)mid <= slot) lo = mid;
      else hi = mid - 1;
    }
    e = lo;
    first = min(max(__ldg(p.cu_tokens + e), 0), p.tokens);
    count = min(max(__ldg(p.cu_tokens + e + 1), 0), p.tokens) - first;
    j = slot - (first / B + 2 * (int64_t)e);
  } else {
    e = (int)slot;
    first = slot;
    count = 1;
    j = 0;
  }
  const int64_t start = __ldg(p.starts + e);
  const int64_t req = p.reqs ? __ldg(p.reqs + e) : e;
  if (count <= 0 || j < 0 || start < 0 || req < 0 || req >= p.num_reqs) return false;
  const int64_t base = (start / B + j) * B;  // logical position of the block's row 0
  const int64_t from = max(base, start), to = min(base + B, start + count);
  if (from >= to) return false;
  const int64_t lp = base / p.page_size;
  if (lp >= p.pages_per_req) return false;
  const int64_t page = __ldg(p.btable + req * p.btable_stride + lp);
  if (page < 0 || page >= p.num_pages) return false;
  b.token = first + (from - start);
  b.pos = from;
  b.kept = (int)(from - base);
  b.count = (int)(to - from);
  b.slot = page * p.page_size + base % p.page_size;
  return true;
}

template <typename T>
__global__ void __launch_bounds__(32 * kApWarps) qsa_block_append_kernel(const __grid_constant__ BlockAppendParams p,
                                                                         int64_t items) {
  const int lane = threadIdx.x % 32;
  const int l = lane % kRowLanes, side = lane / kRowLanes;
  const int64_t item = (int64_t)blockIdx.x * kApWarps + threadIdx.x / 32;
  if (item >= items) return;
  const int g = (int)(item / 2 % p.num_kv_heads);
  const bool is_k = item % 2 == 0;
  ApBlock b;
  if (!find_block(p, item / 2 / p.num_kv_heads, b)) return;
  const T* src = static_cast<const T*>(is_k ? p.k : p.v) + (int64_t)g * kHeadDim + 8 * l;
  uint8_t* cache = is_k ? p.k_cache : p.v_cache;
  float* scale = (is_k ? p.k_scales : p.v_scales) + b.slot / p.block_size * p.num_kv_heads + g;
  const float old = b.kept > 0 ? *scale : 0.f;
  float w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = 1.f;
  const bool norm = is_k && p.k_weight, turn = is_k && p.rope.table;
  if (norm) load_weight8(p.k_weight, p.weight_dtype, l, w);

  // new row i of the block (i < count, else row 0's values: every lane goes
  // through the exchanges)
  auto row = [&](int i, float (&x)[8]) {
    const int64_t t = b.token + (i < b.count ? i : 0);
    Raw8<T> raw;
    load8(src + t * p.token_stride, raw);
    widen8(raw, x);
    if (norm) rms_norm8(x, w, p.eps);
    if (turn) {
      Turn8 tr;
      load_turn8(p.rope, t, b.pos + (t - b.token), l, tr);
      rotate8(p.rope, tr, l, x);
    }
  };
  float top = 0.f;
  for (int i = side; i - side < b.count; i += 2) {
    float x[8];
    row(i, x);
#pragma unroll
    for (int d = 0; d < 8; ++d) top = fabsf(x[d]) <= FLT_MAX ? fmaxf(top, fabsf(x[d])) : top;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float s = fmaxf(old, fmaxf(__fdiv_rn(top, 448.f), kMinScale));
  const float inv = __fdiv_rn(1.f, s);
  const int64_t step = (int64_t)p.num_kv_heads * kHeadDim;
  uint8_t* dst = cache + b.slot * step + (int64_t)g * kHeadDim + 8 * l;
  for (int i = side; i - side < b.count; i += 2) {
    float x[8];
    row(i, x);
#pragma unroll
    for (int d = 0; d < 8; ++d) x[d] = divide(x[d], s, inv);
    if (i < b.count) *reinterpret_cast<uint2*>(dst + (b.kept + i) * step) = to_e4m3(x);
  }
  if (old != s) {
    const float ratio = __fdiv_rn(old, s);
    for (int i = side; i < b.kept; i += 2) {
      const uint2 was = *reinterpret_cast<const uint2*>(dst + i * step);
      const uint32_t c[2] = {was.x, was.y};
      float x[8];
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const float2 f = e4m3x2_to_f32x2((uint16_t)(c[d / 2] >> (16 * (d % 2))));
        x[2 * d] = f.x * ratio;
        x[2 * d + 1] = f.y * ratio;
      }
      *reinterpret_cast<uint2*>(dst + i * step) = to_e4m3(x);
    }
    if (lane == 0) *scale = s;
  }
}

}  // namespace

cudaError_t launch_block_append(const BlockAppendParams& p, cudaStream_t stream) {
  const int64_t slots = p.cu_tokens ? (int64_t)(p.tokens / p.block_size) + 2 * (int64_t)p.entries : p.entries;
  const int64_t items = slots * p.num_kv_heads * 2;
  const int64_t grid = (items + kApWarps - 1) / kApWarps;
  if (grid > 0x7fffffffll) return cudaErrorInvalidValue;
  switch (p.dtype) {
    case QSA_B200_DTYPE_BF16: qsa_block_append_kernel<__nv_bfloat16><<<(unsigned)grid, 32 * kApWarps, 0, stream>>>(p, items); break;
    case QSA_B200_DTYPE_F16: qsa_block_append_kernel<__half><<<(unsigned)grid, 32 * kApWarps, 0, stream>>>(p, items); break;
    default: qsa_block_append_kernel<float><<<(unsigned)grid, 32 * kApWarps, 0, stream>>>(p, items); break;
  }
  return cudaGetLastError();
}

}  // namespace qsa
