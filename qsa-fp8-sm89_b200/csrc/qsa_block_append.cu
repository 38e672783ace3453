// Appends new keys and values to the block-scaled paged caches; the keys are
// normed and rotated on the way.
//
//   s = max(s_old if the block keeps earlier tokens, max|x| / 448, 2^-126)
//   new rows: e4m3fn(x / s)      kept rows: e4m3fn(code * (s_old / s))
//
// Bound by HBM: a new row is read once (128 elements) and written once (128
// bytes). A block belongs to one request, so one group of warps owns a (block,
// KV head, K or V) and needs no atomics. A warp holds 16 rows of it in
// registers as fp32, a half warp a row (qsa_rope.cuh), from their loads over
// the block's maximum to their stores: one warp for blocks of up to 16 tokens,
// 2 to 8 for up to 128, which share their maxima in shared memory. Larger
// blocks are read twice, 128 rows at a time.
//
// Entry e has at most floor(n_e / B) + 2 blocks of B tokens, so its blocks get
// the slots floor(cu[e] / B) + 2e + j, which never overlap and end below
// tokens / B + 2 entries: the grid is known without reading the device, and a
// slot finds its entry by a search that splits the list 32 ways a step. The new
// rows' loads go out before the block table is read, and a kept block's codes
// before it is known whether its scale grows.
#include <cfloat>

#include "qsa_common.cuh"
#include "qsa_rope.cuh"

namespace qsa {
namespace {

constexpr int kApWarps = 8;
constexpr int kApSteps = 8;                   // row pairs that a warp holds
constexpr int kApRows = 2 * kApSteps;
constexpr float kMinScale = 1.17549435e-38f;  // 2^-126: 1 / scale stays finite

__device__ __forceinline__ uint32_t to_e4m3(const float* x) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[0], x[1]), __NV_SATFINITE, __NV_E4M3) |
         (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[2], x[3]), __NV_SATFINITE, __NV_E4M3) << 16;
}

struct ApBlock {
  int64_t token;  // first new token of the block
  int64_t pos;    // its logical position
  int kept;       // rows of the block before it that stay
  int count;      // new rows, 0: there is no such block
  int64_t req;    // block-table row
};

// The block of a slot, but for its page.
__device__ __forceinline__ ApBlock find_block(const BlockAppendParams& p, int64_t slot, int lane) {
  const int B = p.block_size;
  int e = 0;
  int64_t j = 0, first = slot, count = 1;
  if (p.cu_tokens) {
    // the last entry whose first slot, floor(cu[e] / B) + 2e, is <= slot
    for (int n = p.entries; n > 1;) {
      const int step = (n + 31) / 32;
      const int at = e + lane * step;
      const bool below = lane * step < n && (int64_t)(__ldg(p.cu_tokens + at) / B) + 2 * (int64_t)at <= slot;
      const int k = max(__popc(__ballot_sync(0xffffffffu, below)) - 1, 0);
      e += k * step;
      n = min(step, n - k * step);
    }
    first = min(max(__ldg(p.cu_tokens + e), 0), p.tokens);
    count = min(max(__ldg(p.cu_tokens + e + 1), 0), p.tokens) - first;
    j = slot - (first / B + 2 * (int64_t)e);
  } else {
    e = (int)slot;
  }
  const int64_t start = __ldg(p.starts + e);
  ApBlock b;
  b.req = p.reqs ? __ldg(p.reqs + e) : e;
  const int64_t base = (start / B + j) * B;  // logical position of the block's row 0
  const int64_t from = max(base, start), to = min(base + B, start + count);
  b.token = first + (from - start);
  b.pos = from;
  b.kept = (int)(from - base);
  b.count = count <= 0 || j < 0 || start < 0 || from >= to ? 0 : (int)(to - from);
  return b;
}

// Physical slot of the block's row 0, -1 where it has no page.
__device__ __forceinline__ int64_t block_slot(const BlockAppendParams& p, const ApBlock& b) {
  const int64_t base = b.pos - b.kept;
  const int64_t lp = base / p.page_size;
  if (b.count == 0 || b.req < 0 || b.req >= p.num_reqs || lp >= p.pages_per_req) return -1;
  const int64_t page = __ldg(p.btable + b.req * p.btable_stride + lp);
  return page < 0 || page >= p.num_pages ? -1 : page * p.page_size + base % p.page_size;
}

// kHold: the group's warps hold all rows of a block.
template <typename T, bool kHold>
__global__ void __launch_bounds__(32 * kApWarps, 2)
    qsa_block_append_kernel(const __grid_constant__ BlockAppendParams p, int64_t items, int group) {
  __shared__ float tops[kApWarps];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int l = lane % kRowLanes, side = lane / kRowLanes;
  const int64_t item = (int64_t)blockIdx.x * (kApWarps / group) + warp / group;
  // neighbours are the heads of one block: their rows of the rotation's table
  // are the same
  const int g = (int)(item % p.num_kv_heads);
  const bool is_k = item / p.num_kv_heads % 2 == 0;
  ApBlock b = {};
  if (item < items) b = find_block(p, item / p.num_kv_heads / 2, lane);
  const bool norm = is_k && p.k_weight, turn = is_k && p.rope.table;
  RopeParams rope = p.rope;
  if (!turn) rope.table = nullptr;
  const Pieces pieces = lane_pieces(rope, l);
  const T* src = static_cast<const T*>(is_k ? p.k : p.v) + (int64_t)g * kHeadDim;
  float w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = 1.f;
  if (norm) load_weight8(p.k_weight, p.weight_dtype, pieces, w);

  // Row pairs row0, row0 + 2, ... of the block's new rows: zeros past the last
  const int row0 = warp % group * kApRows + side;
  auto load = [&](int first, Raw8<T> (&raw)[kApSteps]) {
#pragma unroll
    for (int i = 0; i < kApSteps; ++i) {
      raw[i] = {};
      if (first + 2 * i < b.count) load8(src + (b.token + first + 2 * i) * p.token_stride, pieces, raw[i]);
    }
  };
  auto value = [&](int row, const Raw8<T>& raw, float (&x)[8]) {
    widen8(raw, x);
    if (norm) rms_norm8(x, w, p.eps);
    if (turn && row < b.count) {
      Turn4 t;
      load_turn4(rope, b.token + row, b.pos + row, l, t);
      rotate8(rope, t, x);
    }
  };
  // the largest |x|, over the group; NaN counts for none, infinity neither
  auto largest = [&](float top, bool again) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (group > 1) {
      if (again) __syncthreads();
      if (lane == 0) tops[warp] = top;
      __syncthreads();
      for (int i = 0; i < group; ++i) top = fmaxf(top, tops[warp / group * group + i]);
    }
    return top;
  };

  Raw8<T> raw[kApSteps];
  load(row0, raw);
  const int64_t slot = block_slot(p, b);
  const int64_t step = (int64_t)p.num_kv_heads * kHeadDim;
  uint8_t* dst = (is_k ? p.k_cache : p.v_cache) + max(slot, (int64_t)0) * step + (int64_t)g * kHeadDim;
  float* scale = (is_k ? p.k_scales : p.v_scales) + max(slot, (int64_t)0) / p.block_size * p.num_kv_heads + g;
  const int kept = slot < 0 ? 0 : b.kept;
  const float old = kept > 0 ? *scale : 0.f;
  uint2 codes[kApSteps];  // of kept rows
  if (kHold && kept > 0) {
#pragma unroll
    for (int i = 0; i < kApSteps; ++i)
      if (row0 + 2 * i < kept) codes[i] = *reinterpret_cast<const uint2*>(dst + (row0 + 2 * i) * step + 8 * l);
  }

  float x[kHold ? kApSteps : 1][8];
  float top = 0.f;
  if constexpr (kHold) {
#pragma unroll
    for (int i = 0; i < kApSteps; ++i) {
      value(row0 + 2 * i, raw[i], x[i]);
#pragma unroll
      for (int d = 0; d < 8; ++d) top = fmaxf(top, fabsf(x[i][d]));
    }
  } else {
    for (int first = row0; first - row0 < b.count; first += kApWarps * kApRows) {
      if (first > row0) load(first, raw);
#pragma unroll
      for (int i = 0; i < kApSteps; ++i) {
        value(first + 2 * i, raw[i], x[0]);
#pragma unroll
        for (int d = 0; d < 8; ++d)
          if (fabsf(x[0][d]) <= FLT_MAX) top = fmaxf(top, fabsf(x[0][d]));
      }
    }
  }
  top = largest(top, false);
  const bool infinite = top > FLT_MAX;
  if constexpr (kHold) {
    if (__syncthreads_or(infinite)) {  // rare, and then for the whole CTA
      float finite = 0.f;
#pragma unroll
      for (int i = 0; i < kApSteps; ++i)
#pragma unroll
        for (int d = 0; d < 8; ++d)
          if (fabsf(x[i][d]) <= FLT_MAX) finite = fmaxf(finite, fabsf(x[i][d]));
      top = largest(finite, true);
    }
  }
  if (slot < 0) return;
  const float s = fmaxf(old, fmaxf(__fdiv_rn(top, 448.f), kMinScale));
  const float inv = __fdiv_rn(1.f, s);
  // x / s rounded to nearest: a product with the reciprocal and a residual step
  // (an IEEE division for each element costs several times as much; without
  // the step, ties of x / s fall to the other side more often)
  auto store = [&](int row, float (&v)[8]) {
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      const float q = v[d] * inv;
      const float r = fmaf(-q, s, v[d]);
      v[d] = fabsf(q) <= FLT_MAX ? fmaf(r, inv, q) : q;
    }
    uint8_t* to = dst + (b.kept + row) * step;
    const uint32_t u0 = to_e4m3(v), u1 = to_e4m3(v + 4);
    if (pieces.b == pieces.a + 4) {
      *reinterpret_cast<uint2*>(to + pieces.a) = make_uint2(u0, u1);
    } else {
      *reinterpret_cast<uint32_t*>(to + pieces.a) = u0;
      *reinterpret_cast<uint32_t*>(to + pieces.b) = u1;
    }
  };
  if constexpr (kHold) {
#pragma unroll
    for (int i = 0; i < kApSteps; ++i)
      if (row0 + 2 * i < b.count) store(row0 + 2 * i, x[i]);
  } else {
    for (int first = row0; first - row0 < b.count; first += kApWarps * kApRows) {
      load(first, raw);
#pragma unroll
      for (int i = 0; i < kApSteps; ++i) {
        value(first + 2 * i, raw[i], x[0]);
        if (first + 2 * i < b.count) store(first + 2 * i, x[0]);
      }
    }
  }
  if (old == s) return;
  const float ratio = __fdiv_rn(old, s);
  auto rescale = [&](int row, uint2 was) {
    const uint32_t c[2] = {was.x, was.y};
    float v[8];
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const float2 f = e4m3x2_to_f32x2((uint16_t)(c[d / 2] >> (16 * (d % 2))));
      v[2 * d] = f.x * ratio;
      v[2 * d + 1] = f.y * ratio;
    }
    *reinterpret_cast<uint2*>(dst + row * step + 8 * l) = make_uint2(to_e4m3(v), to_e4m3(v + 4));
  };
  if constexpr (kHold) {
#pragma unroll
    for (int i = 0; i < kApSteps; ++i)
      if (row0 + 2 * i < kept) rescale(row0 + 2 * i, codes[i]);
  } else {
    for (int first = row0; first < kept; first += kApWarps * kApRows)
#pragma unroll
      for (int i = 0; i < kApSteps; ++i)
        if (first + 2 * i < kept)
          rescale(first + 2 * i, *reinterpret_cast<const uint2*>(dst + (first + 2 * i) * step + 8 * l));
  }
  if (warp % group == 0 && lane == 0) *scale = s;
}

template <typename T>
cudaError_t launch(const BlockAppendParams& p, int64_t items, cudaStream_t stream) {
  int group = 1;
  while (group < kApWarps && group * kApRows < p.block_size) group *= 2;
  const int64_t grid = (items * group + kApWarps - 1) / kApWarps;
  if (grid > 0x7fffffffll) return cudaErrorInvalidValue;
  if (p.block_size <= kApWarps * kApRows)
    qsa_block_append_kernel<T, true><<<(unsigned)grid, 32 * kApWarps, 0, stream>>>(p, items, group);
  else
    qsa_block_append_kernel<T, false><<<(unsigned)grid, 32 * kApWarps, 0, stream>>>(p, items, group);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_block_append(const BlockAppendParams& p, cudaStream_t stream) {
  const int64_t slots = p.cu_tokens ? (int64_t)(p.tokens / p.block_size) + 2 * (int64_t)p.entries : p.entries;
  const int64_t items = slots * p.num_kv_heads * 2;
  switch (p.dtype) {
    case QSA_B200_DTYPE_BF16: return launch<__nv_bfloat16>(p, items, stream);
    case QSA_B200_DTYPE_F16: return launch<__half>(p, items, stream);
    default: return launch<float>(p, items, stream);
  }
}

}  // namespace qsa
