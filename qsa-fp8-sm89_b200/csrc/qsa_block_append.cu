// Appends new keys and values to the block-scaled paged caches; the keys are
// normed and rotated on the way.
//
//   s = max(s_old if the block keeps earlier tokens, max|x| / 448, 2^-126)
//   new rows: e4m3fn(x / s)      kept rows: e4m3fn(code * (s_old / s))
//
// Bound by HBM: a new row is read once (128 elements) and written once (128
// bytes). A block belongs to one request, so one group of warps owns a (block,
// KV head, K or V) and needs no atomics. A warp holds 8 rows of it in registers
// as fp32, a half warp a row (qsa_rope.cuh), from their loads over the block's
// maximum to their stores; up to 8 warps share a block of up to 64 tokens and
// exchange their maxima in shared memory. Larger blocks are read twice, 64 rows
// at a time; blocks of up to 4 tokens go several to a warp, each row with the
// scale of its own block. A group goes through up to 8 heads of its block: where it lies and
// the cosines and sines of its rows are looked up once for them, and a head's
// rows are loaded while the one before is worked on.
//
// Entry e has at most floor(n_e / B) + 2 blocks of B tokens, so its blocks get
// the slots floor(cu[e] / B) + 2e + j, which never overlap and end below
// tokens / B + 2 entries: the grid is known without reading the device, and a
// slot finds its entry by a search that splits the list 32 ways a step. The new
// rows' loads go out before the block table is read, and a kept block's codes
// before it is known whether its scale grows.
//
// Prompts of 52224 tokens in all, 8 KV heads, blocks of 64: 348 MB in 96 us, 3.6
// TB/s; 37 % of DRAM, 59 % of the issue slots with 16 warps an SM (128
// registers): what bounds it is the arithmetic's latency. Without norm and rotation
// 71 us. The steps: two passes over the rows 348; rows held in registers 299;
// loads without guards, the pairing known at compile time 158; no IEEE division,
// one redux a maximum 139; rows through cp.async a head ahead 108 (two or three
// heads ahead: the same); the norm's exchanges side by side 104; no branches
// around whole blocks 98; packed fp32 arithmetic 96. 3 CTAs of 80 registers an SM
// pay only where nothing rotates (76 against 79).
// 256 entries of one token: 3.5 us one after the other in a graph, 5.7 where every
// block's scale grows and its kept rows are rescaled; with a cold L2 8 to 10, and
// 12. Blocks above 64 tokens read twice: 200 us;
// blocks of 1 token 125 us, of 2 to 4 tokens 163 (each row's scale, its page and
// its place are its own, so the registers hold no row ahead).
#include <atomic>
#include <cfloat>

#include "qsa_common.cuh"
#include "qsa_rope.cuh"

namespace qsa {
namespace {

constexpr int kApWarps = 8;
constexpr int kApSteps = 4;                   // row pairs that a warp holds
constexpr int kApRows = 2 * kApSteps;
constexpr int kApStages = 2;                  // heads whose rows are under way or at hand
constexpr int kApHeads = 8;                   // heads that a group goes through, at most
constexpr float kMinScale = 1.17549435e-38f;  // 2^-126: 1 / scale stays finite

// x / s, nearly always rounded to nearest, inv = 1 / s within a few ulp: a product
// and one Newton step on the residual x - q s. (An IEEE division for each element costs several times as
// much; without the step, ties of x / s fall to the other side more often.)
__device__ __forceinline__ float divide(float x, float s, float inv) {
  const float q = x * inv;
  return fmaf(fmaf(-q, s, x), inv, q);
}

__device__ __forceinline__ uint32_t to_e4m3(const float* x) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[0], x[1]), __NV_SATFINITE, __NV_E4M3) |
         (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[2], x[3]), __NV_SATFINITE, __NV_E4M3) << 16;
}

// Whole numbers stay in 32 bits (a 64-bit division is over 100 instructions,
// and a warp makes several): logical positions are below 2^32 where a start
// and a count of tokens, both below 2^31, are added.
struct ApBlock {
  int token;     // first new token of the block
  uint32_t pos;  // its logical position
  int kept;      // rows of the block before it that stay
  int count;     // new rows, 0: there is no such block
  int req;       // block-table row
};

// The block of a slot, but for its page. B: tokens of a block.
__device__ __forceinline__ ApBlock find_block(const BlockAppendParams& p, uint32_t slot, int lane, uint32_t B) {
  int e = 0;
  // the last entry whose first slot, floor(cu[e] / B) + 2e, is <= slot
  for (int n = p.entries; n > 1;) {
    const int step = (n + 31) / 32;
    const int at = e + lane * step;
    const bool below = lane * step < n && (uint32_t)max(__ldg(p.cu_tokens + at), 0) / B + 2u * at <= slot;
    const int k = max(__popc(__ballot_sync(0xffffffffu, below)) - 1, 0);
    e += k * step;
    n = min(step, n - k * step);
  }
  const int first = min(max(__ldg(p.cu_tokens + e), 0), p.tokens);
  const int count = min(max(__ldg(p.cu_tokens + e + 1), 0), p.tokens) - first;
  const uint32_t slot0 = (uint32_t)first / B + 2u * e;
  const bool is = count > 0 && slot >= slot0;
  const uint32_t j = slot - slot0;
  const int start = __ldg(p.starts + e);
  ApBlock b;
  b.req = p.reqs ? __ldg(p.reqs + e) : e;
  const uint32_t lead = (uint32_t)max(start, 0) % B;  // rows of the first block that stay
  const uint32_t skip = j == 0 ? 0 : j * B - lead;    // new tokens before this block
  b.kept = j == 0 ? (int)lead : 0;
  b.token = first + (int)skip;
  b.pos = (uint32_t)start + skip;
  b.count = is && start >= 0 && j <= (uint32_t)count / B + 1 && skip < (uint32_t)count
                ? (int)min(B - (uint32_t)b.kept, (uint32_t)count - skip)
                : 0;
  return b;
}

// Physical page of a block, -1 where it has none; off: its row 0 in the page.
__device__ __forceinline__ int block_page(const BlockAppendParams& p, const ApBlock& b, uint32_t& off) {
  const uint32_t base = b.pos - b.kept;
  const uint32_t lp = base / (uint32_t)p.page_size;
  off = base - lp * p.page_size;
  if (b.count == 0 || b.req < 0 || b.req >= p.num_reqs || lp >= (uint32_t)p.pages_per_req) return -1;
  const int page = __ldg(p.btable + b.req * p.btable_stride + lp);
  return page < 0 || page >= p.num_pages ? -1 : page;
}

// Eight values over their scale, as codes.
__device__ __forceinline__ uint2 quantise8(float (&v)[8], float s, float inv, bool infinite) {
  if (infinite) {  // an infinity's residual would be NaN
#pragma unroll
    for (int d = 0; d < 8; ++d) v[d] = fabsf(v[d]) > FLT_MAX ? v[d] : divide(v[d], s, inv);
  } else {
    const uint64_t by = pair2(inv, inv), back = pair2(-s, -s);  // divide()'s steps, two at a time
#pragma unroll
    for (int d = 0; d < 8; d += 2) {
      const uint64_t x = pair2(v[d], v[d + 1]), q = mul2(x, by);
      unpair2(fma2(fma2(q, back, x), by, q), v[d], v[d + 1]);
    }
  }
  return make_uint2(to_e4m3(v), to_e4m3(v + 4));
}

// Eight codes over a larger scale.
__device__ __forceinline__ uint2 rescale8(uint2 was, float ratio) {
  const uint32_t c[2] = {was.x, was.y};
  float v[8];
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const float2 f = e4m3x2_to_f32x2((uint16_t)(c[d / 2] >> (16 * (d % 2))));
    v[2 * d] = f.x * ratio;
    v[2 * d + 1] = f.y * ratio;
  }
  return make_uint2(to_e4m3(v), to_e4m3(v + 4));
}

__device__ __forceinline__ void store_codes(uint8_t* row, Pieces at, bool halves, uint2 codes) {
  if (halves) {
    *reinterpret_cast<uint32_t*>(row + at.a) = codes.x;
    *reinterpret_cast<uint32_t*>(row + at.b) = codes.y;
  } else {  // the two pieces are one
    *reinterpret_cast<uint2*>(row + at.a) = codes;
  }
}

// One group's blocks: see the kernel. kTurn: the rows are rotated.
template <typename T, bool kHold, int kTurn>
__device__ __forceinline__ void append_block(const BlockAppendParams& p, const ApBlock& b, bool is_k, int g0, int group,
                                             int per, float (*tops)[kApWarps], T* ring) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int l = lane % kRowLanes, side = lane / kRowLanes;
  const bool norm = is_k && p.k_weight;
  const int turning = kTurn == kPlain ? 0 : p.rope.rotary >> 3;  // lanes that hold rotated elements
  const bool halves = kTurn == kHalves && l < turning;
  const Pieces pieces = lane_pieces<kTurn>(l, p.rope.rotary);
  const T* src = static_cast<const T*>(is_k ? p.k : p.v);

  // The half warp's rows of the block's new ones: row0, row0 + 2, ... Past the
  // last row the last one is read again, which changes no maximum.
  const int row0 = warp % group * kApRows + side;
  auto clamped = [&](int row) { return b.count > 0 ? b.token + min(row, b.count - 1) : 0; };
  // without halves the two pieces are one
  auto load_row = [&](const T* row, Raw8<T>& r) {
    if constexpr (kTurn == kHalves || sizeof(T) == 4) {
      load8(row, pieces, r);
    } else {
      const uint4 v = *reinterpret_cast<const uint4*>(row + 8 * l);
      r.a = make_uint2(v.x, v.y), r.b = make_uint2(v.z, v.w);
    }
  };
  const T* rows[kApSteps];
#pragma unroll
  for (int i = 0; i < kApSteps; ++i) rows[i] = src + (int64_t)clamped(row0 + 2 * i) * p.token_stride;
  // head h's rows into its stage of the warp's ring
  auto fetch = [&](int h) {
    if (h < per) {
      const int g = min(g0 + h, p.num_kv_heads - 1);
      T* to = ring + (h % kApStages * kApRows + side * kApSteps) * kHeadDim;
#pragma unroll
      for (int i = 0; i < kApSteps; ++i)
#pragma unroll
        for (int c = l * 16; c < kHeadDim * (int)sizeof(T); c += kRowLanes * 16)
          cp_async_16(smem_u32(to + i * kHeadDim) + c, reinterpret_cast<const uint8_t*>(rows[i] + g * kHeadDim) + c, 16u);
    }
    cp_async_commit();
  };
  Raw8<T> raw[kApSteps];
  if constexpr (kHold) {
#pragma unroll
    for (int h = 0; h < kApStages - 1; ++h) fetch(h);
  }
  float w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = 1.f;
  if (norm) load_weight8(p.k_weight, p.weight_dtype, pieces, w);
  uint32_t off;
  const int page = block_page(p, b, off);
  const int step = p.num_kv_heads * kHeadDim;
  uint8_t* cache = (is_k ? p.k_cache : p.v_cache) + ((int64_t)max(page, 0) * p.page_size + off) * step;
  float* scales = (is_k ? p.k_scales : p.v_scales) +
                  ((int64_t)max(page, 0) * (p.page_size / p.block_size) + off / (uint32_t)p.block_size) * p.num_kv_heads;
  const int kept = page < 0 ? 0 : b.kept;
  const bool all_rows = __all_sync(0xffffffffu, row0 + 2 * (kApSteps - 1) < b.count);

  auto turn_of = [&](int row, float4& c, float4& sn) {
    return load_turn(p.rope, clamped(row), b.pos + min(row, max(b.count - 1, 0)), l, turning, c, sn);
  };
  // the lane's cosines and sines of its rows wait in shared memory
  float4* turns = reinterpret_cast<float4*>(ring + kApStages * kApRows * kHeadDim) + lane;
  uint32_t inside = 0xffffffffu;  // bit i: row i's positions lie inside the table
  if (kTurn != kPlain && kHold) {
#pragma unroll
    for (int i = 0; i < kApSteps; ++i) {
      float4 c = {}, sn = {};
      if (!turn_of(row0 + 2 * i, c, sn)) inside &= ~(1u << i);
      turns[(2 * i) * 32] = c, turns[(2 * i + 1) * 32] = sn;
    }
  }
  auto normed = [&](float (&x)[kApSteps][8]) {
#pragma unroll
    for (int i = 0; i < kApSteps; ++i) widen8(raw[i], x[i]);
    if (norm) rms_norm8(x, w, p.eps);
  };
  auto row_top = [&](const float (&x)[8], float top) {  // NaN counts for none
#pragma unroll
    for (int d = 0; d < 8; ++d) top = fmaxf(top, fabsf(x[d]));
    return top;
  };
  auto finite_top = [&](const float (&x)[8], float top) {
#pragma unroll
    for (int d = 0; d < 8; ++d) top = fabsf(x[d]) <= FLT_MAX ? fmaxf(top, fabsf(x[d])) : top;
    return top;
  };
  // largest of values that are not negative: their bits order as they do
  auto warp_max = [](float v) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v))); };
  auto group_max = [&](int slot) { return warp_max(tops[slot][warp / group * group + lane % group]); };

#pragma unroll 1
  for (int h = 0; h < per; ++h) {  // as often for every warp of the CTA
    const int g = g0 + h;
    const bool live = page >= 0 && g < p.num_kv_heads;
    uint8_t* dst = cache + g * kHeadDim;
    float* scale = scales + g;
    const float old = live && kept > 0 ? *scale : 0.f;
    uint2 codes[kApSteps];  // of kept rows
    if (kHold && live && kept > 0) {
#pragma unroll
      for (int i = 0; i < kApSteps; ++i)
        if (row0 + 2 * i < kept) codes[i] = *reinterpret_cast<const uint2*>(dst + (int64_t)(row0 + 2 * i) * step + 8 * l);
    }
    float x[kApSteps][8];
    float top = 0.f;
    // larger blocks: the rows again, 64 at a time, through `with`
    auto each_row = [&](auto with) {
      for (int first = row0; first - row0 < b.count; first += kApWarps * kApRows) {
#pragma unroll
        for (int i = 0; i < kApSteps; ++i) {
          load_row(src + (int64_t)clamped(first + 2 * i) * p.token_stride + min(g, p.num_kv_heads - 1) * kHeadDim, raw[i]);
        }
        normed(x);
#pragma unroll
        for (int i = 0; i < kApSteps; ++i) {
          float4 c = {}, sn = {};
          const bool in = kTurn == kPlain || turn_of(first + 2 * i, c, sn);
          turn_row<kTurn>(c, sn, in, l < turning, x[i]);
          with(first + 2 * i, x[i]);
        }
      }
    };
    if constexpr (kHold) {
      cp_async_wait<kApStages - 2>();
      __syncwarp();  // the head's rows are there, and every lane has read the one's before
      fetch(h + kApStages - 1);
#pragma unroll
      for (int i = 0; i < kApSteps; ++i)
        load_row(ring + (h % kApStages * kApRows + side * kApSteps + i) * kHeadDim, raw[i]);
      normed(x);
      // all lanes hold rotated elements: nothing to choose between the rows
      auto turn = [&](bool turns_too) {
#pragma unroll
        for (int i = 0; i < kApSteps; ++i) {
          float4 c = {}, sn = {};
          if (kTurn != kPlain) c = turns[(2 * i) * 32], sn = turns[(2 * i + 1) * 32];
          turn_row<kTurn>(c, sn, (inside >> i) & 1u, turns_too, x[i]);
          top = row_top(x[i], top);
        }
      };
      if (turning == kRowLanes)
        turn(true);
      else
        turn(l < turning);
    } else {
      each_row([&](int, const float(&v)[8]) { top = finite_top(v, top); });
    }
    top = warp_max(top);
    bool infinite = top > FLT_MAX;
    if (group > 1) {
      // the buffers alternate: a warp that sets one again has passed the
      // barrier after the last readings of it
      if (lane == 0) tops[h % 2][warp] = top;
      infinite = __syncthreads_or(infinite);
      top = group_max(h % 2);
    }
    if constexpr (kHold) {
      if (infinite) {  // rare: once more, without the infinities
        top = 0.f;
#pragma unroll
        for (int i = 0; i < kApSteps; ++i) top = finite_top(x[i], top);
        top = warp_max(top);
        if (group > 1) {
          if (lane == 0) tops[2][warp] = top;
          __syncthreads();
          top = group_max(2);
        }
      }
    } else {
      infinite = true;  // not known: only the finite ones were looked at
    }
    if (!live) continue;
    const float s = fmaxf(old, fmaxf(divide(top, 448.f, 1.0f / 448.f), kMinScale));
    const float inv = __fdividef(1.f, s);  // s is below 2^126
    auto store = [&](int row, float (&v)[8]) {
      store_codes(dst + (int64_t)(b.kept + row) * step, pieces, halves, quantise8(v, s, inv, infinite));
    };
    if constexpr (kHold) {
      if (all_rows && !infinite) {
#pragma unroll
        for (int i = 0; i < kApSteps; ++i)
          store_codes(dst + (int64_t)(b.kept + row0 + 2 * i) * step, pieces, halves, quantise8(x[i], s, inv, false));
      } else {
#pragma unroll
        for (int i = 0; i < kApSteps; ++i)
          if (row0 + 2 * i < b.count) store(row0 + 2 * i, x[i]);
      }
    } else {
      each_row([&](int row, float(&v)[8]) {
        if (row < b.count) store(row, v);
      });
    }
    if (old == s) continue;
    const float ratio = divide(old, s, inv);
    auto rescale = [&](int row, uint2 was) {
      *reinterpret_cast<uint2*>(dst + (int64_t)row * step + 8 * l) = rescale8(was, ratio);
    };
    if constexpr (kHold) {
      if (kept > 0) {
#pragma unroll
        for (int i = 0; i < kApSteps; ++i)
          if (row0 + 2 * i < kept) rescale(row0 + 2 * i, codes[i]);
      }
    } else {
      for (int row = row0; row < kept; row += 2)
        if ((row - row0) / 2 % (kApWarps * kApSteps) < kApSteps)
          rescale(row, *reinterpret_cast<const uint2*>(dst + (int64_t)row * step + 8 * l));
    }
    __syncwarp();  // the old scale is read before a lane writes it
    if (warp % group == 0 && lane == 0) *scale = s;
  }
}

// Blocks of up to 4 tokens: a warp takes as many as its 8 rows hold, b being
// their run (a block of `run` = 8 / block_size * block_size tokens to
// find_block). Each row has a scale, and a page, of its own block.
// kSingle: blocks of one token, so that rows have nothing to do with each other
// and nothing is kept. turns: the lane's cosines and sines of its rows wait here.
template <typename T, int kTurn, bool kSingle>
__device__ __forceinline__ void append_packed(const BlockAppendParams& p, const ApBlock& b, bool is_k, int g0, int per,
                                              float4* turns) {
  const int lane = threadIdx.x % 32, l = lane % kRowLanes, side = lane / kRowLanes;
  const bool norm = is_k && p.k_weight;
  const int turning = kTurn == kPlain ? 0 : p.rope.rotary >> 3;
  const bool halves = kTurn == kHalves && l < turning;
  const Pieces pieces = lane_pieces<kTurn>(l, p.rope.rotary);
  const int B = p.block_size;
  const uint32_t half_mask = 0xffffu << (16 * side);
  if (b.count == 0 || b.req < 0 || b.req >= p.num_reqs) return;

  // the half warp's new rows side, side + 2, ...: where they are and go
  const T* src[kApSteps];
  int64_t row_at[kApSteps], scale_at[kApSteps];  // -1: not written
  uint32_t inside = 0xffffffffu;
  // byte i: which of the half warp's rows (bits 0 .. 3) and of the other's are
  // of row i's block; bit i: row i is its block's first new one, and its block
  // keeps rows (known ahead: a head's work has no divisions)
  uint32_t same = 0, begins = 0, leads = 0;
#pragma unroll
  for (int i = 0; i < kApSteps; ++i) {
    const int row = side + 2 * i, in_run = min(row, b.count - 1);
    const int token = b.token + in_run;
    const uint32_t pos = b.pos + in_run;
    src[i] = static_cast<const T*>(is_k ? p.k : p.v) + (int64_t)token * p.token_stride;
    const uint32_t lp = pos / (uint32_t)p.page_size, off = pos - lp * p.page_size;
    const int page = lp < (uint32_t)p.pages_per_req ? __ldg(p.btable + b.req * p.btable_stride + lp) : -1;
    const bool goes = row < b.count && page >= 0 && page < p.num_pages;
    row_at[i] = goes ? (int64_t)page * p.page_size + off : -1;
    scale_at[i] = goes ? (int64_t)page * (p.page_size / B) + off / (uint32_t)B : -1;
    if constexpr (!kSingle) {
      const int block = (b.kept + in_run) / B;
#pragma unroll
      for (int k = 0; k < kApSteps; ++k) {
        const int mine = (b.kept + min(side + 2 * k, b.count - 1)) / B, other = (b.kept + min(1 - side + 2 * k, b.count - 1)) / B;
        same |= (mine == block ? 1u : 0u) << (8 * i + k) | (other == block ? 1u : 0u) << (8 * i + 4 + k);
      }
      if (row == 0 || (b.kept + row) % B == 0) begins |= 1u << i;
      if (b.kept % B > 0 && block == b.kept / B) leads |= 1u << i;
    }
    if (kTurn != kPlain) {
      float4 c = {}, sn = {};
      if (!load_turn(p.rope, token, pos, l, turning, c, sn)) inside &= ~(1u << i);
      turns[(2 * i) * 32] = c, turns[(2 * i + 1) * 32] = sn;  // read by this lane alone
    }
  }
  float w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = 1.f;
  if (norm) load_weight8(p.k_weight, p.weight_dtype, pieces, w);
  const int lead = kSingle ? 0 : b.kept % B;  // rows that the first new row's block keeps
  uint8_t* cache = is_k ? p.k_cache : p.v_cache;
  float* scales = is_k ? p.k_scales : p.v_scales;

  const int g1 = min(g0 + per, p.num_kv_heads);
  Raw8<T> raw[kApSteps];
  auto load = [&](int g) {
#pragma unroll
    for (int i = 0; i < kApSteps; ++i) load8(src[i] + g * kHeadDim, pieces, raw[i]);
  };
  constexpr bool kAhead = kSingle;  // otherwise there are no registers for it
  if (kAhead) load(g0);
#pragma unroll 1
  for (int g = g0; g < g1; ++g) {
    if (!kAhead) load(g);
    float old[kApSteps];
    if constexpr (!kSingle) {
#pragma unroll
      for (int i = 0; i < kApSteps; ++i)
        old[i] = (leads >> i & 1u) && scale_at[i] >= 0 ? scales[scale_at[i] * p.num_kv_heads + g] : 0.f;
    }
    float x[kApSteps][8], top[2 * kApSteps];  // of every row of the warp
    bool infinite = false;
#pragma unroll
    for (int i = 0; i < kApSteps; ++i) widen8(raw[i], x[i]);
    if (kAhead && g + 1 < g1) load(g + 1);  // under way while this head is worked on
    if (norm) rms_norm8(x, w, p.eps);
#pragma unroll
    for (int i = 0; i < kApSteps; ++i) {
      float4 c = {}, sn = {};
      if (kTurn != kPlain) c = turns[(2 * i) * 32], sn = turns[(2 * i + 1) * 32];
      turn_row<kTurn>(c, sn, (inside >> i) & 1u, l < turning, x[i]);
      float v = 0.f;  // NaN counts for none
#pragma unroll
      for (int d = 0; d < 8; ++d) v = fmaxf(v, fabsf(x[i][d]));
      infinite = infinite || v > FLT_MAX;
      top[i] = v;
    }
    infinite = __any_sync(0xffffffffu, infinite);
    if (infinite) {  // rare: infinities count for none
#pragma unroll
      for (int i = 0; i < kApSteps; ++i) {
        top[i] = 0.f;
#pragma unroll
        for (int d = 0; d < 8; ++d) top[i] = fabsf(x[i][d]) <= FLT_MAX ? fmaxf(top[i], fabsf(x[i][d])) : top[i];
      }
    }
#pragma unroll
    for (int i = 0; i < kApSteps; ++i) {
      top[i] = __uint_as_float(__reduce_max_sync(half_mask, __float_as_uint(top[i])));
      if (!kSingle) top[kApSteps + i] = __shfl_xor_sync(0xffffffffu, top[i], 16);
    }
    if constexpr (kSingle) {
      float s[kApSteps], inv[kApSteps];
#pragma unroll
      for (int i = 0; i < kApSteps; ++i) {
        s[i] = fmaxf(divide(top[i], 448.f, 1.0f / 448.f), kMinScale);
        inv[i] = __fdividef(1.f, s[i]);
      }
#pragma unroll
      for (int i = 0; i < kApSteps; ++i) {
        const uint2 codes = quantise8(x[i], s[i], inv[i], infinite);
        if (row_at[i] < 0) continue;
        store_codes(cache + (row_at[i] * p.num_kv_heads + g) * kHeadDim, pieces, halves, codes);
        if (l == 0) scales[row_at[i] * p.num_kv_heads + g] = s[i];  // a row is a block
      }
      continue;
    }
    __syncwarp();  // the old scales are read before a lane writes them
#pragma unroll
    for (int i = 0; i < kApSteps; ++i) {
      // the maximum of the row's block, whose other rows are this half's or the
      // other's; rows past the last one repeat it
      float v = top[i];
#pragma unroll
      for (int k = 0; k < 2 * kApSteps; ++k) v = same >> (8 * i + k) & 1u ? fmaxf(v, top[k]) : v;
      const float s = fmaxf(old[i], fmaxf(divide(v, 448.f, 1.0f / 448.f), kMinScale));
      const float inv = __fdividef(1.f, s);
      if (row_at[i] < 0) continue;
      store_codes(cache + (row_at[i] * p.num_kv_heads + g) * kHeadDim, pieces, halves, quantise8(x[i], s, inv, infinite));
      // the first row of a block that goes sees to its scale and its kept rows
      if (!(begins >> i & 1u) || old[i] == s) continue;
      if (i == 0 && side == 0 && lead > 0) {
        const float ratio = divide(old[i], s, inv);
        for (int back = 1; back <= lead; ++back) {
          uint2* at = reinterpret_cast<uint2*>(cache + ((row_at[i] - back) * p.num_kv_heads + g) * kHeadDim + 8 * l);
          *at = rescale8(*at, ratio);
        }
      }
      if (l == 0) scales[scale_at[i] * p.num_kv_heads + g] = s;
    }
  }
}

// A warp's shared memory: its ring, and four cosines and sines a lane and row.
template <typename T>
__host__ __device__ constexpr int ap_warp_bytes() {
  return kApStages * kApRows * kHeadDim * (int)sizeof(T) + kApSteps * 2 * 32 * 16;
}

// kHold: the group's warps hold all rows of a block. per: heads of a group.
template <typename T, bool kHold, int kTurn>
__global__ void __launch_bounds__(32 * kApWarps, sizeof(T) == 2 && kTurn == kPlain ? 3 : 2)
    qsa_block_append_kernel(const __grid_constant__ BlockAppendParams p, uint32_t items, int group, int per) {
  __shared__ float tops[3][kApWarps];
  extern __shared__ __align__(128) uint8_t smem[];
  T* ring = reinterpret_cast<T*>(smem + threadIdx.x / 32 * ap_warp_bytes<T>());
  const uint32_t parts = (p.num_kv_heads + per - 1) / per;
  // K's groups come first, then V's: a CTA's warps do the same work
  const uint32_t item = blockIdx.x * (kApWarps / group) + threadIdx.x / 32 / group;
  const bool is_k = blockIdx.y == 0;
  const uint32_t slot = item / parts;
  const int g0 = (int)(item - slot * parts) * per;
  ApBlock b = {};
  if (item < items) b = find_block(p, slot, threadIdx.x % 32, p.block_size);
  if (is_k)
    append_block<T, kHold, kTurn>(p, b, true, g0, group, per, tops, ring);
  else
    append_block<T, kHold, kPlain>(p, b, false, g0, group, per, tops, ring);
}

template <typename T, int kTurn, bool kSingle>
__global__ void __launch_bounds__(32 * kApWarps, 2)
    qsa_block_append_packed_kernel(const __grid_constant__ BlockAppendParams p, uint32_t items, int run, int per) {
  __shared__ float4 turns[kTurn == kPlain ? 1 : kApWarps * kApSteps * 2 * 32];
  float4* own_turns = turns + (kTurn == kPlain ? 0 : threadIdx.x / 32 * kApSteps * 2 * 32 + threadIdx.x % 32);
  const uint32_t parts = (p.num_kv_heads + per - 1) / per;
  const uint32_t item = blockIdx.x * kApWarps + threadIdx.x / 32;
  if (item >= items) return;
  const uint32_t slot = item / parts;
  const int g0 = (int)(item - slot * parts) * per;
  const ApBlock b = find_block(p, slot, threadIdx.x % 32, run);
  if (blockIdx.y == 0)
    append_packed<T, kTurn, kSingle>(p, b, true, g0, per, own_turns);
  else
    append_packed<T, kPlain, kSingle>(p, b, false, g0, per, own_turns);
}

// One token an entry, a decode step's append: a warp takes an entry and head, its
// lower half warp the key, the upper one the value. The call is bound by the
// latency of what hangs together (start, page, old scale), so the row's load
// goes out first.
template <typename T, int kTurn>
__global__ void __launch_bounds__(32 * kApWarps) qsa_block_append_one_kernel(const __grid_constant__ BlockAppendParams p) {
  const int lane = threadIdx.x % 32, l = lane % kRowLanes, side = lane / kRowLanes;
  const uint32_t item = blockIdx.x * kApWarps + threadIdx.x / 32;
  const uint32_t e = item / (uint32_t)p.num_kv_heads;
  const int g = (int)(item - e * p.num_kv_heads);
  if (e >= (uint32_t)p.entries) return;
  const bool is_k = side == 0;
  const int turning = kTurn == kPlain ? 0 : p.rope.rotary >> 3;
  const bool halves = kTurn == kHalves && is_k && l < turning;
  const Pieces pieces = halves ? lane_pieces<kTurn>(l, p.rope.rotary) : Pieces{8 * l, 8 * l + 4};
  Raw8<T> raw;
  load8(static_cast<const T*>(is_k ? p.k : p.v) + (int64_t)e * p.token_stride + g * kHeadDim, pieces, raw);
  const int start = __ldg(p.starts + e);
  const int req = p.reqs ? __ldg(p.reqs + e) : (int)e;
  const int B = p.block_size;
  const int lp = max(start, 0) / p.page_size, off = max(start, 0) - lp * p.page_size;
  int page = -1;
  if (start >= 0 && req >= 0 && req < p.num_reqs && lp < p.pages_per_req) page = __ldg(p.btable + req * p.btable_stride + lp);
  const bool goes = page >= 0 && page < p.num_pages;
  float4 c = {}, sn = {};
  bool in = true;
  if (kTurn != kPlain && is_k) in = load_turn(p.rope, e, max(start, 0), l, turning, c, sn);
  float w[8], x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = 1.f;
  if (p.k_weight) load_weight8(p.k_weight, p.weight_dtype, pieces, w);
  float* scale = (is_k ? p.k_scales : p.v_scales) +
                 ((int64_t)max(page, 0) * (p.page_size / B) + off / B) * p.num_kv_heads + g;
  const int lead = off % B;  // rows that the block keeps
  const float old = goes && lead > 0 ? *scale : 0.f;

  widen8(raw, x);
  if (p.k_weight) {
    float y[1][8];
#pragma unroll
    for (int d = 0; d < 8; ++d) y[0][d] = x[d];
    rms_norm8(y, w, p.eps);
#pragma unroll
    for (int d = 0; d < 8; ++d) x[d] = is_k ? y[0][d] : x[d];
  }
  if (is_k) turn_row<kTurn>(c, sn, in, l < turning, x);
  float top = 0.f, finite = 0.f;
#pragma unroll
  for (int d = 0; d < 8; ++d) {
    top = fmaxf(top, fabsf(x[d]));
    finite = fabsf(x[d]) <= FLT_MAX ? fmaxf(finite, fabsf(x[d])) : finite;
  }
#pragma unroll
  for (int o = kRowLanes / 2; o > 0; o >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    finite = fmaxf(finite, __shfl_xor_sync(0xffffffffu, finite, o));
  }
  if (!goes) return;  // the whole warp: one page for both
  const float s = fmaxf(old, fmaxf(divide(finite, 448.f, 1.0f / 448.f), kMinScale));
  const float inv = __fdividef(1.f, s);
  const int step = p.num_kv_heads * kHeadDim;
  uint8_t* row = (is_k ? p.k_cache : p.v_cache) + ((int64_t)page * p.page_size + off) * step + g * kHeadDim;
  store_codes(row, pieces, halves, quantise8(x, s, inv, top > FLT_MAX));
  if (old != s) {
    const float ratio = divide(old, s, inv);
    for (int back = 1; back <= lead; back += 8) {
      uint2 codes[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (back + i <= lead) codes[i] = *reinterpret_cast<const uint2*>(row - (int64_t)(back + i) * step + 8 * l);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (back + i <= lead) *reinterpret_cast<uint2*>(row - (int64_t)(back + i) * step + 8 * l) = rescale8(codes[i], ratio);
    }
  }
  __syncwarp();  // the old scales are read before a lane writes them
  if (old != s && l == 0) *scale = s;
}

template <typename T>
cudaError_t launch_one(const BlockAppendParams& p, cudaStream_t stream) {
  const int64_t items = (int64_t)p.entries * p.num_kv_heads;
  if (items > 0xffffffffll - kApWarps) return cudaErrorInvalidValue;
  const unsigned grid = (unsigned)((items + kApWarps - 1) / kApWarps);
  const int threads = 32 * kApWarps;
  if (!p.rope.table)
    qsa_block_append_one_kernel<T, kPlain><<<grid, threads, 0, stream>>>(p);
  else if (!p.rope.interleaved)
    qsa_block_append_one_kernel<T, kHalves><<<grid, threads, 0, stream>>>(p);
  else
    qsa_block_append_one_kernel<T, kNeighbours><<<grid, threads, 0, stream>>>(p);
  return cudaGetLastError();
}

template <typename T, bool kHold, int kTurn>
cudaError_t launch(const BlockAppendParams& p, uint32_t items, dim3 grid, int group, int per, cudaStream_t stream) {
  constexpr int kSmem = kHold ? kApWarps * ap_warp_bytes<T>() : 0;
  // shared memory beyond the default limit, once per device
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (kSmem > 0 && !(ready.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(qsa_block_append_kernel<T, kHold, kTurn>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    ready.fetch_or(bit, std::memory_order_acq_rel);
  }
  qsa_block_append_kernel<T, kHold, kTurn><<<grid, 32 * kApWarps, kSmem, stream>>>(p, items, group, per);
  return cudaGetLastError();
}

template <typename T, bool kHold>
cudaError_t launch(const BlockAppendParams& p, int64_t slots, cudaStream_t stream) {
  int group = 1;
  while (group < kApWarps && group * kApRows < p.block_size) group *= 2;
  // more heads a group while 148 SMs of 16 warps are filled twice
  int per = 1;
  while (per < kApHeads && per < p.num_kv_heads && slots * 2 * ((p.num_kv_heads + 2 * per - 1) / (2 * per)) * group >= 148 * 32)
    per *= 2;
  const int64_t items = slots * ((p.num_kv_heads + per - 1) / per);
  const int64_t blocks = (items * group + kApWarps - 1) / kApWarps;
  if (items > 0xffffffffll - kApWarps || blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  const dim3 grid((unsigned)blocks, 2);
  if (!p.rope.table) return launch<T, kHold, kPlain>(p, (uint32_t)items, grid, group, per, stream);
  if (!p.rope.interleaved) return launch<T, kHold, kHalves>(p, (uint32_t)items, grid, group, per, stream);
  return launch<T, kHold, kNeighbours>(p, (uint32_t)items, grid, group, per, stream);
}

template <typename T, bool kSingle>
cudaError_t launch_packed(const BlockAppendParams& p, int64_t slots, int run, cudaStream_t stream) {
  int per = 1;
  while (per < kApHeads && per < p.num_kv_heads && slots * 2 * ((p.num_kv_heads + 2 * per - 1) / (2 * per)) >= 148 * 32) per *= 2;
  const int64_t items = slots * ((p.num_kv_heads + per - 1) / per);
  const int64_t blocks = (items + kApWarps - 1) / kApWarps;
  if (items > 0xffffffffll - kApWarps || blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  const dim3 grid((unsigned)blocks, 2);
  const int threads = 32 * kApWarps;
  if (!p.rope.table)
    qsa_block_append_packed_kernel<T, kPlain, kSingle><<<grid, threads, 0, stream>>>(p, (uint32_t)items, run, per);
  else if (!p.rope.interleaved)
    qsa_block_append_packed_kernel<T, kHalves, kSingle><<<grid, threads, 0, stream>>>(p, (uint32_t)items, run, per);
  else
    qsa_block_append_packed_kernel<T, kNeighbours, kSingle><<<grid, threads, 0, stream>>>(p, (uint32_t)items, run, per);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_type(const BlockAppendParams& p, cudaStream_t stream) {
  if (!p.cu_tokens) return launch_one<T>(p, stream);
  // blocks of up to 4 tokens leave half of a warp's 8 rows empty, or more
  const int run = p.block_size <= kApRows / 2 ? kApRows / p.block_size * p.block_size : p.block_size;
  const int64_t slots = (int64_t)(p.tokens / run) + 2 * (int64_t)p.entries;
  if (run > p.block_size)
    return p.block_size == 1 ? launch_packed<T, true>(p, slots, run, stream) : launch_packed<T, false>(p, slots, run, stream);
  return p.block_size <= kApWarps * kApRows ? launch<T, true>(p, slots, stream) : launch<T, false>(p, slots, stream);
}

}  // namespace

cudaError_t launch_block_append(const BlockAppendParams& p, cudaStream_t stream) {
  switch (p.dtype) {
    case QSA_B200_DTYPE_BF16: return launch_type<__nv_bfloat16>(p, stream);
    case QSA_B200_DTYPE_F16: return launch_type<__half>(p, stream);
    default: return launch_type<float>(p, stream);
  }
}

}  // namespace qsa
