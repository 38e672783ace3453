// Attention in the latent's space over the latent cache (the absorbed form).
//
//   out[r,i,h] = softmax_t(q[r,i,h] . key_t scale) . value_t,
//   key_t = s_t (codes_t, rope_t),  value_t = s_t codes_t
//
// A row's (node, head) pairs share every token, 64 of them a CTA, so that the
// tokens are an operand of large tensor-core products and are fetched once:
//   S   = Q K^T     128 lanes x 64 tokens. Q lies in tensor memory as two
//                   E4M3 terms a value, q 2^a = t0 + t1 / 16, in neighbouring
//                   lanes: a product of codes with codes needs no conversion of
//                   the cache, and a warp's lane pair has both terms' scores of
//                   one head: a shuffle joins them, and each lane goes on with
//                   32 of the tokens. The rotated part is a bf16 product
//                   into the same accumulator (q 2^a exact in bf16, zeros in the
//                   lanes of the second terms).
//   O^T = V^T P^T   128 values of the latent x 64 pairs, four times for a rank of
//                   512. V^T is the same codes in shared memory, read the other
//                   way; P is two E4M3 terms a weight. A transposed O takes 256
//                   columns of tensor memory for 64 pairs (O itself would need
//                   all 512 for its 128 lanes).
//
// q: the terms are exact for a bf16 value within 2^13 of the head's largest and
// off by 2^-21 of the largest at most below.
//
// P: with s_t a weight on the codes is w_t = 2^(score_t + log2 s_t - r). Each 32
// tokens of a pair have a power of two of their own, which the product applies
// (block scales), with their largest weight brought to 2^7 .. 2^8: a weight is
// rounded to bf16's 8 bits, which two terms hold down to 2^-10 of the 32's largest,
// and to steps of 2^-17 of it below. One scale for all tokens would lose what many
// small weights add up to beside a few large ones (E4M3 ends at 2^-9). The sum of
// weights takes the bf16 value, so that most of this rounding cancels in the
// quotient: l = sum w_t / s_t, in fp32. A row's largest weight is 1 to 2^60 (below), scales
// are 2^-60 .. 2^60 and tokens 2^31 at most, so that l is 2^-60 to 2^151: it is held
// times 2^-30, by the 1 / s that go into it, and results are brought back by as much
// after their division. (A margin that keeps l itself in range, 2^32, was passed so
// often that 32 contexts of 128 heads took 112 us instead of 99.)
// (The conversions to E4M3 share a unit with 2^x that they kept 94 % busy: the terms
// are cut out of the fp32 weights by integer operations instead.)
// r is the largest score + log2 s of the first tile that has one. It moves, and O
// with it, only when a tile passes it by 2^60; each set tells the other its r, tile
// by tile.
//
// Tiles of 64 tokens go in turn to two sets of warps, each with a ring, scores and
// weights of its own, so that one set's softmax runs beside the other's and beside
// the products. A set is two loaders, which bring a tile 128 bytes of each token at a
// time into 8 KiB slots by cp.async (gathered rows, in the 128-byte swizzle that the
// matrix unit reads), and four softmax warps. One warp issues the products of scores
// and one those of weights, of both sets, in the tiles' order.
//
// A first kernel turns the queries into what the products take and shares out the
// work: done in this one, at the start of each segment, it held up everything for 10
// us. The second starts while the first still runs, and the joins likewise.
//
// Work: group g of CTAs (one CTA for each 64 pairs of a row, so that the CTAs that
// read the same tokens run side by side) has an even share of all rows' tiles: at
// most two pieces of rows and any whole rows between. Pieces are joined by their
// log-sums in a last kernel. Few short rows are a CTA each.
//
// Measured at a rank of 512: 8 contexts of 90001 to 131072 tokens, 16 heads, 163 us (3.5
// TB/s; the main kernel 141); 32 of 4096 to 8192, 128 heads, 104 us (530 TFLOP/s); 16
// trees of 24 nodes and 16 heads 108 us; 256 rows of 512 selected tokens, 32 heads, 59
// us; 4 rows of 64 tokens 13 us. A tile takes a set some 3300 cycles of softmax, more
// than twice what the same steps take in a loop by themselves. On the trees a warp's
// time goes to loads and barrier looks (27 % of it), fixed latencies (18 %) and named
// barriers (12 %), waits of the roles for one another among them; instructions that are
// not there yet are 5 %.
//
// Every wait is bounded; a CTA that gives up records it in the device error word,
// waits for its own copies and products, frees its tensor memory and returns.
#include <atomic>

#include "qsa_latent.cuh"
#include "qsa_latent_tc.cuh"

namespace qsa {
namespace {

constexpr int kLdPairs = 64;     // (node, head) pairs of a CTA
constexpr int kLdTile = 64;      // tokens of a tile
constexpr int kLdSlot = kLdTile * 128;
constexpr int kLdSlots = 11;     // of a set's ring
constexpr int kLdMeta = 4;       // tiles whose scales are held
constexpr int kLdReady = 16;     // tiles that may be ready at once: a ring holds 5 of two pieces each
constexpr int kLdSoft = 256;     // threads of the softmax, half of them in each set
constexpr int kLdLoader0 = 8, kLdFenceWarp = 13, kLdWeighWarp = 14, kLdMmaWarp = 15;
// Four warpgroups: a set's softmax each, loaders, and the warps of the two products and
// of the fence with an idle one. The softmax takes registers that the others hand back:
// 2 x 160 + 96 + 96 of the 4 x 128 that the block is launched with.
constexpr int kLdThreads = 512;
// Tiles of a row that is not split, where there is an SM for each. One CTA a row against
// rows shared out, 16 heads, us: 8 tiles, 1 row 18.4 and 15.8, 4 rows 18.0 and 16.6, 32
// rows 18.2 and 21.6, 74 rows 18.8 and 19.4, 140 rows 20.5 and 30.9; 4 tiles, 1 row 13.7
// and 14.7, 140 rows 15.5 and 24.4; 16 tiles, 1 row 27.5 and 18.2, 32 rows 27.4 and 23.6.
constexpr int64_t kLdDirectTiles = 8;
constexpr float kLdOne = 8.f;    // log2 that bounds the largest weight of 32
constexpr float kLdFar = 60.f;   // log2 by which a weight may pass the reference
constexpr float kLdSum = 0x1p-30f;  // what the sum of weights is held times
constexpr float kLdNear = -110.f;  // log2 below it under which 32 weights get no smaller scale
constexpr float kLowest = -3.402823466e38f;
constexpr uint64_t kLdDrainNs = 1000000000ull;

// Scales of a tile: s, log2 s, kLdSum / s, in two halves of 32 tokens that a lane pair
// reads at once, apart by a bank group.
constexpr int kLdHalf = 36;
struct LdMeta {
  float s[2 * kLdHalf], lg[2 * kLdHalf], inv[2 * kLdHalf];
};

constexpr int kLdBarSet = 1, kLdBarAll = 3;  // named barriers: of a set (1, 2), of both

// A block of 16 pairs' queries: words [rank / 16][32 lanes][4] for tensor memory (a
// pair's first terms in lane 2 i, its second ones in 2 i + 1), bf16 [16][64] rotated
// ones, float [16] what a product is to be multiplied by (-0: the query is not finite).
constexpr int kLdBlockPairs = 16;
__host__ __device__ constexpr int ld_block_bytes(int rank) { return 32 * rank + 16 * 128 + 256; }

constexpr int kLdQr = 0;                // rotated queries: 128 rows of 64 bf16
constexpr int kLdP = kLdQr + 16384;     // weights: two terms of 64 rows of 64 tokens of either set
constexpr int kLdRing = kLdP + 16384;   // [2 sets][kLdSlots]
constexpr int kLdQx = kLdRing + 2 * kLdSlots * kLdSlot;            // a rank of 512: the last 32 values of Q
constexpr int kLdMetaAt = kLdQx + 4096;
constexpr int kLdRow = kLdMetaAt + kLdMeta * (int)sizeof(LdMeta);  // float [64]: factors of pairs at a segment's end
constexpr int kLdRef = kLdRow + kLdPairs * 4;                      // float [64]: r
constexpr int kLdMove = kLdRef + kLdPairs * 4;                     // float [2 sets][64]: factors of a moving r
constexpr int kLdScales = kLdMove + 2 * kLdPairs * 4;              // bytes [2 sets][2 tiles][64][4], of 32 tokens each
constexpr int kLdBars = kLdScales + 4 * kLdPairs * 4;
constexpr int kLdNumBars = 4 * kLdSlots + 2 * kLdMeta + kLdReady + 16;
constexpr int kLdMisc = kLdBars + kLdNumBars * 8;  // tensor memory address, group's range
constexpr int kLdSmem = kLdMisc + 64 + 1024;
static_assert(kLdSmem + 256 <= 232448 && kLdBars % 8 == 0 && kLdMisc % 8 == 0 && kLdMetaAt % 16 == 0, "shared memory");

// Columns of tensor memory: Q from 0, up to 120 (of a rank of 512 the last 32 values,
// which would take 8 more, lie in shared memory), the scales of V^T (ones) and P.
constexpr uint32_t kLdTmemOnes = 120, kLdTmemScales = 124, kLdTmemS = 128, kLdTmemO = 256;

// Columns of a row that may hold a token.
__device__ __forceinline__ int ld_columns(const LatentDecodeParams& p, int row, int& count) {
  const int64_t req = p.t2r ? (int64_t)__ldg(p.t2r + row) : (int64_t)row;
  const int capacity = p.indices ? p.topk : p.cache.pages_per_req * p.cache.page_size;
  count = p.counts ? max(__ldg(p.counts + row), 0) : capacity;
  return req >= 0 && req < p.cache.num_reqs ? min(count, capacity) : 0;
}
__device__ __forceinline__ int ld_tiles(const LatentDecodeParams& p, int row) {
  int count;
  return (ld_columns(p, row, count) + kLdTile - 1) / kLdTile;
}

// The segments of a group: tiles from .. to - 1 of a row.
struct LdWalk {
  int row, from, to;
  int64_t left;
  bool whole;
  __device__ __forceinline__ bool next(const LatentDecodeParams& p) {
    // `row` and `from` name where the group's next tile lies, at or after it
    while (left > 0) {
      const int tiles = ld_tiles(p, row);
      if (tiles > from) {
        to = from + (int)min((int64_t)(tiles - from), left);
        whole = from == 0 && to == tiles;
        left -= to - from;
        return true;
      }
      ++row;
      from = 0;
    }
    return false;
  }
  __device__ __forceinline__ void advance() { from = to; }
};

// What a node sees of its row's nodes: bit j % 32 of word j / 32.
__device__ __forceinline__ uint32_t ld_seen_word(const LatentDecodeParams& p, int row, int node, int word) {
  if (word < 0) return 0xffffffffu;  // the tokens before them
  if (word >= (p.nodes + 31) / 32) return 0u;
  if (p.tree) return (uint32_t)__ldg(p.tree + ((int64_t)row * p.nodes + node) * p.tree_words + word);
  const int n = node + 1 - 32 * word;
  return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
}

// Bits 20 to 27 of four words as the bytes of one.
__device__ __forceinline__ uint32_t pack_codes(const uint32_t (&x)[4]) {
  const uint32_t even = __byte_perm(x[0], x[2], 0x7632), odd = __byte_perm(x[1], x[3], 0x7632);
  return ((even >> 4) & 0x00ff00ffu) | ((odd << 4) & 0xff00ff00u);
}

// kChunks: 128-byte pieces of a token's codes.
template <int kChunks>
__global__ void __launch_bounds__(kLdThreads, 1) qsa_latent_decode_kernel(const __grid_constant__ LatentDecodeParams p) {
  constexpr int kRank = 128 * kChunks;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_s = smem_u32(smem_raw);
  const uint32_t base_s = (raw_s + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base_s - raw_s);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kLdBars);
  uint64_t* full = bars;                       // [2 sets][slots] loaders -> fence
  uint64_t* empty = full + 2 * kLdSlots;       // [2 sets][slots] products -> loaders
  uint64_t* meta_full = empty + 2 * kLdSlots;  // [kLdMeta] loaders -> softmax
  uint64_t* meta_empty = meta_full + kLdMeta;  // [kLdMeta] softmax -> loaders
  uint64_t* ready = meta_empty + kLdMeta;      // [kLdReady] fence -> products, each tile
  uint64_t* s_full = ready + kLdReady;         // [2 sets] products -> softmax
  uint64_t* s_empty = s_full + 2;              // [2 sets] softmax -> products
  uint64_t* p_full = s_empty + 2;              // [2 sets] softmax -> products
  uint64_t* o_full = p_full + 2;               // [2 sets] products -> softmax
  uint64_t* r_done = o_full + 2;               // [2 sets] softmax -> the other set's
  uint64_t* q_full = r_done + 2;               // softmax -> products, each segment
  uint64_t* o_done = q_full + 1;               // products -> softmax, each segment
  uint64_t* o_empty = o_done + 1;              // results taken -> products, each segment
  uint64_t* drain = o_empty + 1;               // [2]
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(smem + kLdMisc);
  const uint32_t tries = tries_of(p.wait_limit_ns);
  int* begin = reinterpret_cast<int*>(smem + kLdMisc + 16);          // row, tile
  int64_t* share = reinterpret_cast<int64_t*>(smem + kLdMisc + 24);  // tiles
  LdMeta* metas = reinterpret_cast<LdMeta*>(smem + kLdMetaAt);
  float* head_f = reinterpret_cast<float*>(smem + kLdRow);
  float* pair_r = reinterpret_cast<float*>(smem + kLdRef);

  const int rt = (int)(blockIdx.x % p.row_tiles), group = (int)(blockIdx.x / p.row_tiles);
  const int pairs = p.nodes * p.heads;
  const int mine = min(kLdPairs, pairs - rt * kLdPairs);  // pairs of this CTA
  // Up to 32 pairs have both terms of the weights side by side as columns of one
  // product, which is half the products (their number, not their width, is what
  // they cost: 62 cycles each from 16 to 64 columns), and two columns of O each.
  const bool few = mine <= kLdPairs / 2;
  const int cols = (mine + 15) / 16 * 16;            // columns of the first terms
  const int lo_row = few ? cols : kLdPairs;          // where the second terms' rows of P begin
  const int blocks = cols / 16;                      // of 16 pairs: a softmax warp of each set has one

  if (tid == 0) {
    for (int i = 0; i < 2 * kLdSlots; ++i) mbar_init(full + i, 64), mbar_init(empty + i, 1);
    for (int i = 0; i < kLdMeta; ++i) mbar_init(meta_full + i, 2), mbar_init(meta_empty + i, blocks);
    for (int i = 0; i < kLdReady; ++i) mbar_init(ready + i, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(s_empty + i, 32 * blocks);
      mbar_init(p_full + i, kLdSoft / 2);
      mbar_init(o_full + i, 1);
      mbar_init(r_done + i, blocks);
      mbar_init(drain + i, 1);
    }
    mbar_init(q_full, kLdSoft);
    mbar_init(o_done, 1);
    mbar_init(o_empty, kLdSoft);
    fence_mbar_init();
  }
  if (warp == kLdMmaWarp) {
    tmem_alloc(tmem_at, 512);
    tmem_relinquish();
    tc_fence_before();
  }
  if (tid < 64) {  // the rotated part has no second terms: every other row stays zero
#pragma unroll
    for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(smem + kLdQr + (2 * tid + 1) * 128 + i * 16) = make_uint4(0u, 0u, 0u, 0u);
    fence_proxy_async_smem();
  }

  wait_for_prerequisites();
  launch_dependents();
  if (tid == 0) {
    // the group's share of the tiles
    begin[0] = group, begin[1] = 0;
    if (p.planned) {
      const int2 b = p.begins[group];
      const int64_t total = *p.total, groups = min((int64_t)p.groups, total);
      begin[0] = b.x, begin[1] = b.y;
      *share = group < groups ? total * (group + 1) / groups - total * group / groups : 0;
    } else {
      *share = ld_tiles(p, group);
    }
  }
  __syncwarp();
  __syncthreads();
  tc_fence_after();
  constexpr uint32_t tmem = 0;  // all of it is this block's
  LdWalk walk;
  walk.row = begin[0], walk.from = begin[1], walk.left = *share;
  bool failed = false;

  if (warp >= kLdLoader0 && warp < kLdLoader0 + 4) {
    // =============================== loaders ================================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;\n");
    // Two warps a set, 32 tokens of each of its tiles each: a lane looks up its own
    // token, and 8 lanes fetch a token's 128 bytes.
    const int w = warp - kLdLoader0, set = w >> 1;
    const int piece = lane & 7, sub = lane >> 3;
    const int tok = 32 * (w & 1) + lane;  // the lane's own token
    const int first_node = rt * kLdPairs / p.heads, last_node = (rt * kLdPairs + mine - 1) / p.heads;
    uint64_t* const my_full = full + set * kLdSlots;
    uint64_t* const my_empty = empty + set * kLdSlots;
    int issued = 0, tile_n = 0;
    auto wait_free = [&](uint64_t* bar, uint32_t parity) -> bool {
      return __all_sync(0xffffffffu, wait_tries(bar, parity, tries));
    };
    while (!failed && walk.next(p)) {
      int count;
      const int row = walk.row;
      const int columns = ld_columns(p, row, count);
      const int64_t req = p.t2r ? (int64_t)__ldg(p.t2r + row) : (int64_t)row;
      const int own = p.nodes > 1 ? count - p.nodes : 0x7fffffff;
      // A token's lookup is three loads in a row (its index, its page, its scale):
      // each is made a tile before the next one needs it.
      auto token = [&](int tile) -> int {  // -1: masked
        const int col = tile * kLdTile + tok;
        if (tile >= walk.to || col >= columns) return -1;
        if (col >= own) {  // seen by a node of this CTA?
          const int d = col - own;
          uint32_t any = 0;
          if (p.tree) {
#pragma unroll 4
            for (int i = first_node; i <= last_node; ++i) any |= ld_seen_word(p, row, i, d / 32);
          } else {
            any = ld_seen_word(p, row, last_node, d / 32);
          }
          if (!((any >> (d % 32)) & 1u)) return -1;
        }
        return p.indices ? __ldg(p.indices + (int64_t)row * p.indices_stride + col) : col;
      };
      struct Page {
        int page, off;
      };
      auto find = [&](int t) -> Page {
        const uint32_t lp = __umulhi(2u * (uint32_t)max(t, 0), p.cache.page_mul) >> p.cache.page_shift;
        const bool in = t >= 0 && (int)lp < p.cache.pages_per_req;
        return {in ? __ldg(p.cache.btable + req * p.cache.btable_stride + lp) : -1, t - (int)lp * p.cache.page_size};
      };
      auto slot_of = [&](Page x) -> int {
        return x.page >= 0 && x.page < p.cache.num_pages ? x.page * p.cache.page_size + x.off : -1;
      };
      auto scale_of = [&](int slot) -> float { return slot >= 0 ? __ldg(p.cache.scales + slot) : 0.f; };
      // this set's tiles: every other one
      const int begin_at = walk.from + ((set ^ tile_n) & 1);
      const int t0 = token(begin_at), t1 = token(begin_at + 2);
      int ahead = token(begin_at + 4);
      const Page p0 = find(t0);
      Page page = find(t1);
      int slot = slot_of(p0);
      float scale = scale_of(slot);
#pragma unroll 1
      for (int tile = begin_at; tile < walk.to; tile += 2) {
        const int n = tile_n + tile - walk.from;
        const int next_slot = slot_of(page);
        const float next_scale = scale_of(next_slot);
        page = find(ahead);
        ahead = token(tile + 6);
        int from[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) from[k] = __shfl_sync(0xffffffffu, slot, 4 * k + sub);
        // row of pass k: 32 (w & 1) + 4 k + sub, so its swizzle is (4 (k & 1) + sub)'s
        const uint32_t dst0 = base_s + kLdRing + set * kLdSlots * kLdSlot + (32 * (w & 1) + sub) * 128;
        const uint32_t even = (uint32_t)(piece ^ sub) << 4, odd = (uint32_t)(piece ^ (4 + sub)) << 4;
#pragma unroll 1
        for (int c = 0; c <= kChunks; ++c) {
          const int s = issued % kLdSlots;
          if (issued >= kLdSlots && !wait_free(my_empty + s, (uint32_t)((issued / kLdSlots - 1) & 1))) {
            failed = true;
            break;
          }
          const uint8_t* src = (c < kChunks ? p.cache.codes + c * 128 : reinterpret_cast<const uint8_t*>(p.cache.rope)) + piece * 16;
          const int64_t stride = c < kChunks ? kRank : 2 * kLatentRope;
#pragma unroll
          for (int k = 0; k < 8; ++k)
            cp_async_16(dst0 + s * kLdSlot + k * 512 + (k & 1 ? odd : even), src + (int64_t)max(from[k], 0) * stride,
                        from[k] < 0 ? 0u : 16u);
          cp_async_mbar_arrive_noinc(smem_u32(my_full + s));
          ++issued;
        }
        const int m = n % kLdMeta;
        if (failed || (n >= kLdMeta && !wait_free(meta_empty + m, (uint32_t)((n / kLdMeta - 1) & 1)))) {
          failed = true;
          break;
        }
        {
          const int at = (w & 1) * kLdHalf + lane;
          const float s = slot < 0 ? 0.f : scale != scale ? scale : fminf(fmaxf(scale, kLatentLeastScale), kLatentMostScale);
          metas[m].s[at] = s;
          metas[m].lg[at] = slot < 0 ? -INFINITY : log2f(s);
          // a NaN token is a NaN in the weights of those that see it, and nothing in the others'
          metas[m].inv[at] = slot < 0 || s != s ? 0.f : kLdSum / s;
          __syncwarp();
          if (lane == 0) mbar_arrive(meta_full + m);
        }
        slot = next_slot;
        scale = next_scale;
      }
      tile_n += walk.to - walk.from;
      walk.advance();
    }
    cp_async_wait_all();
    // rows without a column: zeros, by this CTA's warps in turn
    for (int64_t r = p.planned ? (int64_t)group + (int64_t)p.groups * w : (w == 0 ? (int64_t)group : (int64_t)p.rows); r < p.rows;
         r += (int64_t)p.groups * 4) {
      if (ld_tiles(p, (int)r) > 0) continue;
      uint4* out = reinterpret_cast<uint4*>(p.out + (r * pairs + rt * kLdPairs) * kRank);
      for (int i = lane; i < mine * kRank / 8; i += 32) out[i] = make_uint4(0u, 0u, 0u, 0u);
    }
  } else if (warp >= kLdLoader0 + 4) {
    // =============================== products ===============================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;\n");
    const uint32_t ring = desc_low(base_s + kLdRing);  // K: tokens by bytes (V^T: the same, MN-major)
    auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
      if (!__all_sync(0xffffffffu, wait_tries(bar, parity, tries))) return false;
      tc_fence_after();
      return true;
    };
    // Scores and weighted sums are issued by a warp each: a wait costs some 200 cycles even where there is nothing to wait for, in which the other's
    // products go on.
    if (warp == kLdMmaWarp) {
      // S = Q K^T
      constexpr uint32_t kIdescS = idesc_e4m3(128, kLdTile, false, false);
      constexpr uint32_t kIdescR = idesc_f16(128, kLdTile, true, false);
      const uint32_t rotated = desc_low(base_s + kLdQr), last = desc_low(base_s + kLdQx, 2048);
      int slot[2] = {0, 0}, n = 0, seg = 0;  // ring slots, tile, segment
      while (!failed && walk.next(p)) {
        failed = !wait(q_full, (uint32_t)(seg & 1));
#pragma unroll 1
        for (int tile = walk.from; tile < walk.to && !failed; ++tile, ++n) {
          const int set = n & 1;
          failed = !wait(ready + n % kLdReady, (uint32_t)((n / kLdReady) & 1)) ||
                   (n >= 2 && !wait(s_empty + set, (uint32_t)(((n >> 1) - 1) & 1)));
          if (failed) break;
          const uint32_t d = tmem + kLdTmemS + set * kLdTile;
          int s = set ? slot[1] : slot[0];
          // rolled: the roles' code together is large
#pragma unroll 1
          for (int c = 0; c < kChunks; ++c) {
            const uint32_t bd = ring + (set * kLdSlots + s) * (kLdSlot / 16);
            const uint32_t a = tmem + c * 32;
            mma_f8_ts(d, a, bd, kIdescS, c > 0);
            mma_f8_ts(d, a + 8, bd + 2, kIdescS, 1u);
            mma_f8_ts(d, a + 16, bd + 4, kIdescS, 1u);
            if (kChunks == 4 && c == 3)
              mma_f8_ss_plain_a(d, last, bd + 6, kIdescS, 1u);
            else
              mma_f8_ts(d, a + 24, bd + 6, kIdescS, 1u);
            s = s + 1 == kLdSlots ? 0 : s + 1;
          }
          const uint32_t bd = ring + (set * kLdSlots + s) * (kLdSlot / 16);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) mma_f16_ss(d, rotated + kk * 2, bd + kk * 2, kIdescR, 1u);
          warp_commit(s_full + set);
          warp_commit(empty + set * kLdSlots + s);
          s = s + 1 == kLdSlots ? 0 : s + 1;
          if (set) slot[1] = s; else slot[0] = s;
        }
        ++seg;
        walk.advance();
      }
      warp_commit(drain);
      if (!mbar_wait_bounded(drain, 0u, kLdDrainNs)) failed = true;
    } else if (warp == kLdWeighWarp) {
      // O^T (+)= V^T P^T
      const uint32_t idesc_o = idesc_mxf8(128, few ? 2 * cols : cols, true, false);
      const uint32_t weights = desc_low(base_s + kLdP), second = kLdPairs * 128 / 16;
      int slot[2] = {0, 0}, n = 0, seg = 0;
      while (!failed && walk.next(p)) {
#pragma unroll 1
        for (int tile = walk.from; tile < walk.to && !failed; ++tile, ++n) {
          const int set = n & 1;
          const bool first = tile == walk.from;
          failed = !wait(p_full + set, (uint32_t)((n >> 1) & 1)) ||
                   (first && seg > 0 && !wait(o_empty, (uint32_t)((seg - 1) & 1)));
          if (failed) break;
          const uint32_t ones = tmem + kLdTmemOnes, scales = tmem + kLdTmemScales + 2 * set;
          const uint32_t pd = weights + set * 4;
          int s = set ? slot[1] : slot[0];
#pragma unroll 1
          for (int c = 0; c < kChunks; ++c) {
            const uint32_t ad = ring + (set * kLdSlots + s) * (kLdSlot / 16), d = tmem + kLdTmemO + c * kLdPairs;
#pragma unroll
            for (int kk = 0; kk < kLdTile / 32; ++kk) {
              const uint32_t idesc = idesc_o | kk << 4;  // the kk-th 32 tokens' scales
              mma_mxf8_ss(d, ad + kk * 256, pd + kk * 2, idesc, ones, scales, kk > 0 ? 1u : !first);
              if (!few) mma_mxf8_ss(d, ad + kk * 256, pd + second + kk * 2, idesc, ones, scales, 1u);
            }
            warp_commit(empty + set * kLdSlots + s);
            s = s + 1 == kLdSlots ? 0 : s + 1;
          }
          warp_commit(o_full + set);
          s = s + 1 == kLdSlots ? 0 : s + 1;  // the rotated part's
          if (set) slot[1] = s; else slot[0] = s;
        }
        warp_commit(o_done);
        ++seg;
        walk.advance();
      }
      warp_commit(drain + 1);
      if (!mbar_wait_bounded(drain + 1, 0u, kLdDrainNs)) failed = true;
    } else if (warp == kLdFenceWarp && lane == 0) {
      // The copies wrote by one path to shared memory and the products read by
      // another: the fence between them waits for what its own thread has under
      // way, 1 us in a thread that copies or multiplies, and nothing in this one.
      int slot[2] = {0, 0}, n = 0;
      uint32_t turn[2] = {0, 0};
      while (!failed && walk.next(p)) {
#pragma unroll 1
        for (int tile = walk.from; tile < walk.to && !failed; ++tile, ++n) {
          const int set = n & 1;
          int s = set ? slot[1] : slot[0];
          uint32_t t = set ? turn[1] : turn[0];
#pragma unroll 1
          for (int c = 0; c <= kChunks && !failed; ++c) {
            failed = !wait_tries(full + set * kLdSlots + s, t, tries);
            if (++s == kLdSlots) s = 0, t ^= 1u;
          }
          if (set) slot[1] = s, turn[1] = t; else slot[0] = s, turn[0] = t;
          fence_proxy_async_smem();
          mbar_arrive(ready + n % kLdReady);
        }
        walk.advance();
      }
    }
    __syncwarp();
  } else {
    // ========================== softmax, results ===========================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 160;\n");
    const bool odd = (lane & 1) != 0;
    const int set = warp >> 2, q4 = warp & 3;
    // Quarter q of the lanes has the pairs 16 q .. 16 q + 15. Up to 32 pairs stand
    // there twice, in a quarter or two for each set, so that the sets' warps run on
    // different quarters of the SM too.
    const int block0 = few ? q4 % blocks : q4;          // the quarter's
    const bool placed = few ? q4 < 2 * blocks : q4 < blocks;
    const int pair = 16 * block0 + (lane >> 1);         // this lane pair's (node, head) in the CTA
    const bool live = placed && (!few || q4 / blocks == set);  // the warp has scores to look at
    const int rho = rt * kLdPairs + pair;
    const int node = min(rho / p.heads, p.nodes - 1);
    const int half = odd ? 1 : 0;                       // this lane's 32 tokens of a tile
    const uint32_t lane_base = (uint32_t)(q4 * 32) << 16;
    int first_n = 0, seg = 0;  // tiles before the segment, segments
    // A segment's queries go to their places once the scores of the one before it are
    // done, while its last product is under way; returns what a product of them is to
    // be multiplied by.
    const int row_blocks = (pairs + kLdBlockPairs - 1) / kLdBlockPairs;
    auto place_q = [&](int row) -> float {
      float qs = 0.f;
      if (placed) {
        const uint8_t* block = p.queries + ((int64_t)row * row_blocks + rt * 4 + block0) * ld_block_bytes(kRank);
        const uint4* words = reinterpret_cast<const uint4*>(block) + set * 4 * kChunks * 32 + lane;
        const uint4* rotated = reinterpret_cast<const uint4*>(block + 32 * kRank) + set * 64 + lane;
        uint4 w[4 * kChunks], t[2];
#pragma unroll
        for (int i = 0; i < 4 * kChunks; ++i) w[i] = __ldg(words + i * 32);
#pragma unroll
        for (int i = 0; i < 2; ++i) t[i] = __ldg(rotated + i * 32);
        qs = __ldg(reinterpret_cast<const float*>(block + 32 * kRank + 16 * 128) + (lane >> 1));
#pragma unroll
        for (int i = 0; i < 4 * kChunks; i += 2) {
          const uint32_t v[8] = {w[i].x, w[i].y, w[i].z, w[i].w, w[i + 1].x, w[i + 1].y, w[i + 1].z, w[i + 1].w};
          if (kChunks == 4 && set == 1 && i == 14) {
            uint8_t* at = smem + kLdQx + (4 * q4 + (lane >> 3)) * 128 + (lane & 7) * 16;
            *reinterpret_cast<uint4*>(at) = w[i];
            *reinterpret_cast<uint4*>(at + 2048) = w[i + 1];
          } else {
            tmem_st(tmem + lane_base + (set * 4 * kChunks + i) * 4, v);
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int piece = set * 64 + i * 32 + lane;  // 16 bytes of row piece / 8
          *reinterpret_cast<uint4*>(smem + kLdQr + sw128_offset(32 * q4 + 2 * (piece >> 3), 16 * (piece & 7))) = t[i];
        }
        tmem_wait_st();
        fence_proxy_async_smem();
      }
      tc_fence_before();
      mbar_arrive(q_full);
      return qs;
    };
    if (set == 0) {
      const uint32_t ones[4] = {0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu};
      tmem_st(tmem + lane_base + kLdTmemOnes, ones);
      tmem_wait_st();
    }
    // the rows of P whose scales this lane's two words hold
    const int scale0 = few && lane >= cols ? lane - cols : lane, scale1 = few ? lane : lane + 32;
    bool more = walk.next(p);
    float next_qs = 0.f;
    if (more) next_qs = place_q(walk.row);
    while (more) {
      const LdWalk now = walk;
      int count;
      ld_columns(p, now.row, count);
      const int own = p.nodes > 1 ? count - p.nodes : 0x7fffffff;
      walk.advance();
      more = walk.next(p);
      const float qs = next_qs;
      float r = kLowest, l = 0.f;
      const float km = odd ? qs * 0.0625f : qs, kr = odd ? qs : qs * 0.0625f;  // own and the other lane's term
#pragma unroll 1
      for (int tile = now.from + ((set ^ first_n) & 1); tile < now.to; tile += 2) {
        const int n = first_n + tile - now.from;
        const int m = n % kLdMeta;
        const uint32_t turn = (uint32_t)((n >> 1) & 1);
        const bool begun = tile > now.from;
        float u[32];
        float top = -INFINITY;
        if (live) {
          if (!failed)
            failed = !(wait_tries(meta_full + m, (uint32_t)((n / kLdMeta) & 1), tries) && wait_tries(s_full + set, turn, tries));
          failed = __any_sync(0xffffffffu, failed);
          tc_fence_after();
          const float* ms = metas[m].s + half * kLdHalf;
          const float* ml = metas[m].lg + half * kLdHalf;
          float x[32], y[32];
          const uint32_t at = tmem + lane_base + kLdTmemS + kLdTile * set;
          tmem_ld_2x32_wait(at, at + 32, x, y);
          tc_fence_before();
          mbar_arrive(s_empty + set);
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 s4 = *reinterpret_cast<const float4*>(ms + j);
            const float4 l4 = *reinterpret_cast<const float4*>(ml + j);
            const float ss[4] = {s4.x, s4.y, s4.z, s4.w}, ll[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              const float a = __shfl_xor_sync(0xffffffffu, odd ? x[j + i] : y[j + i], 1);
              const float b = __shfl_xor_sync(0xffffffffu, odd ? x[j + i + 1] : y[j + i + 1], 1);
              const uint64_t own_term = pair2(odd ? y[j + i] : x[j + i], odd ? y[j + i + 1] : x[j + i + 1]);
              const uint64_t v = fma2(own_term, pair2(km, km), mul2(pair2(a, b), pair2(kr, kr)));
              unpair2(fma2(v, pair2(ss[i], ss[i + 1]), pair2(ll[i], ll[i + 1])), u[j + i], u[j + i + 1]);
            }
          }
          if (__builtin_expect(p.nodes > 1 && tile * kLdTile + kLdTile > own, 0)) {
            const int d0 = tile * kLdTile + 32 * half - own;
            const int word = d0 >> 5;
            const uint32_t bits = __funnelshift_r(ld_seen_word(p, now.row, node, word), ld_seen_word(p, now.row, node, word + 1), d0 & 31);
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (!((bits >> j) & 1u)) u[j] = -INFINITY;
          }
#pragma unroll
          for (int j = 0; j < 32; j += 2) top = max3_nan(top, u[j], u[j + 1]);
          // the reference, as the tile before left it
          if (begun) {
            if (!failed) failed = !wait_tries(r_done + (set ^ 1), (uint32_t)(((n - 1) >> 1) & 1), tries);
            failed = __any_sync(0xffffffffu, failed);
            const float next = pair_r[pair];
            if (next != r) l *= ex2(r - next), r = next;
          }
        }
        // the scale of this lane's 32 weights
        uint8_t* scales = smem + kLdScales + (2 * set + (int)turn) * 4 * kLdPairs;
        auto scale32 = [&]() -> float {
          const float e = fminf(fmaxf(ceilf(top - r), kLdNear), kLdFar);
          if (live) scales[4 * pair + half] = (uint8_t)(127 - (int)kLdOne + (int)e);
          return e;
        };
        float e = scale32();
        // a reference that a weight passes by too much moves, and O and l with it
        if (__builtin_expect(bar_vote(kLdBarSet + set, kLdSoft / 2, top > r + kLdFar || failed), 0)) {
          float* move = reinterpret_cast<float*>(smem + kLdMove) + set * kLdPairs;
          if (live) {
            const float next = fmaxf(r, fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1)));
            const float f = ex2(r - next);  // 0 before the first weight
            l *= f;
            r = next;
            if (!odd) move[pair] = f;
          }
          // all products before this tile's
          if (begun && !failed)
            failed = !((n < 2 || wait_tries(o_full + set, turn ^ 1u, tries)) &&
                       wait_tries(o_full + (set ^ 1), (uint32_t)(((n - 1) >> 1) & 1), tries));
          failed = __any_sync(0xffffffffu, failed);
          if (bar_vote(kLdBarSet + set, kLdSoft / 2, failed)) {
            failed = true;
            break;
          }
          if (begun) {
            tc_fence_after();
            // 16 pairs at a time, where one has moved
#pragma unroll 1
            for (int b = 0; b < cols; b += 16) {
              const float f = move[b + (lane & 15)];
              if (__all_sync(0xffffffffu, f == 1.f)) continue;
#pragma unroll 1
              for (int c = 0; c < kChunks * (few ? 2 : 1); ++c) {
                const uint32_t at = tmem + lane_base + kLdTmemO + (few ? c / 2 : c) * kLdPairs + b + (few ? c % 2 * cols : 0);
                float x[16];
                uint32_t y[16];
                tmem_ld_wait<16>(at, x);
#pragma unroll
                for (int j = 0; j < 16; ++j) y[j] = __float_as_uint(x[j] * __shfl_sync(0xffffffffu, f, j));
                tmem_st(at, y);
              }
            }
            tmem_wait_st();
            tc_fence_before();
          }
          e = scale32();
          bar_sync(kLdBarSet + set, kLdSoft / 2);
        }
        if (live) {
          if (!odd) pair_r[pair] = r;
          __syncwarp();
          if (lane == 0) mbar_arrive(r_done + set);
        }
        // ---- weights
        uint32_t hi[8], lo[8];
        if (live) {
          const float* mi = metas[m].inv + half * kLdHalf;
          const float rb = r + (e - kLdOne);
          uint64_t sum2 = 0;
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 i4 = *reinterpret_cast<const float4*>(mi + j);
            const float ii[4] = {i4.x, i4.y, i4.z, i4.w};
            uint32_t first[4], second[4];  // codes in bits 20 to 26
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              float a, b, c, d;
              unpair2(add2(pair2(u[j + i], u[j + i + 1]), pair2(-rb, -rb)), a, b);
              // rounded to 8 bits
              const uint64_t w = pair2(__uint_as_float((__float_as_uint(ex2(a)) + 0x8000u) & 0xffff0000u),
                                       __uint_as_float((__float_as_uint(ex2(b)) + 0x8000u) & 0xffff0000u));
              sum2 = fma2(w, pair2(ii[i], ii[i + 1]), sum2);
              // times 2^-120 an E4M3 value is an fp32 one whose bits 20 to 26 are its code,
              // subnormal values too; half of the last step goes in before it is cut off
              const uint64_t t = fma2(w, pair2(0x1p-120f, 0x1p-120f), pair2(0x1p-130f, 0x1p-130f));
              unpair2(t, a, b);
              first[i] = __float_as_uint(a) & 0xfff00000u, first[i + 1] = __float_as_uint(b) & 0xfff00000u;
              unpair2(add2(t, pair2(-__uint_as_float(first[i]), -__uint_as_float(first[i + 1]))), c, d);
              second[i] = __float_as_uint(c), second[i + 1] = __float_as_uint(d);
            }
            hi[j / 4] = pack_codes(first);
            lo[j / 4] = pack_codes(second);
          }
          float sum, sum_b;
          unpair2(sum2, sum, sum_b);
          sum += sum_b;
          l = fmaf(sum, ex2(e - kLdOne), l);
          if (!(top <= 3.402823466e38f)) l = __int_as_float(0x7fffffff);  // a NaN, or a score past fp32
        }
        if (live) {
          __syncwarp();
          if (lane == 0) mbar_arrive(meta_empty + m);
        }
        // the product of the set's tile before has read its weights and their scales
        if (n >= 2 && !failed) failed = !wait_tries(o_full + set, turn ^ 1u, tries);
        failed = __any_sync(0xffffffffu, failed);
        if (live) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            uint8_t* at = smem + kLdP + sw128_offset(pair, 64 * set + 32 * half + 16 * k);
            *reinterpret_cast<uint4*>(at) = make_uint4(hi[4 * k], hi[4 * k + 1], hi[4 * k + 2], hi[4 * k + 3]);
            *reinterpret_cast<uint4*>(at + lo_row * 128) = make_uint4(lo[4 * k], lo[4 * k + 1], lo[4 * k + 2], lo[4 * k + 3]);
          }
          fence_proxy_async_smem();
        }
        {
          const uint32_t* words = reinterpret_cast<const uint32_t*>(scales);
          const uint32_t both[2] = {words[scale0], words[scale1]};
          tmem_st(tmem + lane_base + kLdTmemScales + 2 * set, both);
          tmem_wait_st();
          tc_fence_before();
        }
        mbar_arrive(p_full + set);
      }
      // ---- the segment's results
      const int last = first_n + (now.to - now.from) - 1;
      if ((last & 1) != set && !failed)  // the other set's last tile
        failed = !wait_tries(r_done + (set ^ 1), (uint32_t)((last >> 1) & 1), tries);
      failed = __any_sync(0xffffffffu, failed);
      if (bar_vote(kLdBarAll, kLdSoft, failed)) {
        failed = true;
        break;
      }
      // all scores are done, and the queries free
      if (more) next_qs = place_q(walk.row);
      failed = !wait_tries(o_done, (uint32_t)(seg & 1), tries);
      failed = __any_sync(0xffffffffu, failed);
      if (live) {
        const float end_r = pair_r[pair];
        l *= ex2(r - end_r);
        r = end_r;
      }
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      if (live && !odd && set == 1) head_f[pair] = l;
      if (bar_vote(kLdBarAll, kLdSoft, failed)) {
        failed = true;
        break;
      }
      const int piece = 2 * group + (now.from > 0 ? 0 : 1);
      if (live && !odd && set == 0) {
        l += head_f[pair];
        if (__float_as_uint(km) == 0x80000000u && l != 0.f) l = __int_as_float(0x7fffffff);  // a query that is not finite
        head_f[pair] = l == 0.f ? 0.f : 1.0f / l;
        if (!now.whole && pair < mine)
          p.part_lse[((int64_t)piece * p.row_tiles + rt) * kLdPairs + pair] = l == 0.f ? -INFINITY : log2f(l) + r;
      }
      bar_sync(kLdBarAll, kLdSoft);
      tc_fence_after();
      const int64_t at = now.whole ? ((int64_t)now.row * pairs + rt * kLdPairs) * kRank
                                    : ((int64_t)piece * p.row_tiles + rt) * kLdPairs * kRank;
      auto store = [&](auto* to, auto round) {
#pragma unroll 1
        for (int c = set; c < 4 * kChunks; c += 2) {
          const int b = c % 4 * 16;
          if (b >= mine) continue;
          float x[16];
          tmem_ld_wait<16>(tmem + lane_base + kLdTmemO + c / 4 * kLdPairs + b, x);
          if (few) {
            float y[16];
            tmem_ld_wait<16>(tmem + lane_base + kLdTmemO + c / 4 * kLdPairs + cols + b, y);
#pragma unroll
            for (int j = 0; j < 16; ++j) x[j] += y[j];
          }
          auto* out = to + (int64_t)b * kRank + c / 4 * 128;
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            const float4 f = *reinterpret_cast<const float4*>(head_f + b + j);
            x[j] *= f.x, x[j + 1] *= f.y, x[j + 2] *= f.z, x[j + 3] *= f.w;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[j + i] *= kLdSum;
          }
          const int some = mine - b;
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (j < some) out[j * kRank] = round(x[j]);
        }
      };
      if (now.whole)
        store(p.out + at + 32 * q4 + lane, [](float v) { return __float2bfloat16_rn(v); });
      else
        store(p.part_o + at + 32 * q4 + lane, [](float v) { return v; });
      tc_fence_before();
      mbar_arrive(o_empty);
      bar_sync(kLdBarAll, kLdSoft);  // the factors are read before the next segment's
      first_n = last + 1;
      ++seg;
    }
  }

  if (failed) {
    if (p.err) atomicOr(p.err, 1);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kLdMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// The queries as the products take them, 16 pairs a block and a pair a warp: q 2^a =
// t0 + t1 / 16 in E4M3, with 2^a taking the largest latent query into [128, 256) as
// far as the rotated ones stay far from bf16's end. A block before those shares out the
// tiles where the rows are shared out.
constexpr int kLpreThreads = 32 * kLdBlockPairs;
template <int kChunks>
__global__ void __launch_bounds__(kLpreThreads) qsa_latent_prepare_kernel(const __grid_constant__ LatentDecodeParams p) {
  constexpr int kRank = 128 * kChunks;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int pairs = p.nodes * p.heads, row_blocks = (pairs + kLdBlockPairs - 1) / kLdBlockPairs;
  launch_dependents();
  // the first block shares out the tiles: it takes longest
  const int64_t at = (int64_t)blockIdx.x - p.planned;
  if (at >= 0) {
    const int row = (int)(at / row_blocks), pair = (int)(at - (int64_t)row * row_blocks) * kLdBlockPairs + warp;
    uint8_t* block = p.queries + at * ld_block_bytes(kRank);
    uint32_t* words = reinterpret_cast<uint32_t*>(block);
    uint2 raw[kChunks];  // 4 values of each of this lane's words
    uint32_t rot = 0;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) raw[i] = make_uint2(0u, 0u);
    if (pair < pairs) {
      const __nv_bfloat16* q = p.q + ((int64_t)row * pairs + pair) * (kRank + kLatentRope);
#pragma unroll
      for (int i = 0; i < kChunks; ++i) raw[i] = __ldg(reinterpret_cast<const uint2*>(q) + 32 * i + lane);
      rot = __ldg(reinterpret_cast<const uint32_t*>(q + kRank) + lane);
    }
    uint32_t top = 0;  // largest |q| as bits, two at a time
#pragma unroll
    for (int i = 0; i < kChunks; ++i) top = __vmaxu2(top, __vmaxu2(raw[i].x & 0x7fff7fffu, raw[i].y & 0x7fff7fffu));
    const uint32_t rtop = rot & 0x7fff7fffu;
    uint32_t both = max(top & 0xffffu, top >> 16) | max(rtop & 0xffffu, rtop >> 16) << 16;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) both = __vmaxu2(both, __shfl_xor_sync(0xffffffffu, both, o));
    const int t = (int)(both & 0xffffu), u = (int)(both >> 16);
    int a = t == 0 ? 0 : 7 - (max(t >> 7, 1) - 127);
    if (u != 0) a = min(a, 40 - (max(u >> 7, 1) - 127));
    a = min(max(a, -120), 120);
    const float up = __uint_as_float((uint32_t)(127 + a) << 23);
    float qs = pair < pairs ? __uint_as_float((uint32_t)(127 - a) << 23) * p.score_scale_log2 : 0.f;
    qs += 0.f;  // no -0 but this one:
    if (t >= 0x7f80 || u >= 0x7f80 || !(fabsf(qs) <= 3.402823466e38f)) {
      // a pair that is NaN where it sees a token and zeros where it sees none: the factor
      // -0 tells, and zeros for its values leave the masks of its scores as they are
      qs = -0.f;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) raw[i] = make_uint2(0u, 0u);
      rot = 0;
    }
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const uint32_t v[2] = {raw[i].x, raw[i].y};
      uint32_t hi[2], lo[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float x = __uint_as_float(v[j] << 16) * up, y = __uint_as_float(v[j] & 0xffff0000u) * up;
        hi[j] = __nv_cvt_float2_to_fp8x2(make_float2(x, y), __NV_SATFINITE, __NV_E4M3);
        const float2 back = e4m3x2_to_f32x2((uint16_t)hi[j]);
        lo[j] = __nv_cvt_float2_to_fp8x2(make_float2((x - back.x) * 16.f, (y - back.y) * 16.f), __NV_SATFINITE, __NV_E4M3);
      }
      const int col = 32 * i + lane;
      uint32_t* to = words + ((col >> 2) * 32 + 2 * warp) * 4 + (col & 3);
      to[0] = hi[0] | hi[1] << 16;
      to[4] = lo[0] | lo[1] << 16;
    }
    const __nv_bfloat162 r2 = __floats2bfloat162_rn(__uint_as_float(rot << 16) * up, __uint_as_float(rot & 0xffff0000u) * up);
    reinterpret_cast<__nv_bfloat162*>(block + 32 * kRank)[warp * 32 + lane] = r2;
    if (lane == 0) reinterpret_cast<float*>(block + 32 * kRank + 16 * 128)[warp] = qs;
    return;
  }
  // each thread counts the tiles of a run of rows
  __shared__ int64_t before[kLpreThreads + 1];
  __shared__ int64_t warp_sum[kLpreThreads / 32];
  const int run = (p.rows + kLpreThreads - 1) / kLpreThreads;
  const int r0 = min(tid * run, p.rows), r1 = min(r0 + run, p.rows);
  int64_t sum = 0;
#pragma unroll 8
  for (int r = r0; r < r1; ++r) sum += ld_tiles(p, r);
  int64_t upto = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) warp_sum[warp] = upto;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kLpreThreads / 32; ++w)
    if (w < warp) upto += warp_sum[w];
  before[tid + 1] = upto;
  if (tid == 0) before[0] = 0;
  __syncthreads();
  const int64_t total = before[kLpreThreads];
  const int64_t groups = min((int64_t)p.groups, total);  // each has a tile at least
  if (tid == 0) *p.total = total;
  for (int g = tid; g < p.groups; g += kLpreThreads) {
    if (g >= groups) {
      p.begins[g] = make_int2(p.rows, 0);
      continue;
    }
    const int64_t u = total * g / groups;
    int lo = 0, hi = kLpreThreads;  // the last run that begins at or before the group's first tile
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (before[mid] <= u) lo = mid; else hi = mid;
    }
    int64_t first = before[lo];
    for (int r = lo * run;; ++r) {
      const int t = ld_tiles(p, r);
      if (u < first + t) {
        p.begins[g] = make_int2(r, (int)(u - first));
        break;
      }
      first += t;
    }
  }
}

// Joins the pieces of a row that several groups share: one block for each group
// that ends a row's first piece, 64-pair part and pair.
__global__ void __launch_bounds__(128) qsa_latent_join_kernel(const __grid_constant__ LatentDecodeParams p) {
  const int pair = blockIdx.x, rt = blockIdx.y, g = blockIdx.z + 1;
  const int pairs = p.nodes * p.heads;
  if (rt * kLdPairs + pair >= pairs) return;
  wait_for_prerequisites();
  // A load for all lanes at a time: one after the other, the pieces' loads took most of
  // 20 us.
  const int lane = threadIdx.x & 31;
  auto begin_of = [&](int at) { return at < p.groups ? p.begins[at] : make_int2(-1, 0); };
  int2 e = begin_of(g - 1 + lane);
  const int2 b = make_int2(__shfl_sync(0xffffffffu, e.x, 1), __shfl_sync(0xffffffffu, e.y, 1));
  if (b.x >= p.rows || b.y == 0) return;
  const int2 before = make_int2(__shfl_sync(0xffffffffu, e.x, 0), __shfl_sync(0xffffffffu, e.y, 0));
  if (before.x == b.x && before.y > 0) return;  // the row's second piece lies further back
  if (lane == 0) e = b;  // looked at, as group g's is
  int last = g - 1;      // of the row's groups
  for (;;) {
    const uint32_t others = __ballot_sync(0xffffffffu, e.x != b.x || e.y == 0);
    if (others) {
      last += __ffs(others) - 2;
      break;
    }
    last += 32;
    e = begin_of(last + lane);
  }
  // pieces: the second of group g - 1, the first of groups g .. last
  auto place = [&](int i) { return ((int64_t)(i == 0 ? 2 * g - 1 : 2 * (g + i - 1)) * p.row_tiles + rt) * kLdPairs + pair; };
  const int pieces = last - g + 2;
  float top = -INFINITY;
  bool nan = false;
  float first_v = -INFINITY;
  for (int i = lane; i < pieces; i += 32) {
    const float v = p.part_lse[place(i)];
    if (i == lane) first_v = v;
    top = fmaxf(top, v);
    nan = nan || v != v;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  nan = __any_sync(0xffffffffu, nan);
  const int rank = p.cache.rank;
  const int d = 4 * threadIdx.x;
  if (d >= rank) return;  // whole warps
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
  if (top > -INFINITY || nan) {
    for (int first = 0; first < pieces; first += 32) {
      // a piece without a visible token has written no results
      const float v = first == 0 ? first_v : first + lane < pieces ? p.part_lse[place(first + lane)] : -INFINITY;
      const float mine = v == -INFINITY ? 0.f : exp2f(v - top);
#pragma unroll 1
      for (int k = 0; k < min(32, pieces - first); k += 4) {
        float w[4];
        float4 x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          w[j] = __shfl_sync(0xffffffffu, mine, k + j);
          x[j] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (w[j] != 0.f) x[j] = *reinterpret_cast<const float4*>(p.part_o + place(first + k + j) * rank + d);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          sum += w[j];
          o.x = fmaf(w[j], x[j].x, o.x), o.y = fmaf(w[j], x[j].y, o.y), o.z = fmaf(w[j], x[j].z, o.z), o.w = fmaf(w[j], x[j].w, o.w);
        }
      }
    }
    const float inv = 1.0f / sum;
    o.x *= inv, o.y *= inv, o.z *= inv, o.w *= inv;
  }
  const __nv_bfloat162 lo = __floats2bfloat162_rn(o.x, o.y), hi = __floats2bfloat162_rn(o.z, o.w);
  *reinterpret_cast<uint2*>(p.out + ((int64_t)b.x * pairs + rt * kLdPairs + pair) * rank + d) =
      make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}

int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

// Launches a kernel that waits for its prerequisites itself (early: it may start
// before the stream's last kernel has ended).
template <typename Kernel>
cudaError_t start(Kernel kernel, dim3 grid, int threads, int smem, bool early, cudaStream_t stream, const LatentDecodeParams& p) {
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = early ? 1 : 0;
  return cudaLaunchKernelEx(&config, kernel, p);
}

template <int kChunks>
cudaError_t launch(const LatentDecodeParams& p, cudaStream_t stream) {
  // the shared memory beyond the default limit, once per device
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(ready.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(qsa_latent_decode_kernel<kChunks>, cudaFuncAttributeMaxDynamicSharedMemorySize, kLdSmem);
    if (e != cudaSuccess) return e;
    ready.fetch_or(bit, std::memory_order_acq_rel);
  }
  const int64_t grid = (int64_t)p.groups * p.row_tiles;
  const int64_t blocks = (int64_t)p.rows * ((p.nodes * p.heads + kLdBlockPairs - 1) / kLdBlockPairs) + p.planned;
  if (grid > 0x7fffffffll || blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  e = start(qsa_latent_prepare_kernel<kChunks>, dim3((unsigned)blocks), kLpreThreads, 0, false, stream, p);
  if (e == cudaSuccess) e = start(qsa_latent_decode_kernel<kChunks>, dim3((unsigned)grid), kLdThreads, kLdSmem, true, stream, p);
  if (e == cudaSuccess && p.planned && p.groups > 1)
    e = start(qsa_latent_join_kernel, dim3((unsigned)(p.nodes * p.heads < kLdPairs ? p.nodes * p.heads : kLdPairs), (unsigned)p.row_tiles, (unsigned)(p.groups - 1)), 128, 0, true, stream, p);
  return e;
}

int64_t query_bytes(const LatentDecodeParams& p) {
  return align256((int64_t)p.rows * ((p.nodes * p.heads + kLdBlockPairs - 1) / kLdBlockPairs) * ld_block_bytes(p.cache.rank));
}

}  // namespace

int64_t latent_decode_plan(LatentDecodeParams& p) {
  p.row_tiles = (p.nodes * p.heads + kLdPairs - 1) / kLdPairs;
  const int64_t columns = p.indices ? p.topk : (int64_t)p.cache.pages_per_req * p.cache.page_size;
  const int sms = latent_sm_count();
  p.planned = (columns + kLdTile - 1) / kLdTile > kLdDirectTiles || (int64_t)p.rows * p.row_tiles > sms;
  p.groups = p.planned ? (sms / p.row_tiles > 1 ? sms / p.row_tiles : 1) : p.rows;
  int64_t need = query_bytes(p);
  if (p.planned) {
    const int64_t pieces = 2ll * p.groups * p.row_tiles * kLdPairs;
    need += align256(pieces * p.cache.rank * 4) + align256(pieces * 4) + align256(8ll * p.groups) + 256;
  }
  return need;
}

void latent_decode_place(LatentDecodeParams& p, void* workspace) {
  char* at = static_cast<char*>(workspace);
  auto take = [&](int64_t bytes) {
    char* here = at;
    at += align256(bytes);
    return here;
  };
  p.queries = reinterpret_cast<uint8_t*>(take(query_bytes(p)));
  if (!p.planned) return;
  const int64_t pieces = 2ll * p.groups * p.row_tiles * kLdPairs;
  p.part_o = reinterpret_cast<float*>(take(pieces * p.cache.rank * 4));
  p.part_lse = reinterpret_cast<float*>(take(pieces * 4));
  p.begins = reinterpret_cast<int2*>(take(8ll * p.groups));
  p.total = reinterpret_cast<int64_t*>(take(8));
}

cudaError_t launch_latent_decode(const LatentDecodeParams& p, cudaStream_t stream) {
  switch (p.cache.rank / 128) {
    case 1: return launch<1>(p, stream);
    case 2: return launch<2>(p, stream);
    case 3: return launch<3>(p, stream);
    default: return launch<4>(p, stream);
  }
}

}  // namespace qsa
