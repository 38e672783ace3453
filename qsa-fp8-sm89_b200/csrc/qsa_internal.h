// Internal launch parameters shared by the C-ABI layer and the kernels.
// Not part of the public interface (that is include/qsa_b200.h).
#pragma once

#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <stdint.h>

namespace qsa {

struct DecodeParams {
  // Tensors (device pointers). Q, gate and out are contiguous [rows, Hq, 128]
  // bf16; the caches are contiguous [num_pages, P, Hkv, 128] FP8 E4M3FN.
  const __nv_bfloat16* q;
  const __nv_bfloat16* gate;
  __nv_bfloat16* out;
  const uint8_t* k;
  const uint8_t* v;
  const int32_t* indices;  // [rows, indices_stride]; the first topk columns are the Top-K list
  const int32_t* counts;   // optional [rows]
  const int32_t* btable;   // [num_reqs, btable_stride]; the first pages_per_req columns are used
  const int32_t* t2r;      // optional [rows]

  float score_scale_log2;  // softmax_scale * k_scale * log2(e)
  float v_scale;

  int rows;
  int num_q_heads;
  int num_kv_heads;
  int group;  // num_q_heads / num_kv_heads
  int page_size;
  int page_shift;  // log2(page_size) when it is a power of two, else -1
  int pages_per_req;
  int num_reqs;
  int64_t num_pages;
  int topk;
  int64_t indices_stride;
  int count_column;  // count read from indices[row * stride + topk]
  int64_t btable_stride;

  // Split of each Top-K row into chunks of `chunk_tokens` (flash-decoding).
  // With num_chunks == 1 the kernel writes `out` directly; otherwise it writes
  // per-chunk partial results that qsa_combine merges.
  int chunk_tokens;
  int num_chunks;
  float* part_o;    // [rows, Hq, num_chunks, 128] normalised partial outputs
  float* part_lse;  // [rows, Hq, num_chunks] log2-sum-exp2 of each chunk (-inf if empty)

  // Row map of the tensor-core kernel (workspace, filled by its row-map
  // kernel): for every Top-K entry of every row, the physical token slot
  // phys * P + t % P, or -1 when masked; row r's entries start at
  // rowmap + r * rowmap_stride (num_chunks * chunk_tokens entries, the tail
  // past topk -1).
  int32_t* rowmap;
  int rowmap_stride;
  // Tile flags (workspace, filled with the row map): one byte per 128-entry
  // tile of each (row, chunk), nonzero when the tile holds a valid entry;
  // 16 bytes per (row, chunk).
  uint8_t* tile_flags;
  // Claim counter of the tensor-core kernel (workspace, zeroed by its row-map
  // kernel): with split rows, CTAs claim windows of items from it.
  int* item_counter;
  // Tensor-core kernel, split rows: 1 when each CTA walks all chunks of a
  // (row, KV head) in turn and merges them itself (no partials, no combine
  // kernel); set by the launcher from tc_merges_chunks.
  int merge_chunks;
  // Tensor-core kernel: log2 of the virtual KV heads per cache KV head (1
  // when a group above 16 runs as two halves), and the caches' own group
  // size Hq / Hkv; set by the launcher.
  int kv_shift;
  int real_group;

  int* err;  // device error word of the current device
  // Limit of each pipeline wait of the tensor-core kernel, in ns of
  // globaltimer: 1 s, unless the test hook qsa_b200_testing_set_wait_limit_ns
  // shortened it. A CTA whose wait runs out sets err and returns.
  uint64_t wait_limit_ns;
};

// Wait limit the launches of this process use (the test hook's value, else
// the 1 s default).
uint64_t wait_limit_ns();

// Kernel launchers (return cudaGetLastError() of the launch).
cudaError_t launch_decode_tc(const DecodeParams& p, cudaStream_t stream);
cudaError_t launch_decode_simt(const DecodeParams& p, cudaStream_t stream);
cudaError_t launch_combine(const DecodeParams& p, cudaStream_t stream);
cudaError_t launch_slots(const DecodeParams& p, int64_t* slots, cudaStream_t stream);
// Paged FP8 cache writer (qsa_cache_write.cu).
struct CacheWriteParams {
  const void* k;  // [tokens, Hkv, 128] new keys, rows token_stride elements apart
  const void* v;
  const int64_t* slots;  // [tokens] physical token slots; outside [0, num_pages * P) = skipped
  uint8_t* k_cache;      // [num_pages, P, Hkv, 128] e4m3fn
  uint8_t* v_cache;
  float k_inv_scale, v_inv_scale;  // 1 / scale, rounded to fp32
  int tokens;
  int num_kv_heads;
  int page_size;
  int64_t num_pages;
  int64_t token_stride;
  int dtype;  // QSA_B200_DTYPE_*
};
cudaError_t launch_cache_write(const CacheWriteParams& p, cudaStream_t stream);

// Top-K index producer (qsa_topk.cu).
struct TopkParams {
  const float* scores;
  const int32_t* lengths;  // may be null
  int32_t* out;
  int rows, ctx, k;
  int64_t score_stride, out_stride;
};
cudaError_t launch_topk(const TopkParams& p, cudaStream_t stream);

// The block-scaled cache: head norm with rotation (qsa_qk_rope.cu), paged
// append (qsa_block_append.cu) and attention (qsa_block_decode.cu).
constexpr int kRopeMaxAxes = 4;
constexpr int kBlockMaxHeads = 0x7fffffff / 128;  // elements of a token's heads are counted in int32
struct RopeParams {
  const float* table;        // [table_len, rotary] cosines, then sines; null = no rotation
  const int32_t* positions;  // [axes, tokens]; null = the caller's own position (append)
  int64_t axis_stride;
  int table_len;
  int rotary;  // multiple of 16, <= 128
  int interleaved;
  int axes;
  int ends[kRopeMaxAxes];  // first pair past each axis' section
  int quads;               // every section is a multiple of 4 pairs
};

struct QkRopeParams {
  const void* x[2];  // q, k
  void* out[2];
  const void* weight[2];  // may be null
  int64_t stride[2], out_stride[2];
  int heads[2];
  float eps;
  int tokens;
  int dtype, weight_dtype;
  RopeParams rope;
};
cudaError_t launch_qk_rope(const QkRopeParams& p, cudaStream_t stream);

struct BlockAppendParams {
  const void* k;
  const void* v;
  uint8_t* k_cache;
  uint8_t* v_cache;
  float* k_scales;
  float* v_scales;
  const int32_t* btable;
  const int32_t* reqs;
  const int32_t* starts;
  const int32_t* cu_tokens;
  const void* k_weight;
  float eps;
  int entries, tokens, num_kv_heads;
  int page_size, block_size, pages_per_req, num_reqs;
  int64_t num_pages, btable_stride, token_stride;
  int dtype, weight_dtype;
  RopeParams rope;
};
cudaError_t launch_block_append(const BlockAppendParams& p, cudaStream_t stream);

struct BlockDecodeParams {
  const __nv_bfloat16* q;
  const __nv_bfloat16* gate;  // may be null
  __nv_bfloat16* out;
  const uint8_t* k;
  const uint8_t* v;
  const float* k_scales;
  const float* v_scales;
  const int32_t* indices;  // null: column t is token t
  const int32_t* counts;   // may be null
  const int32_t* btable;
  const int32_t* t2r;  // may be null
  float score_scale_log2;  // softmax_scale * log2(e)
  int rows, num_q_heads, num_kv_heads, group;
  int page_size, block_size, pages_per_req, num_reqs;
  int64_t num_pages;
  int topk;  // columns of a row
  int64_t indices_stride, btable_stride;
  // A group above 8 (above 16 where there is much work) goes as head_parts
  // virtual KV heads of part_heads query heads each (the last one may have
  // fewer); a CTA takes cta_heads of the virtual_heads of a row.
  int head_parts, part_heads, virtual_heads, cta_heads;
  // slot / block_size = umulhi(2 slot, block_mul) >> block_shift, exact below
  // 2^31; token / page_size likewise
  uint32_t block_mul, block_shift, page_mul, page_shift;
  // Rows of many columns: units (of a CTA's warps times 16 columns) in the
  // order row, head group, columns, shared evenly by `ctas` CTAs (workspace).
  bool planned;
  struct BlockDecodePlan* plan;  // null: a CTA takes a whole row
  int64_t* prefix;               // [rows + 1] units of one head group before each row
  int* lengths;                  // [rows] columns up to the last valid one
  float* part_o;                 // [2 ctas, cta_heads, part_heads, 128] normalised results of pieces of rows
  float* part_lse;               // [2 ctas, cta_heads, part_heads] their log2-sum-exp2, -inf for none
};
// Columns of a row: they are counted in int32, a CTA's table of slots at a time,
// which may begin up to a table past the last one.
constexpr int kBlockMaxColumns = 0x7fffffff - 2048;
constexpr int kPlanMaxCtas = 1024;
struct BlockDecodePlan {
  int ctas;
  int num_joins[2];                 // rows and head groups of few pieces, and of many
  int4 joins[kPlanMaxCtas];         // row, head group, CTAs of the second and the last piece: the few
                                    // from the front, the many from the back
  int first_row[kPlanMaxCtas + 1];  // row that each CTA begins in
  int64_t cut[kPlanMaxCtas + 1];    // its first unit
};
// Chooses the split and gives the workspace's size; places it in a workspace.
int64_t block_decode_plan(BlockDecodeParams& p);
void block_decode_place(BlockDecodeParams& p, void* workspace);
cudaError_t launch_block_decode(const BlockDecodeParams& p, cudaStream_t stream);

// QSA_B200_OK when the current device is an sm_100 part, else QSA_B200_ERR_DEVICE.
int device_status();

// Top-K entries per work item for a GQA group size (both kernels split rows
// the same way, so the workspace size depends only on the shape), and the
// group sizes of the tensor-core kernel.
int tc_chunk_tokens(int group);
bool tc_supports_group(int group);
// Whether the tensor-core decode merges the chunks of split rows itself, so
// that the split combine is not launched.
bool tc_merges_chunks(const DecodeParams& p);

// Largest group size (Hq / Hkv) the tensor-core kernel handles.
constexpr int kMaxGroupTc = 16;

}  // namespace qsa
