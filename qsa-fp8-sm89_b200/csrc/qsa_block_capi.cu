// C ABI of the block-scaled cache (declared in include/qsa_b200.h):
// qsa_b200_qk_rope, qsa_b200_block_append, qsa_b200_block_decode. Checks the
// arguments before any device call, fills the launch parameters and launches.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "../../include/qsa_b200.h"
#include "qsa_internal.h"

namespace qsa {
namespace {

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
bool dtype_ok(int d) { return d >= QSA_B200_DTYPE_BF16 && d <= QSA_B200_DTYPE_F32; }
int64_t dtype_bytes(int d) { return d == QSA_B200_DTYPE_F32 ? 4 : 2; }

// Checks a rotation and fills its launch parameters. own_positions: the
// kernel has positions of its own where none are given.
int check_rotation(const qsa_b200_rotation& r, int64_t tokens, bool own_positions, RopeParams* p) {
  *p = RopeParams{};
  if (!r.table) return QSA_B200_OK;
  if (r.rotary_dim < 16 || r.rotary_dim > 128 || r.rotary_dim % 16 != 0) return QSA_B200_ERR_UNSUPPORTED;
  if (r.num_axes < 1 || r.num_axes > QSA_B200_ROPE_MAX_AXES) return QSA_B200_ERR_UNSUPPORTED;
  if (r.table_len < 1) return QSA_B200_ERR_BAD_SHAPE;
  if (!r.positions && (!own_positions || r.num_axes > 1)) return QSA_B200_ERR_NULL_POINTER;
  int end = 0;
  p->quads = 1;
  for (int a = 0; a < r.num_axes; ++a) {
    const int n = r.num_axes == 1 ? r.rotary_dim / 2 : r.sections[a];
    if (n < 0 || n > r.rotary_dim / 2) return QSA_B200_ERR_BAD_SHAPE;
    end += n;
    p->ends[a] = end;
    if (n % 4 != 0) p->quads = 0;
  }
  if (end != r.rotary_dim / 2) return QSA_B200_ERR_BAD_SHAPE;
  if (r.num_axes > 1 && r.axis_stride < tokens) return QSA_B200_ERR_BAD_SHAPE;
  if (!aligned(r.table, 16) || !aligned(r.positions, 4)) return QSA_B200_ERR_MISALIGNED;
  p->table = r.table;
  p->positions = r.positions;
  p->axis_stride = r.axis_stride;
  p->table_len = r.table_len;
  p->rotary = r.rotary_dim;
  p->interleaved = r.interleaved;
  p->axes = r.num_axes;
  return QSA_B200_OK;
}

int check_pages(int32_t page_size, int32_t block_size, int32_t pages_per_req, int32_t num_reqs, int64_t num_pages,
                int64_t btable_stride) {
  if (page_size < 1 || block_size < 1 || page_size % block_size != 0 || pages_per_req < 1 || num_reqs < 1 ||
      num_pages < 1 || btable_stride < pages_per_req)
    return QSA_B200_ERR_BAD_SHAPE;
  return QSA_B200_OK;
}

int check_block_decode(const qsa_b200_block_decode_args* a, BlockDecodeParams* p) {
  if (!a) return QSA_B200_ERR_NULL_POINTER;
  const int st = check_pages(a->page_size, a->block_size, a->pages_per_req, a->num_reqs, a->num_pages, a->btable_stride);
  if (st != QSA_B200_OK) return st;
  if (a->rows < 0 || a->num_q_heads < 1 || a->num_kv_heads < 1 || a->num_q_heads % a->num_kv_heads != 0)
    return QSA_B200_ERR_BAD_SHAPE;
  if (a->indices && (a->topk < 0 || a->indices_stride < a->topk)) return QSA_B200_ERR_BAD_SHAPE;
  if (a->head_dim != 128 || a->num_q_heads / a->num_kv_heads > 32 || a->num_kv_heads > kBlockMaxHeads)
    return QSA_B200_ERR_UNSUPPORTED;
  // token slots, columns and the tiles of a row over its (up to 4 virtual) KV
  // heads are held as int32
  const int64_t columns = a->indices ? a->topk : (int64_t)a->pages_per_req * a->page_size;
  if (a->num_pages > 0x7fffffffll / a->page_size || columns > kBlockMaxColumns ||
      (columns / 128 + 1) * 4 > 0x7fffffffll / a->num_kv_heads)
    return QSA_B200_ERR_UNSUPPORTED;
  if ((int64_t)a->rows * a->num_q_heads > 0x7fffffffll) return QSA_B200_ERR_BAD_SHAPE;
  if (a->rows > 0) {
    if (!a->q || !a->k_cache || !a->v_cache || !a->k_scales || !a->v_scales || !a->btable || !a->out)
      return QSA_B200_ERR_NULL_POINTER;
    if (!aligned(a->q, 16) || !aligned(a->k_cache, 16) || !aligned(a->v_cache, 16) || !aligned(a->out, 16) ||
        !aligned(a->gate, 16) || !aligned(a->k_scales, 4) || !aligned(a->v_scales, 4) || !aligned(a->indices, 4) ||
        !aligned(a->counts, 4) || !aligned(a->btable, 4) || !aligned(a->t2r, 4))
      return QSA_B200_ERR_MISALIGNED;
  }
  *p = BlockDecodeParams{};
  p->q = static_cast<const __nv_bfloat16*>(a->q);
  p->gate = static_cast<const __nv_bfloat16*>(a->gate);
  p->out = static_cast<__nv_bfloat16*>(a->out);
  p->k = static_cast<const uint8_t*>(a->k_cache);
  p->v = static_cast<const uint8_t*>(a->v_cache);
  p->k_scales = a->k_scales;
  p->v_scales = a->v_scales;
  p->indices = a->indices;
  p->counts = a->counts;
  p->btable = a->btable;
  p->t2r = a->t2r;
  p->score_scale_log2 = a->softmax_scale * 1.4426950408889634f;
  p->rows = a->rows;
  p->num_q_heads = a->num_q_heads;
  p->num_kv_heads = a->num_kv_heads;
  p->group = a->num_q_heads / a->num_kv_heads;
  p->page_size = a->page_size;
  p->block_size = a->block_size;
  p->pages_per_req = a->pages_per_req;
  p->num_reqs = a->num_reqs;
  p->num_pages = a->num_pages;
  p->topk = a->indices ? a->topk : a->pages_per_req * a->page_size;
  p->indices_stride = a->indices_stride;
  p->btable_stride = a->btable_stride;
  return QSA_B200_OK;
}

}  // namespace
}  // namespace qsa

using namespace qsa;

extern "C" {

int qsa_b200_qk_rope(const qsa_b200_qk_rope_args* a, qsa_b200_stream_t stream) {
  if (!a) return QSA_B200_ERR_NULL_POINTER;
  if (a->tokens < 0 || a->num_q_heads < 1 || a->num_kv_heads < 0 || (a->k && a->num_kv_heads < 1))
    return QSA_B200_ERR_BAD_SHAPE;
  if (a->head_dim != 128 || !dtype_ok(a->dtype) || ((a->q_weight || a->k_weight) && !dtype_ok(a->weight_dtype)) ||
      a->num_q_heads > kBlockMaxHeads || a->num_kv_heads > kBlockMaxHeads)
    return QSA_B200_ERR_UNSUPPORTED;
  if (!(a->eps >= 0.f) || !std::isfinite(a->eps)) return QSA_B200_ERR_BAD_VALUE;
  const int64_t q_row = (int64_t)a->num_q_heads * 128, k_row = (int64_t)a->num_kv_heads * 128;
  if (a->q_stride < q_row || a->q_out_stride < q_row || (a->k && (a->k_stride < k_row || a->k_out_stride < k_row)))
    return QSA_B200_ERR_BAD_SHAPE;
  QkRopeParams p = {};
  int st = check_rotation(a->rope, a->tokens, false, &p.rope);
  if (st != QSA_B200_OK) return st;
  if (a->tokens == 0) return QSA_B200_OK;
  if (!a->q || !a->q_out || (a->k && !a->k_out)) return QSA_B200_ERR_NULL_POINTER;
  const int64_t elem = dtype_bytes(a->dtype);
  if (!aligned(a->q, 16) || !aligned(a->q_out, 16) || (a->q_stride * elem) % 16 || (a->q_out_stride * elem) % 16 ||
      !aligned(a->q_weight, 16) || !aligned(a->k_weight, 16))
    return QSA_B200_ERR_MISALIGNED;
  if (a->k && (!aligned(a->k, 16) || !aligned(a->k_out, 16) || (a->k_stride * elem) % 16 || (a->k_out_stride * elem) % 16))
    return QSA_B200_ERR_MISALIGNED;
  st = device_status();
  if (st != QSA_B200_OK) return st;
  p.x[0] = a->q, p.x[1] = a->k;
  p.out[0] = a->q_out, p.out[1] = a->k_out;
  p.weight[0] = a->q_weight, p.weight[1] = a->k_weight;
  p.stride[0] = a->q_stride, p.stride[1] = a->k_stride;
  p.out_stride[0] = a->q_out_stride, p.out_stride[1] = a->k_out_stride;
  p.heads[0] = a->num_q_heads, p.heads[1] = a->k ? a->num_kv_heads : 0;
  p.eps = a->eps;
  p.tokens = a->tokens;
  p.dtype = a->dtype;
  p.weight_dtype = a->weight_dtype;
  return launch_qk_rope(p, reinterpret_cast<cudaStream_t>(stream)) == cudaSuccess ? QSA_B200_OK : QSA_B200_ERR_LAUNCH;
}

int qsa_b200_block_append(const qsa_b200_block_append_args* a, qsa_b200_stream_t stream) {
  if (!a) return QSA_B200_ERR_NULL_POINTER;
  int st = check_pages(a->page_size, a->block_size, a->pages_per_req, a->num_reqs, a->num_pages, a->btable_stride);
  if (st != QSA_B200_OK) return st;
  if (a->entries < 0 || a->tokens < 0 || a->num_kv_heads < 1 || (!a->cu_tokens && a->tokens != a->entries))
    return QSA_B200_ERR_BAD_SHAPE;
  if (a->head_dim != 128 || !dtype_ok(a->input_dtype) || (a->k_weight && !dtype_ok(a->weight_dtype)) ||
      a->num_kv_heads > kBlockMaxHeads)
    return QSA_B200_ERR_UNSUPPORTED;
  if (!(a->eps >= 0.f) || !std::isfinite(a->eps)) return QSA_B200_ERR_BAD_VALUE;
  if (a->token_stride < (int64_t)a->num_kv_heads * 128) return QSA_B200_ERR_BAD_SHAPE;
  BlockAppendParams p = {};
  st = check_rotation(a->rope, a->tokens, true, &p.rope);
  if (st != QSA_B200_OK) return st;
  if (a->entries == 0 || a->tokens == 0) return QSA_B200_OK;
  if (!a->k || !a->v || !a->k_cache || !a->v_cache || !a->k_scales || !a->v_scales || !a->btable || !a->starts)
    return QSA_B200_ERR_NULL_POINTER;
  if (!aligned(a->k, 16) || !aligned(a->v, 16) || !aligned(a->k_cache, 16) || !aligned(a->v_cache, 16) ||
      (a->token_stride * dtype_bytes(a->input_dtype)) % 16 || !aligned(a->k_weight, 16) || !aligned(a->k_scales, 4) ||
      !aligned(a->v_scales, 4) || !aligned(a->btable, 4) || !aligned(a->reqs, 4) || !aligned(a->starts, 4) ||
      !aligned(a->cu_tokens, 4))
    return QSA_B200_ERR_MISALIGNED;
  st = device_status();
  if (st != QSA_B200_OK) return st;
  p.k = a->k;
  p.v = a->v;
  p.k_cache = static_cast<uint8_t*>(a->k_cache);
  p.v_cache = static_cast<uint8_t*>(a->v_cache);
  p.k_scales = a->k_scales;
  p.v_scales = a->v_scales;
  p.btable = a->btable;
  p.reqs = a->reqs;
  p.starts = a->starts;
  p.cu_tokens = a->cu_tokens;
  p.k_weight = a->k_weight;
  p.eps = a->eps;
  p.entries = a->entries;
  p.tokens = a->tokens;
  p.num_kv_heads = a->num_kv_heads;
  p.page_size = a->page_size;
  p.block_size = a->block_size;
  p.pages_per_req = a->pages_per_req;
  p.num_reqs = a->num_reqs;
  p.num_pages = a->num_pages;
  p.btable_stride = a->btable_stride;
  p.token_stride = a->token_stride;
  p.dtype = a->input_dtype;
  p.weight_dtype = a->weight_dtype;
  return launch_block_append(p, reinterpret_cast<cudaStream_t>(stream)) == cudaSuccess ? QSA_B200_OK
                                                                                      : QSA_B200_ERR_LAUNCH;
}

int64_t qsa_b200_block_decode_workspace_bytes(const qsa_b200_block_decode_args* a) {
  BlockDecodeParams p;
  const int st = check_block_decode(a, &p);
  if (st != QSA_B200_OK) return st;
  return p.rows == 0 ? 0 : block_decode_plan(p);
}

int qsa_b200_block_decode(const qsa_b200_block_decode_args* a, void* workspace, size_t workspace_bytes,
                          qsa_b200_stream_t stream) {
  BlockDecodeParams p;
  int st = check_block_decode(a, &p);
  if (st != QSA_B200_OK) return st;
  if (p.rows == 0) return QSA_B200_OK;
  st = device_status();
  if (st != QSA_B200_OK) return st;
  const int64_t need = block_decode_plan(p);
  if (need > 0) {
    if (!workspace || (int64_t)workspace_bytes < need) return QSA_B200_ERR_WORKSPACE;
    if (!aligned(workspace, 256)) return QSA_B200_ERR_MISALIGNED;
    block_decode_place(p, workspace);
  }
  return launch_block_decode(p, reinterpret_cast<cudaStream_t>(stream)) == cudaSuccess ? QSA_B200_OK
                                                                                      : QSA_B200_ERR_LAUNCH;
}

}  // extern "C"
