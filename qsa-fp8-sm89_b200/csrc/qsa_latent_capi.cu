// C ABI of the latent cache (declared in include/qsa_b200.h):
// qsa_b200_latent_append, _read, _decode, _prefill. Checks the arguments before
// any device call, fills the launch parameters and launches.
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

// Sizes of a cache, and (used: the call touches it) its tensors.
int check_cache(const qsa_b200_latent_cache& c, bool used, LatentCache* p) {
  if (c.page_size < 1 || c.pages_per_req < 1 || c.num_reqs < 1 || c.num_pages < 1 || c.btable_stride < c.pages_per_req)
    return QSA_B200_ERR_BAD_SHAPE;
  if (c.rope_dim != kLatentRope || c.rank < 128 || c.rank > 512 || c.rank % 128 != 0) return QSA_B200_ERR_UNSUPPORTED;
  if (c.num_pages > kLatentMaxTokens / c.page_size || c.pages_per_req > kLatentMaxTokens / c.page_size)
    return QSA_B200_ERR_UNSUPPORTED;
  if (used) {
    if (!c.codes || !c.rope || !c.scales || !c.btable) return QSA_B200_ERR_NULL_POINTER;
    if (!aligned(c.codes, 16) || !aligned(c.rope, 16) || !aligned(c.scales, 4) || !aligned(c.btable, 4))
      return QSA_B200_ERR_MISALIGNED;
  }
  p->codes = static_cast<uint8_t*>(c.codes);
  p->rope = static_cast<__nv_bfloat16*>(c.rope);
  p->scales = c.scales;
  p->btable = c.btable;
  p->rank = c.rank;
  p->page_size = c.page_size;
  p->pages_per_req = c.pages_per_req;
  p->num_reqs = c.num_reqs;
  p->num_pages = c.num_pages;
  p->btable_stride = c.btable_stride;
  // mul = ceil(2^(31 + shift) / d) with d <= 2^shift: n mul exceeds
  // n 2^(31 + shift) / d by less than n, so n / d is exact for n < 2^31
  p->page_shift = 0;
  while ((1ll << p->page_shift) < c.page_size) ++p->page_shift;
  p->page_mul = (uint32_t)((((uint64_t)1 << (31 + p->page_shift)) + c.page_size - 1) / c.page_size);
  return QSA_B200_OK;
}

int check_tokens(const int32_t* starts, const int32_t* reqs, const int32_t* cu_tokens, int entries, int tokens,
                 LatentTokens* p) {
  if (entries < 0 || tokens < 0 || (!cu_tokens && tokens != entries)) return QSA_B200_ERR_BAD_SHAPE;
  if (entries > 0 && tokens > 0) {
    if (!starts) return QSA_B200_ERR_NULL_POINTER;
    if (!aligned(starts, 4) || !aligned(reqs, 4) || !aligned(cu_tokens, 4)) return QSA_B200_ERR_MISALIGNED;
  }
  *p = {starts, reqs, cu_tokens, entries, tokens};
  return QSA_B200_OK;
}

// A rotation of the cached part: one axis, the logical positions by default.
int check_rotation(const qsa_b200_rotation& r, RopeParams* p) {
  if (!r.table) return QSA_B200_OK;
  if (r.rotary_dim < 16 || r.rotary_dim > kLatentRope || r.rotary_dim % 16 != 0 || r.num_axes != 1)
    return QSA_B200_ERR_UNSUPPORTED;
  if (r.table_len < 1) return QSA_B200_ERR_BAD_SHAPE;
  if (!aligned(r.table, 16) || !aligned(r.positions, 4)) return QSA_B200_ERR_MISALIGNED;
  p->table = r.table;
  p->positions = r.positions;
  p->table_len = r.table_len;
  p->rotary = r.rotary_dim;
  p->interleaved = r.interleaved;
  p->axes = 1;
  return QSA_B200_OK;
}

int check_decode(const qsa_b200_latent_decode_args* a, LatentDecodeParams* p) {
  if (!a) return QSA_B200_ERR_NULL_POINTER;
  *p = LatentDecodeParams{};
  if (a->rows < 0 || a->nodes < 1 || a->heads < 1) return QSA_B200_ERR_BAD_SHAPE;
  if (a->indices && (a->topk < 0 || a->indices_stride < a->topk)) return QSA_B200_ERR_BAD_SHAPE;
  if (a->tree && a->tree_words < (a->nodes + 31) / 32) return QSA_B200_ERR_BAD_SHAPE;
  if (a->heads > 128 || a->nodes > QSA_B200_LATENT_MAX_NODES || (a->indices && (a->nodes > 1 || a->tree)))
    return QSA_B200_ERR_UNSUPPORTED;
  if (a->indices && a->topk > kLatentMaxTokens) return QSA_B200_ERR_UNSUPPORTED;
  if ((int64_t)a->rows * a->nodes * a->heads > 0x7fffffffll) return QSA_B200_ERR_BAD_SHAPE;
  const int st = check_cache(a->cache, a->rows > 0, &p->cache);
  if (st != QSA_B200_OK) return st;
  if (a->rows > 0) {
    if (!a->q || !a->out) return QSA_B200_ERR_NULL_POINTER;
    if (!aligned(a->q, 16) || !aligned(a->out, 16) || !aligned(a->indices, 4) || !aligned(a->counts, 4) ||
        !aligned(a->t2r, 4) || !aligned(a->tree, 4))
      return QSA_B200_ERR_MISALIGNED;
  }
  p->q = static_cast<const __nv_bfloat16*>(a->q);
  p->out = static_cast<__nv_bfloat16*>(a->out);
  p->indices = a->indices;
  p->counts = a->counts;
  p->t2r = a->t2r;
  p->tree = a->nodes > 1 ? a->tree : nullptr;
  p->score_scale_log2 = a->softmax_scale * 1.4426950408889634f;
  p->rows = a->rows;
  p->nodes = a->nodes;
  p->heads = a->heads;
  p->topk = a->topk;
  p->tree_words = a->tree_words;
  p->indices_stride = a->indices_stride;
  return QSA_B200_OK;
}

int launched(cudaError_t e) { return e == cudaSuccess ? QSA_B200_OK : QSA_B200_ERR_LAUNCH; }

}  // namespace
}  // namespace qsa

using namespace qsa;

extern "C" {

int qsa_b200_latent_append(const qsa_b200_latent_append_args* a, qsa_b200_stream_t stream) {
  if (!a) return QSA_B200_ERR_NULL_POINTER;
  LatentAppendParams p = {};
  const bool used = a->entries > 0 && a->tokens > 0;
  int st = check_cache(a->cache, used, &p.cache);
  if (st == QSA_B200_OK) st = check_tokens(a->starts, a->reqs, a->cu_tokens, a->entries, a->tokens, &p.list);
  if (st != QSA_B200_OK) return st;
  if (!dtype_ok(a->input_dtype) || (a->c_weight && !dtype_ok(a->weight_dtype))) return QSA_B200_ERR_UNSUPPORTED;
  if (!(a->eps >= 0.f) || !std::isfinite(a->eps)) return QSA_B200_ERR_BAD_VALUE;
  if (a->c_stride < a->cache.rank || a->r_stride < kLatentRope) return QSA_B200_ERR_BAD_SHAPE;
  st = check_rotation(a->rotation, &p.rope);
  if (st != QSA_B200_OK || !used) return st;
  if (!a->c || !a->r) return QSA_B200_ERR_NULL_POINTER;
  const int64_t elem = dtype_bytes(a->input_dtype);
  if (!aligned(a->c, 16) || !aligned(a->r, 16) || a->c_stride * elem % 16 || a->r_stride * elem % 16 ||
      !aligned(a->c_weight, 16))
    return QSA_B200_ERR_MISALIGNED;
  st = device_status();
  if (st != QSA_B200_OK) return st;
  p.c = a->c;
  p.r = a->r;
  p.c_weight = a->c_weight;
  p.eps = a->eps;
  p.dtype = a->input_dtype;
  p.weight_dtype = a->weight_dtype;
  p.c_stride = a->c_stride;
  p.r_stride = a->r_stride;
  return launched(launch_latent_append(p, reinterpret_cast<cudaStream_t>(stream)));
}

int qsa_b200_latent_read(const qsa_b200_latent_read_args* a, qsa_b200_stream_t stream) {
  if (!a) return QSA_B200_ERR_NULL_POINTER;
  LatentReadParams p = {};
  const bool used = a->entries > 0 && a->tokens > 0;
  int st = check_cache(a->cache, used, &p.cache);
  if (st == QSA_B200_OK) st = check_tokens(a->starts, a->reqs, a->cu_tokens, a->entries, a->tokens, &p.list);
  if (st != QSA_B200_OK) return st;
  if (!dtype_ok(a->output_dtype)) return QSA_B200_ERR_UNSUPPORTED;
  if (!used) return QSA_B200_OK;
  if (!a->c || !a->r) return QSA_B200_ERR_NULL_POINTER;
  if (!aligned(a->c, 16) || !aligned(a->r, 16)) return QSA_B200_ERR_MISALIGNED;
  st = device_status();
  if (st != QSA_B200_OK) return st;
  p.c = a->c;
  p.r = a->r;
  p.dtype = a->output_dtype;
  return launched(launch_latent_read(p, reinterpret_cast<cudaStream_t>(stream)));
}

int64_t qsa_b200_latent_decode_workspace_bytes(const qsa_b200_latent_decode_args* a) {
  LatentDecodeParams p;
  const int st = check_decode(a, &p);
  if (st != QSA_B200_OK) return st;
  return p.rows == 0 ? 0 : latent_decode_plan(p);
}

int qsa_b200_latent_decode(const qsa_b200_latent_decode_args* a, void* workspace, size_t workspace_bytes,
                           qsa_b200_stream_t stream) {
  LatentDecodeParams p;
  int st = check_decode(a, &p);
  if (st != QSA_B200_OK || p.rows == 0) return st;
  st = device_status();
  if (st != QSA_B200_OK) return st;
  const int64_t need = latent_decode_plan(p);
  if (need > 0) {
    if (!workspace || (int64_t)workspace_bytes < need) return QSA_B200_ERR_WORKSPACE;
    if (!aligned(workspace, 256)) return QSA_B200_ERR_MISALIGNED;
    latent_decode_place(p, workspace);
  }
  p.err = error_word();
  p.wait_limit_ns = wait_limit_ns();
  return launched(launch_latent_decode(p, reinterpret_cast<cudaStream_t>(stream)));
}

int qsa_b200_latent_prefill(const qsa_b200_latent_prefill_args* a, qsa_b200_stream_t stream) {
  if (!a) return QSA_B200_ERR_NULL_POINTER;
  if (a->entries < 0 || a->q_tokens < 0 || a->k_tokens < 0 || a->heads < 1 || a->q_head_stride < 192 ||
      a->k_head_stride < 128 || a->v_head_stride < 128 || a->q_stride < 192 || a->k_stride < 128 || a->v_stride < 128 ||
      a->k_rope_stride < kLatentRope)
    return QSA_B200_ERR_BAD_SHAPE;
  if (a->dtype != QSA_B200_DTYPE_BF16 && a->dtype != QSA_B200_DTYPE_F16) return QSA_B200_ERR_UNSUPPORTED;
  if (a->entries == 0 || a->q_tokens == 0) return QSA_B200_OK;
  if (!a->q || !a->out || !a->cu_q || !a->cu_k || (a->k_tokens > 0 && (!a->k || !a->k_rope || !a->v)))
    return QSA_B200_ERR_NULL_POINTER;
  if (!aligned(a->q, 16) || !aligned(a->k, 16) || !aligned(a->k_rope, 16) || !aligned(a->v, 16) || !aligned(a->out, 16) ||
      !aligned(a->cu_q, 4) || !aligned(a->cu_k, 4) || a->q_stride % 8 || a->q_head_stride % 8 || a->k_stride % 8 ||
      a->k_head_stride % 8 || a->v_stride % 8 || a->v_head_stride % 8 || a->k_rope_stride % 8)
    return QSA_B200_ERR_MISALIGNED;
  const int st = device_status();
  if (st != QSA_B200_OK) return st;
  LatentPrefillParams p = {};
  p.q = a->q;
  p.k = a->k;
  p.k_rope = a->k_rope;
  p.v = a->v;
  p.out = a->out;
  p.cu_q = a->cu_q;
  p.cu_k = a->cu_k;
  const float scale = std::fabs(a->softmax_scale) * 1.4426950408889634f;
  p.score_scale_log2 = scale == 0.f ? 0x1p-149f : scale;  // what is masked stays below all else
  p.negative = a->softmax_scale < 0.f ? 1 : 0;
  p.entries = a->entries;
  p.q_tokens = a->q_tokens;
  p.k_tokens = a->k_tokens;
  p.heads = a->heads;
  p.causal = a->causal;
  p.dtype = a->dtype;
  p.q_stride = a->q_stride;
  p.q_head_stride = a->q_head_stride;
  p.k_stride = a->k_stride;
  p.k_head_stride = a->k_head_stride;
  p.v_stride = a->v_stride;
  p.v_head_stride = a->v_head_stride;
  p.k_rope_stride = a->k_rope_stride;
  p.err = error_word();
  p.wait_limit_ns = wait_limit_ns();
  return launched(launch_latent_prefill(p, reinterpret_cast<cudaStream_t>(stream)));
}

}  // extern "C"
