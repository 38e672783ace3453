// torch.ops.qsa_b200.{qk_rope, block_append, block_decode}: the block-scaled
// cache's operators over the C ABI of libqsa_b200.so. Like the other operators
// they check dtypes, devices and layouts, take the current CUDA stream and
// allocate outputs and workspace through PyTorch's caching allocator; CUDA
// tensors only.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <optional>
#include <tuple>

#include "../../include/qsa_b200.h"

namespace {

using OptTensor = std::optional<at::Tensor>;
using OptInts = std::optional<std::vector<int64_t>>;

int32_t dtype_code(const at::Tensor& t, const char* name) {
  if (t.scalar_type() == at::kBFloat16) return QSA_B200_DTYPE_BF16;
  if (t.scalar_type() == at::kHalf) return QSA_B200_DTYPE_F16;
  TORCH_CHECK(t.scalar_type() == at::kFloat, name, " must be bfloat16, float16 or float32, got ", t.scalar_type());
  return QSA_B200_DTYPE_F32;
}

void check_device(const at::Tensor& t, const at::Tensor& ref, const char* name) {
  TORCH_CHECK(t.device() == ref.device(), name, " is on ", t.device(), ", expected ", ref.device());
}

int32_t checked_int32(int64_t x, const char* name) {
  TORCH_CHECK(x >= INT32_MIN && x <= INT32_MAX, name, " is ", x, ", past 32 bits");
  return (int32_t)x;
}

// [tokens, heads, D] with contiguous heads; returns the token stride.
int64_t check_heads(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.dim() == 3 && t.stride(2) == 1 && (t.size(1) == 1 || t.stride(1) == t.size(2)), name,
              " must be [tokens, heads, D] with contiguous heads");
  return t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2);
}

const int32_t* int32_list(const OptTensor& t, const at::Tensor& ref, int64_t n, const char* name) {
  if (!t) return nullptr;
  TORCH_CHECK(t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == n && t->is_contiguous(), name,
              " must be contiguous int32 [", n, "]");
  check_device(*t, ref, name);
  return t->data_ptr<int32_t>();
}

const void* norm_weight(const OptTensor& w, const at::Tensor& ref, const char* name, int32_t& dtype) {
  if (!w) return nullptr;
  TORCH_CHECK(w->dim() == 1 && w->size(0) == ref.size(2) && w->is_contiguous(), name, " must be contiguous [D]");
  check_device(*w, ref, name);
  dtype = dtype_code(*w, name);
  return w->data_ptr();
}

void fill_rotation(qsa_b200_rotation& r, const OptTensor& table, const OptTensor& positions, bool interleaved,
                   const OptInts& sections, const at::Tensor& x, bool own_positions) {
  TORCH_CHECK(table || (!positions && !sections), "positions and sections belong to a rotation table");
  if (!table) return;
  TORCH_CHECK(table->scalar_type() == at::kFloat && table->dim() == 2 && table->is_contiguous(),
              "table must be contiguous float32 [positions, rotary_dim]");
  check_device(*table, x, "table");
  r.table = table->data_ptr<float>();
  r.table_len = checked_int32(table->size(0), "the table's length");
  r.rotary_dim = checked_int32(table->size(1), "rotary_dim");
  r.interleaved = interleaved ? 1 : 0;
  r.num_axes = 1;
  if (sections) {
    TORCH_CHECK(!sections->empty() && sections->size() <= QSA_B200_ROPE_MAX_AXES, "sections must name 1 to ",
                QSA_B200_ROPE_MAX_AXES, " axes");
    TORCH_CHECK(positions, "sections need positions");
    r.num_axes = (int32_t)sections->size();
    for (size_t i = 0; i < sections->size(); ++i) r.sections[i] = checked_int32((*sections)[i], "a section");
  }
  TORCH_CHECK(positions || own_positions, "a rotation table needs positions");
  if (!positions) return;
  const int64_t tokens = x.size(0);
  TORCH_CHECK(positions->scalar_type() == at::kInt, "positions must be int32, got ", positions->scalar_type());
  check_device(*positions, x, "positions");
  const bool flat = positions->dim() == 1 && r.num_axes == 1;
  TORCH_CHECK(flat || (positions->dim() == 2 && positions->size(0) == r.num_axes),
              "positions must be [tokens], or [axes, tokens] with a section for each axis");
  TORCH_CHECK(positions->size(-1) == tokens && (tokens <= 1 || positions->stride(-1) == 1),
              "positions must name every token, with unit stride");
  r.positions = positions->data_ptr<int32_t>();
  r.axis_stride = flat || positions->size(0) == 1 ? tokens : positions->stride(0);
}

void run_qk_rope(const at::Tensor& q, const OptTensor& k, const OptTensor& table, const OptTensor& positions,
                 const OptTensor& q_weight, const OptTensor& k_weight, double eps, bool interleaved,
                 const OptInts& sections, at::Tensor& q_out, const OptTensor& k_out) {
  TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
  qsa_b200_qk_rope_args a = {};
  a.dtype = dtype_code(q, "q");
  a.q_stride = check_heads(q, "q");
  a.q_out_stride = check_heads(q_out, "q_out");
  TORCH_CHECK(q_out.sizes() == q.sizes() && q_out.scalar_type() == q.scalar_type(), "q_out must have q's shape and dtype");
  check_device(q_out, q, "q_out");
  if (k) {
    a.k_stride = check_heads(*k, "k");
    a.k_out_stride = check_heads(*k_out, "k_out");
    TORCH_CHECK(k->scalar_type() == q.scalar_type() && k->size(0) == q.size(0) && k->size(2) == q.size(2),
                "k must have q's dtype, tokens and head_dim");
    TORCH_CHECK(k_out->sizes() == k->sizes() && k_out->scalar_type() == k->scalar_type(),
                "k_out must have k's shape and dtype");
    check_device(*k, q, "k");
    check_device(*k_out, q, "k_out");
    a.k = k->data_ptr();
    a.k_out = k_out->data_ptr();
    a.num_kv_heads = checked_int32(k->size(1), "k's heads");
  }
  int32_t kw_dtype = 0;
  a.q_weight = norm_weight(q_weight, q, "q_weight", a.weight_dtype);
  a.k_weight = norm_weight(k_weight, q, "k_weight", kw_dtype);
  TORCH_CHECK(!k_weight || k, "k_weight needs k");
  TORCH_CHECK(!q_weight || !k_weight || kw_dtype == a.weight_dtype, "q_weight and k_weight must have one dtype");
  if (k_weight) a.weight_dtype = kw_dtype;
  fill_rotation(a.rope, table, positions, interleaved, sections, q, false);
  a.q = q.data_ptr();
  a.q_out = q_out.data_ptr();
  a.eps = (float)eps;
  a.tokens = checked_int32(q.size(0), "tokens");
  a.num_q_heads = checked_int32(q.size(1), "q's heads");
  a.head_dim = checked_int32(q.size(2), "head_dim");
  c10::cuda::CUDAGuard guard(q.device());
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(q.device().index()).stream();
  const int st = qsa_b200_qk_rope(&a, reinterpret_cast<qsa_b200_stream_t>(stream));
  TORCH_CHECK(st == QSA_B200_OK, "qsa_b200_qk_rope failed: ", qsa_b200_status_string(st));
}

std::tuple<at::Tensor, at::Tensor> qk_rope(const at::Tensor& q, const OptTensor& k, const OptTensor& table,
                                           const OptTensor& positions, const OptTensor& q_weight,
                                           const OptTensor& k_weight, double eps, bool interleaved,
                                           const OptInts& sections) {
  at::Tensor q_out = at::empty(q.sizes(), q.options());
  OptTensor k_out;
  if (k) k_out = at::empty(k->sizes(), k->options());
  run_qk_rope(q, k, table, positions, q_weight, k_weight, eps, interleaved, sections, q_out, k_out);
  return {q_out, k_out ? *k_out : at::empty({0}, q.options())};
}

void qk_rope_out(const at::Tensor& q, const OptTensor& k, const OptTensor& table, const OptTensor& positions,
                 const OptTensor& q_weight, const OptTensor& k_weight, double eps, bool interleaved,
                 const OptInts& sections, at::Tensor& q_out, const OptTensor& k_out) {
  TORCH_CHECK(k.has_value() == k_out.has_value(), "k and k_out go together");
  run_qk_rope(q, k, table, positions, q_weight, k_weight, eps, interleaved, sections, q_out, k_out);
}

// The caches and their scales; returns tokens per block.
int64_t check_caches(const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& k_scales,
                     const at::Tensor& v_scales, const at::Tensor& ref) {
  TORCH_CHECK(k_cache.scalar_type() == at::kFloat8_e4m3fn || k_cache.scalar_type() == at::kByte,
              "k_cache must be float8_e4m3fn (or its uint8 bytes)");
  TORCH_CHECK(v_cache.scalar_type() == k_cache.scalar_type(), "v_cache must have k_cache's dtype");
  TORCH_CHECK(k_cache.dim() == 4 && k_cache.is_contiguous() && v_cache.sizes() == k_cache.sizes() &&
                  v_cache.is_contiguous(),
              "k_cache / v_cache must be contiguous [pages, P, Hkv, D]");
  TORCH_CHECK(k_scales.scalar_type() == at::kFloat && v_scales.scalar_type() == at::kFloat, "scales must be float32");
  TORCH_CHECK(k_scales.dim() == 3 && k_scales.is_contiguous() && v_scales.sizes() == k_scales.sizes() &&
                  v_scales.is_contiguous() && k_scales.size(0) == k_cache.size(0) &&
                  k_scales.size(2) == k_cache.size(2),
              "k_scales / v_scales must be contiguous [pages, P / block, Hkv]");
  TORCH_CHECK(k_scales.size(1) > 0 && k_cache.size(1) % k_scales.size(1) == 0, "a page of ", k_cache.size(1),
              " tokens does not split into ", k_scales.size(1), " blocks");
  check_device(k_cache, ref, "k_cache");
  check_device(v_cache, ref, "v_cache");
  check_device(k_scales, ref, "k_scales");
  check_device(v_scales, ref, "v_scales");
  return k_cache.size(1) / k_scales.size(1);
}

void check_btable(const at::Tensor& btable, const at::Tensor& ref) {
  TORCH_CHECK(btable.scalar_type() == at::kInt && btable.dim() == 2 && (btable.size(1) <= 1 || btable.stride(1) == 1),
              "btable must be int32 [num_reqs, pages_per_req] with unit column stride");
  check_device(btable, ref, "btable");
}

int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

void block_append(const at::Tensor& k_new, const at::Tensor& v_new, at::Tensor& k_cache, at::Tensor& v_cache,
                  at::Tensor& k_scales, at::Tensor& v_scales, const at::Tensor& btable, const at::Tensor& starts,
                  const OptTensor& reqs, const OptTensor& cu_tokens, const OptTensor& table,
                  const OptTensor& positions, const OptTensor& k_weight, double eps, bool interleaved,
                  const OptInts& sections) {
  TORCH_CHECK(k_new.is_cuda(), "k_new must be a CUDA tensor");
  qsa_b200_block_append_args a = {};
  a.input_dtype = dtype_code(k_new, "k_new");
  a.token_stride = check_heads(k_new, "k_new");
  TORCH_CHECK(v_new.scalar_type() == k_new.scalar_type() && v_new.sizes() == k_new.sizes() &&
                  check_heads(v_new, "v_new") == a.token_stride,
              "v_new must have k_new's dtype, shape and strides");
  check_device(v_new, k_new, "v_new");
  a.block_size = checked_int32(check_caches(k_cache, v_cache, k_scales, v_scales, k_new), "the block");
  TORCH_CHECK(k_cache.size(2) == k_new.size(1) && k_cache.size(3) == k_new.size(2),
              "heads / head_dim of the new rows and the cache differ");
  check_btable(btable, k_new);
  TORCH_CHECK(starts.dim() == 1, "starts must be int32 [entries]");
  const int64_t n = starts.size(0);
  a.starts = int32_list(starts, k_new, n, "starts");
  a.reqs = int32_list(reqs, k_new, n, "reqs");
  a.cu_tokens = int32_list(cu_tokens, k_new, n + 1, "cu_tokens");
  TORCH_CHECK(cu_tokens || n == k_new.size(0), "without cu_tokens every entry has one token: ", n, " entries, ",
              k_new.size(0), " tokens");
  TORCH_CHECK(reqs || n <= btable.size(0), "btable has ", btable.size(0), " rows for ", n, " entries");
  a.k_weight = norm_weight(k_weight, k_new, "k_weight", a.weight_dtype);
  fill_rotation(a.rope, table, positions, interleaved, sections, k_new, true);
  a.k = k_new.data_ptr();
  a.v = v_new.data_ptr();
  a.k_cache = k_cache.data_ptr();
  a.v_cache = v_cache.data_ptr();
  a.k_scales = k_scales.data_ptr<float>();
  a.v_scales = v_scales.data_ptr<float>();
  a.btable = btable.data_ptr<int32_t>();
  a.eps = (float)eps;
  a.entries = checked_int32(n, "entries");
  a.tokens = checked_int32(k_new.size(0), "tokens");
  a.num_kv_heads = checked_int32(k_cache.size(2), "heads");
  a.head_dim = checked_int32(k_cache.size(3), "head_dim");
  a.page_size = checked_int32(k_cache.size(1), "the page");
  a.pages_per_req = checked_int32(btable.size(1), "pages_per_req");
  a.num_reqs = checked_int32(btable.size(0), "num_reqs");
  a.num_pages = k_cache.size(0);
  a.btable_stride = row_stride(btable);
  c10::cuda::CUDAGuard guard(k_new.device());
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(k_new.device().index()).stream();
  const int st = qsa_b200_block_append(&a, reinterpret_cast<qsa_b200_stream_t>(stream));
  TORCH_CHECK(st == QSA_B200_OK, "qsa_b200_block_append failed: ", qsa_b200_status_string(st));
}

void block_decode_out(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                      const at::Tensor& k_scales, const at::Tensor& v_scales, const at::Tensor& btable,
                      const OptTensor& t2r, const OptTensor& indices, const OptTensor& gate, const OptTensor& counts,
                      double softmax_scale, at::Tensor& out) {
  TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 && out.scalar_type() == at::kBFloat16, "q and out must be bfloat16");
  TORCH_CHECK(q.dim() == 3 && q.is_contiguous(), "q must be contiguous [rows, Hq, D]");
  TORCH_CHECK(out.sizes() == q.sizes() && out.is_contiguous(), "out must be contiguous and shaped like q");
  check_device(out, q, "out");
  qsa_b200_block_decode_args a = {};
  a.block_size = checked_int32(check_caches(k_cache, v_cache, k_scales, v_scales, q), "the block");
  TORCH_CHECK(k_cache.size(3) == q.size(2), "head_dim of q (", q.size(2), ") and cache (", k_cache.size(3), ") differ");
  if (gate) {
    TORCH_CHECK(gate->scalar_type() == at::kBFloat16 && gate->sizes() == q.sizes() && gate->is_contiguous(),
                "gate must be contiguous bfloat16 and shaped like q");
    check_device(*gate, q, "gate");
    a.gate = gate->data_ptr();
  }
  check_btable(btable, q);
  const int64_t rows = q.size(0);
  if (indices) {
    TORCH_CHECK(indices->scalar_type() == at::kInt && indices->dim() == 2 && indices->size(0) == rows &&
                    (indices->size(1) <= 1 || indices->stride(1) == 1),
                "indices must be int32 [", rows, ", K] with unit column stride");
    check_device(*indices, q, "indices");
    a.topk = checked_int32(indices->size(1), "K");
    a.indices_stride = row_stride(*indices);
    // an empty list of columns is still a list
    static const int32_t none = 0;
    a.indices = indices->numel() > 0 ? indices->data_ptr<int32_t>() : &none;
  }
  a.t2r = int32_list(t2r, q, rows, "t2r");
  a.counts = int32_list(counts, q, rows, "counts");
  a.q = q.data_ptr();
  a.k_cache = k_cache.data_ptr();
  a.v_cache = v_cache.data_ptr();
  a.k_scales = k_scales.data_ptr<float>();
  a.v_scales = v_scales.data_ptr<float>();
  a.btable = btable.data_ptr<int32_t>();
  a.out = out.data_ptr();
  a.softmax_scale = (float)softmax_scale;
  a.rows = checked_int32(rows, "rows");
  a.num_q_heads = checked_int32(q.size(1), "q's heads");
  a.num_kv_heads = checked_int32(k_cache.size(2), "heads");
  a.head_dim = checked_int32(q.size(2), "head_dim");
  a.page_size = checked_int32(k_cache.size(1), "the page");
  a.pages_per_req = checked_int32(btable.size(1), "pages_per_req");
  a.num_reqs = checked_int32(btable.size(0), "num_reqs");
  a.num_pages = k_cache.size(0);
  a.btable_stride = row_stride(btable);
  c10::cuda::CUDAGuard guard(q.device());
  const int64_t need = qsa_b200_block_decode_workspace_bytes(&a);
  TORCH_CHECK(need >= 0, "qsa_b200_block_decode failed: ", qsa_b200_status_string((int)need));
  at::Tensor workspace;
  if (need > 0) workspace = at::empty({need}, q.options().dtype(at::kByte));
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(q.device().index()).stream();
  const int st = qsa_b200_block_decode(&a, need > 0 ? workspace.data_ptr() : nullptr, (size_t)need,
                                       reinterpret_cast<qsa_b200_stream_t>(stream));
  TORCH_CHECK(st == QSA_B200_OK, "qsa_b200_block_decode failed: ", qsa_b200_status_string(st));
}

at::Tensor block_decode(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                        const at::Tensor& k_scales, const at::Tensor& v_scales, const at::Tensor& btable,
                        const OptTensor& t2r, const OptTensor& indices, const OptTensor& gate,
                        const OptTensor& counts, double softmax_scale) {
  at::Tensor out = at::empty(q.sizes(), q.options());
  block_decode_out(q, k_cache, v_cache, k_scales, v_scales, btable, t2r, indices, gate, counts, softmax_scale, out);
  return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(qsa_b200, m) {
  m.def(
      "qk_rope(Tensor q, Tensor? k, Tensor? table, Tensor? positions, Tensor? q_weight, Tensor? k_weight, float eps, "
      "bool interleaved, int[]? sections) -> (Tensor, Tensor)");
  m.def(
      "qk_rope_out(Tensor q, Tensor? k, Tensor? table, Tensor? positions, Tensor? q_weight, Tensor? k_weight, "
      "float eps, bool interleaved, int[]? sections, Tensor(a!) q_out, Tensor(b!)? k_out) -> ()");
  m.def(
      "block_append(Tensor k_new, Tensor v_new, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scales, "
      "Tensor(d!) v_scales, Tensor btable, Tensor starts, Tensor? reqs, Tensor? cu_tokens, Tensor? table, "
      "Tensor? positions, Tensor? k_weight, float eps, bool interleaved, int[]? sections) -> ()");
  m.def(
      "block_decode(Tensor q, Tensor k_cache, Tensor v_cache, Tensor k_scales, Tensor v_scales, Tensor btable, "
      "Tensor? t2r, Tensor? indices, Tensor? gate, Tensor? counts, float softmax_scale) -> Tensor");
  m.def(
      "block_decode_out(Tensor q, Tensor k_cache, Tensor v_cache, Tensor k_scales, Tensor v_scales, Tensor btable, "
      "Tensor? t2r, Tensor? indices, Tensor? gate, Tensor? counts, float softmax_scale, Tensor(a!) out) -> ()");
}

TORCH_LIBRARY_IMPL(qsa_b200, CUDA, m) {
  m.impl("qk_rope", &qk_rope);
  m.impl("qk_rope_out", &qk_rope_out);
  m.impl("block_append", &block_append);
  m.impl("block_decode", &block_decode);
  m.impl("block_decode_out", &block_decode_out);
}
