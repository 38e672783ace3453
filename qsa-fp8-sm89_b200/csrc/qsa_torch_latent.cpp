// torch.ops.qsa_b200.{latent_append, latent_read, latent_decode, latent_prefill}:
// the latent cache's operators over the C ABI of libqsa_b200.so. Like the other
// operators they check dtypes, devices and layouts, take the current CUDA stream
// and allocate outputs and workspace through PyTorch's caching allocator; CUDA
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

int32_t dtype_code(at::ScalarType t, const char* name) {
  if (t == at::kBFloat16) return QSA_B200_DTYPE_BF16;
  if (t == at::kHalf) return QSA_B200_DTYPE_F16;
  TORCH_CHECK(t == at::kFloat, name, " must be bfloat16, float16 or float32, got ", t);
  return QSA_B200_DTYPE_F32;
}

void check_device(const at::Tensor& t, const at::Tensor& ref, const char* name) {
  TORCH_CHECK(t.device() == ref.device(), name, " is on ", t.device(), ", expected ", ref.device());
}

int32_t checked_int32(int64_t x, const char* name) {
  TORCH_CHECK(x >= INT32_MIN && x <= INT32_MAX, name, " is ", x, ", past 32 bits");
  return (int32_t)x;
}

const int32_t* int32_list(const OptTensor& t, const at::Tensor& ref, int64_t n, const char* name) {
  if (!t) return nullptr;
  TORCH_CHECK(t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == n && t->is_contiguous(), name,
              " must be contiguous int32 [", n, "]");
  check_device(*t, ref, name);
  return t->data_ptr<int32_t>();
}

int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

qsa_b200_latent_cache check_cache(const at::Tensor& codes, const at::Tensor& rope, const at::Tensor& scales,
                                  const at::Tensor& btable) {
  TORCH_CHECK(codes.is_cuda(), "codes must be a CUDA tensor");
  TORCH_CHECK(codes.scalar_type() == at::kFloat8_e4m3fn || codes.scalar_type() == at::kByte,
              "codes must be float8_e4m3fn (or its uint8 bytes)");
  TORCH_CHECK(codes.dim() == 3 && codes.is_contiguous(), "codes must be contiguous [pages, P, rank]");
  TORCH_CHECK(rope.scalar_type() == at::kBFloat16 && rope.dim() == 3 && rope.is_contiguous() &&
                  rope.size(0) == codes.size(0) && rope.size(1) == codes.size(1),
              "rope must be contiguous bfloat16 [pages, P, rope_dim]");
  TORCH_CHECK(scales.scalar_type() == at::kFloat && scales.dim() == 2 && scales.is_contiguous() &&
                  scales.size(0) == codes.size(0) && scales.size(1) == codes.size(1),
              "scales must be contiguous float32 [pages, P]");
  TORCH_CHECK(btable.scalar_type() == at::kInt && btable.dim() == 2 && (btable.size(1) <= 1 || btable.stride(1) == 1),
              "btable must be int32 [num_reqs, pages_per_req] with unit column stride");
  check_device(rope, codes, "rope");
  check_device(scales, codes, "scales");
  check_device(btable, codes, "btable");
  qsa_b200_latent_cache c = {};
  c.codes = codes.data_ptr();
  c.rope = rope.data_ptr();
  c.scales = scales.data_ptr<float>();
  c.btable = btable.data_ptr<int32_t>();
  c.rank = checked_int32(codes.size(2), "rank");
  c.rope_dim = checked_int32(rope.size(2), "rope_dim");
  c.page_size = checked_int32(codes.size(1), "the page");
  c.pages_per_req = checked_int32(btable.size(1), "pages_per_req");
  c.num_reqs = checked_int32(btable.size(0), "num_reqs");
  c.num_pages = codes.size(0);
  c.btable_stride = row_stride(btable);
  return c;
}

// Entries and their tokens, for a call over `tokens` rows.
template <typename Args>
void fill_tokens(Args& a, const at::Tensor& starts, const OptTensor& reqs, const OptTensor& cu_tokens,
                 const at::Tensor& codes, const at::Tensor& btable, int64_t tokens) {
  TORCH_CHECK(starts.dim() == 1, "starts must be int32 [entries]");
  const int64_t n = starts.size(0);
  a.starts = int32_list(starts, codes, n, "starts");
  a.reqs = int32_list(reqs, codes, n, "reqs");
  a.cu_tokens = int32_list(cu_tokens, codes, n + 1, "cu_tokens");
  TORCH_CHECK(cu_tokens || n == tokens, "without cu_tokens every entry has one token: ", n, " entries, ", tokens, " tokens");
  TORCH_CHECK(reqs || n <= btable.size(0), "btable has ", btable.size(0), " rows for ", n, " entries");
  a.entries = checked_int32(n, "entries");
  a.tokens = checked_int32(tokens, "tokens");
}

void check_status(int64_t st, const char* what) {
  TORCH_CHECK(st >= 0, what, " failed: ", qsa_b200_status_string((int)st));
}

qsa_b200_stream_t current_stream(const at::Tensor& t) {
  return reinterpret_cast<qsa_b200_stream_t>(c10::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

// [tokens, n] with unit inner stride; returns the token stride.
int64_t check_rows(const at::Tensor& t, int64_t n, const char* name) {
  TORCH_CHECK(t.dim() == 2 && t.size(1) == n && t.stride(1) == 1, name, " must be [tokens, ", n, "] with unit inner stride");
  return row_stride(t);
}

void latent_append(const at::Tensor& c_new, const at::Tensor& r_new, at::Tensor& codes, at::Tensor& rope,
                   at::Tensor& scales, const at::Tensor& btable, const at::Tensor& starts, const OptTensor& reqs,
                   const OptTensor& cu_tokens, const OptTensor& table, const OptTensor& positions,
                   const OptTensor& c_weight, double eps, bool interleaved) {
  qsa_b200_latent_append_args a = {};
  a.cache = check_cache(codes, rope, scales, btable);
  a.input_dtype = dtype_code(c_new.scalar_type(), "c_new");
  TORCH_CHECK(r_new.scalar_type() == c_new.scalar_type(), "r_new must have c_new's dtype");
  a.c_stride = check_rows(c_new, codes.size(2), "c_new");
  a.r_stride = check_rows(r_new, rope.size(2), "r_new");
  const int64_t tokens = c_new.size(0);
  TORCH_CHECK(r_new.size(0) == tokens, "r_new must have c_new's tokens");
  check_device(c_new, codes, "c_new");
  check_device(r_new, codes, "r_new");
  fill_tokens(a, starts, reqs, cu_tokens, codes, btable, tokens);
  if (c_weight) {
    TORCH_CHECK(c_weight->dim() == 1 && c_weight->size(0) == codes.size(2) && c_weight->is_contiguous(),
                "c_weight must be contiguous [rank]");
    check_device(*c_weight, codes, "c_weight");
    a.c_weight = c_weight->data_ptr();
    a.weight_dtype = dtype_code(c_weight->scalar_type(), "c_weight");
  }
  TORCH_CHECK(table || !positions, "positions belong to a rotation table");
  if (table) {
    TORCH_CHECK(table->scalar_type() == at::kFloat && table->dim() == 2 && table->is_contiguous(),
                "table must be contiguous float32 [positions, rotary_dim]");
    check_device(*table, codes, "table");
    a.rotation.table = table->data_ptr<float>();
    a.rotation.positions = int32_list(positions, codes, tokens, "positions");
    a.rotation.table_len = checked_int32(table->size(0), "the table's length");
    a.rotation.rotary_dim = checked_int32(table->size(1), "rotary_dim");
    a.rotation.interleaved = interleaved ? 1 : 0;
    a.rotation.num_axes = 1;
  }
  a.c = c_new.data_ptr();
  a.r = r_new.data_ptr();
  a.eps = (float)eps;
  c10::cuda::CUDAGuard guard(codes.device());
  check_status(qsa_b200_latent_append(&a, current_stream(codes)), "qsa_b200_latent_append");
}

void latent_read_out(const at::Tensor& codes, const at::Tensor& rope, const at::Tensor& scales, const at::Tensor& btable,
                     const at::Tensor& starts, const OptTensor& cu_tokens, const OptTensor& reqs, at::Tensor& c,
                     at::Tensor& r) {
  qsa_b200_latent_read_args a = {};
  a.cache = check_cache(codes, rope, scales, btable);
  a.output_dtype = dtype_code(c.scalar_type(), "the output");
  TORCH_CHECK(r.scalar_type() == c.scalar_type() && c.dim() == 2 && r.dim() == 2 && c.size(1) == codes.size(2) &&
                  r.size(1) == rope.size(2) && r.size(0) == c.size(0) && c.is_contiguous() && r.is_contiguous(),
              "the outputs must be contiguous [tokens, rank] and [tokens, rope_dim] of one dtype");
  check_device(c, codes, "the output");
  check_device(r, codes, "the output");
  fill_tokens(a, starts, reqs, cu_tokens, codes, btable, c.size(0));
  a.c = c.data_ptr();
  a.r = r.data_ptr();
  c10::cuda::CUDAGuard guard(codes.device());
  check_status(qsa_b200_latent_read(&a, current_stream(codes)), "qsa_b200_latent_read");
}

std::tuple<at::Tensor, at::Tensor> latent_read(const at::Tensor& codes, const at::Tensor& rope, const at::Tensor& scales,
                                               const at::Tensor& btable, const at::Tensor& starts,
                                               const OptTensor& cu_tokens, int64_t tokens, const OptTensor& reqs,
                                               at::ScalarType dtype) {
  TORCH_CHECK(codes.dim() == 3 && rope.dim() == 3, "codes and rope must be [pages, P, ...]");
  TORCH_CHECK(tokens >= 0, "tokens must not be negative, got ", tokens);
  at::Tensor c = at::empty({tokens, codes.size(2)}, codes.options().dtype(dtype));
  at::Tensor r = at::empty({tokens, rope.size(2)}, codes.options().dtype(dtype));
  latent_read_out(codes, rope, scales, btable, starts, cu_tokens, reqs, c, r);
  return {c, r};
}

void latent_decode_out(const at::Tensor& q, const at::Tensor& codes, const at::Tensor& rope, const at::Tensor& scales,
                       const at::Tensor& btable, const OptTensor& t2r, const OptTensor& indices, const OptTensor& counts,
                       const OptTensor& tree, double softmax_scale, at::Tensor& out) {
  qsa_b200_latent_decode_args a = {};
  a.cache = check_cache(codes, rope, scales, btable);
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 && out.scalar_type() == at::kBFloat16, "q and out must be bfloat16");
  TORCH_CHECK((q.dim() == 3 || q.dim() == 4) && q.is_contiguous(), "q must be contiguous [rows, heads, rank + rope_dim] or "
              "[rows, nodes, heads, rank + rope_dim]");
  TORCH_CHECK(q.size(-1) == codes.size(2) + rope.size(2), "q has ", q.size(-1), " values a head, the cache ",
              codes.size(2) + rope.size(2));
  TORCH_CHECK(out.dim() == q.dim() && out.sizes().slice(0, q.dim() - 1) == q.sizes().slice(0, q.dim() - 1) &&
                  out.size(-1) == codes.size(2) && out.is_contiguous(),
              "out must be contiguous, shaped like q with rank values a head");
  check_device(q, codes, "q");
  check_device(out, codes, "out");
  const int64_t rows = q.size(0), nodes = q.dim() == 4 ? q.size(1) : 1;
  TORCH_CHECK(t2r || rows <= btable.size(0), "btable has ", btable.size(0), " rows for ", rows, " query rows");
  if (indices) {
    TORCH_CHECK(indices->scalar_type() == at::kInt && indices->dim() == 2 && indices->size(0) == rows &&
                    (indices->size(1) <= 1 || indices->stride(1) == 1),
                "indices must be int32 [", rows, ", K] with unit column stride");
    check_device(*indices, codes, "indices");
    a.topk = checked_int32(indices->size(1), "K");
    a.indices_stride = row_stride(*indices);
    // an empty list of columns is still a list
    static const int32_t none = 0;
    a.indices = indices->numel() > 0 ? indices->data_ptr<int32_t>() : &none;
  }
  if (tree) {
    TORCH_CHECK(tree->scalar_type() == at::kInt && tree->dim() == 3 && tree->size(0) == rows && tree->size(1) == nodes &&
                    tree->is_contiguous(),
                "tree must be contiguous int32 [", rows, ", ", nodes, ", words]");
    check_device(*tree, codes, "tree");
    a.tree_words = checked_int32(tree->size(2), "the tree's words");
    a.tree = tree->data_ptr<int32_t>();
  }
  a.t2r = int32_list(t2r, codes, rows, "t2r");
  a.counts = int32_list(counts, codes, rows, "counts");
  a.q = q.data_ptr();
  a.out = out.data_ptr();
  a.softmax_scale = (float)softmax_scale;
  a.rows = checked_int32(rows, "rows");
  a.nodes = checked_int32(nodes, "nodes");
  a.heads = checked_int32(q.size(-2), "heads");
  c10::cuda::CUDAGuard guard(codes.device());
  const int64_t need = qsa_b200_latent_decode_workspace_bytes(&a);
  check_status(need, "qsa_b200_latent_decode");
  at::Tensor workspace;
  if (need > 0) workspace = at::empty({need}, q.options().dtype(at::kByte));
  check_status(qsa_b200_latent_decode(&a, need > 0 ? workspace.data_ptr() : nullptr, (size_t)need, current_stream(codes)),
               "qsa_b200_latent_decode");
}

at::Tensor latent_decode(const at::Tensor& q, const at::Tensor& codes, const at::Tensor& rope, const at::Tensor& scales,
                         const at::Tensor& btable, const OptTensor& t2r, const OptTensor& indices, const OptTensor& counts,
                         const OptTensor& tree, double softmax_scale) {
  TORCH_CHECK(q.dim() >= 1 && codes.dim() == 3, "q must be [rows, (nodes,) heads, rank + rope_dim], codes [pages, P, rank]");
  auto shape = q.sizes().vec();
  shape.back() = codes.size(2);
  at::Tensor out = at::empty(shape, q.options());
  latent_decode_out(q, codes, rope, scales, btable, t2r, indices, counts, tree, softmax_scale, out);
  return out;
}

void head_strides(const at::Tensor& t, int64_t n, const char* name, int64_t& token, int64_t& head) {
  TORCH_CHECK(t.dim() == 3 && t.size(2) == n && t.stride(2) == 1, name, " must be [tokens, heads, ", n,
              "] with unit inner stride");
  head = t.size(1) > 1 ? t.stride(1) : n;
  token = t.size(0) > 1 ? t.stride(0) : t.size(1) * head;
}

void latent_prefill_out(const at::Tensor& q, const at::Tensor& k, const at::Tensor& k_rope, const at::Tensor& v,
                        const at::Tensor& cu_q, const OptTensor& cu_k, bool causal, double softmax_scale, at::Tensor& out) {
  TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
  qsa_b200_latent_prefill_args a = {};
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf, "q must be bfloat16 or float16");
  a.dtype = dtype_code(q.scalar_type(), "q");
  TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type() &&
                  k_rope.scalar_type() == q.scalar_type() && out.scalar_type() == q.scalar_type(),
              "k, k_rope, v and out must have q's dtype");
  head_strides(q, 192, "q", a.q_stride, a.q_head_stride);
  head_strides(k, 128, "k", a.k_stride, a.k_head_stride);
  head_strides(v, 128, "v", a.v_stride, a.v_head_stride);
  a.k_rope_stride = check_rows(k_rope, 64, "k_rope");
  TORCH_CHECK(k.size(1) == q.size(1) && v.size(1) == q.size(1), "k and v must have q's heads");
  TORCH_CHECK(v.size(0) == k.size(0) && k_rope.size(0) == k.size(0), "v and k_rope must have k's tokens");
  TORCH_CHECK(out.dim() == 3 && out.size(0) == q.size(0) && out.size(1) == q.size(1) && out.size(2) == 128 &&
                  out.is_contiguous(),
              "out must be contiguous [tokens, heads, 128]");
  check_device(k, q, "k");
  check_device(k_rope, q, "k_rope");
  check_device(v, q, "v");
  check_device(out, q, "out");
  TORCH_CHECK(cu_q.dim() == 1 && cu_q.size(0) >= 1, "cu_q must be int32 [entries + 1]");
  a.cu_q = int32_list(cu_q, q, cu_q.size(0), "cu_q");
  a.cu_k = cu_k ? int32_list(cu_k, q, cu_q.size(0), "cu_k") : a.cu_q;
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.k_rope = k_rope.data_ptr();
  a.v = v.data_ptr();
  a.out = out.data_ptr();
  a.softmax_scale = (float)softmax_scale;
  a.entries = checked_int32(cu_q.size(0) - 1, "entries");
  a.q_tokens = checked_int32(q.size(0), "q's tokens");
  a.k_tokens = checked_int32(k.size(0), "k's tokens");
  a.heads = checked_int32(q.size(1), "heads");
  a.causal = causal ? 1 : 0;
  c10::cuda::CUDAGuard guard(q.device());
  check_status(qsa_b200_latent_prefill(&a, current_stream(q)), "qsa_b200_latent_prefill");
}

at::Tensor latent_prefill(const at::Tensor& q, const at::Tensor& k, const at::Tensor& k_rope, const at::Tensor& v,
                          const at::Tensor& cu_q, const OptTensor& cu_k, bool causal, double softmax_scale) {
  TORCH_CHECK(q.dim() == 3, "q must be [tokens, heads, 192]");
  at::Tensor out = at::empty({q.size(0), q.size(1), 128}, q.options());
  latent_prefill_out(q, k, k_rope, v, cu_q, cu_k, causal, softmax_scale, out);
  return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(qsa_b200, m) {
  m.def(
      "latent_append(Tensor c_new, Tensor r_new, Tensor(a!) codes, Tensor(b!) rope, Tensor(c!) scales, Tensor btable, "
      "Tensor starts, Tensor? reqs, Tensor? cu_tokens, Tensor? table, Tensor? positions, Tensor? c_weight, float eps, "
      "bool interleaved) -> ()");
  m.def(
      "latent_read(Tensor codes, Tensor rope, Tensor scales, Tensor btable, Tensor starts, Tensor? cu_tokens, int tokens, "
      "Tensor? reqs, ScalarType dtype) -> (Tensor, Tensor)");
  m.def(
      "latent_read_out(Tensor codes, Tensor rope, Tensor scales, Tensor btable, Tensor starts, Tensor? cu_tokens, "
      "Tensor? reqs, Tensor(a!) c, Tensor(b!) r) -> ()");
  m.def(
      "latent_decode(Tensor q, Tensor codes, Tensor rope, Tensor scales, Tensor btable, Tensor? t2r, Tensor? indices, "
      "Tensor? counts, Tensor? tree, float softmax_scale) -> Tensor");
  m.def(
      "latent_decode_out(Tensor q, Tensor codes, Tensor rope, Tensor scales, Tensor btable, Tensor? t2r, Tensor? indices, "
      "Tensor? counts, Tensor? tree, float softmax_scale, Tensor(a!) out) -> ()");
  m.def(
      "latent_prefill(Tensor q, Tensor k, Tensor k_rope, Tensor v, Tensor cu_q, Tensor? cu_k, bool causal, "
      "float softmax_scale) -> Tensor");
  m.def(
      "latent_prefill_out(Tensor q, Tensor k, Tensor k_rope, Tensor v, Tensor cu_q, Tensor? cu_k, bool causal, "
      "float softmax_scale, Tensor(a!) out) -> ()");
}

TORCH_LIBRARY_IMPL(qsa_b200, CUDA, m) {
  m.impl("latent_append", &latent_append);
  m.impl("latent_read", &latent_read);
  m.impl("latent_read_out", &latent_read_out);
  m.impl("latent_decode", &latent_decode);
  m.impl("latent_decode_out", &latent_decode_out);
  m.impl("latent_prefill", &latent_prefill);
  m.impl("latent_prefill_out", &latent_prefill_out);
}
