// The torch binding of the decode-step operators (add_rms_norm, paged_attention, paged_evict,
// token_logprobs): tensor checks, outputs and workspace from torch's caching allocator, and the
// call of the C ABI on torch's current stream. Nothing synchronises.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include "int4gemv_b200.h"
#include "int4gemv_torch.h"

namespace int4gemv {
namespace {

void check_status(int status) { TORCH_CHECK(status == INT4GEMV_OK, int4gemv_last_error()); }

void* stream_of(const at::Tensor& t) {
  return static_cast<void*>(c10::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

// An uninitialised contiguous tensor on the device of `like`, from the caching allocator without
// torch's operator dispatch (a small call's time on the host is mostly such calls: 0.5 us less each).
at::Tensor make(at::IntArrayRef sizes, at::ScalarType dtype, const at::Tensor& like) {
  return at::detail::empty_cuda(sizes, dtype, like.device(), c10::nullopt);
}

int dtype_of(const char* name, const char* what, const at::Tensor& t, bool f32) {
  switch (t.scalar_type()) {
    case at::kHalf: return INT4GEMV_DTYPE_F16;
    case at::kBFloat16: return INT4GEMV_DTYPE_BF16;
    case at::kFloat:
      if (f32) return INT4GEMV_DTYPE_F32;
      [[fallthrough]];
    default:
      TORCH_CHECK(false, name, ": ", what, " must be ", f32 ? "float32, " : "", "float16 or bfloat16, got ",
                  t.scalar_type());
  }
}

// A contiguous tensor of this type and shape on the device of `like`.
void check_like(const char* name, const char* what, const at::Tensor& t, at::ScalarType dtype,
                at::IntArrayRef sizes, const at::Tensor& like) {
  TORCH_CHECK(t.scalar_type() == dtype && t.sizes() == sizes && t.is_contiguous() &&
                  t.device() == like.device(),
              name, ": ", what, " must be a contiguous ", c10::toString(dtype), " ", sizes,
              " tensor on ", like.device(), ", got ", t.scalar_type(), " ", t.sizes(), " on ",
              t.device());
}

struct Norm {
  int dtype;
  at::Tensor h;
  const void* residual;
  void* h_out;
};

Norm check_norm(const char* name, const at::Tensor& x, const at::Tensor& weight,
                const c10::optional<at::Tensor>& residual) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.is_contiguous(), name,
              ": expected a contiguous 2-D CUDA tensor x");
  TORCH_CHECK(x.size(1) > 0, name, ": x has no columns");
  const int dtype = dtype_of(name, "x", x, true);
  check_like(name, "weight", weight, x.scalar_type(), {x.size(1)}, x);
  if (!residual.has_value()) return {dtype, x, nullptr, nullptr};
  check_like(name, "residual", *residual, x.scalar_type(), x.sizes(), x);
  at::Tensor h = make(x.sizes(), x.scalar_type(), x);
  return {dtype, h, residual->data_ptr(), h.data_ptr()};
}

int4gemv_paged_cache_t check_cache(const char* name, const at::Tensor& k, const at::Tensor& v,
                                   const at::Tensor* weights) {
  TORCH_CHECK(k.is_cuda() && k.dim() == 4, name, ": k_cache must be a 4-D CUDA tensor [num_blocks, "
              "block_size, kv_heads, head_dim]");
  TORCH_CHECK(v.scalar_type() == k.scalar_type() && v.sizes() == k.sizes() && v.device() == k.device(),
              name, ": v_cache must be like k_cache, ", k.scalar_type(), " ", k.sizes(), " on ",
              k.device(), ", got ", v.scalar_type(), " ", v.sizes(), " on ", v.device());
  TORCH_CHECK((k.stride(3) == 1 && v.stride(3) == 1) || k.size(3) == 1 || k.numel() == 0, name,
              ": the elements of a head must be contiguous in k_cache and v_cache");
  int4gemv_paged_cache_t c{};
  c.dtype = dtype_of(name, "k_cache", k, false);
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.num_blocks = k.size(0);
  c.block_size = k.size(1);
  c.kv_heads = k.size(2);
  c.head_dim = k.size(3);
  for (int i = 0; i < 3; ++i) {
    // the stride of a dimension of one says nothing
    c.k_strides[i] = k.size(i) > 1 ? k.stride(i) : 0;
    c.v_strides[i] = v.size(i) > 1 ? v.stride(i) : 0;
  }
  if (weights) {
    check_like(name, "weights", *weights, at::kFloat, {c.num_blocks, c.kv_heads, c.block_size}, k);
    c.weights = weights->data_ptr<float>();
  }
  return c;
}

void check_table(const char* name, const char* what, const at::Tensor& t, int64_t batch,
                 const at::Tensor& like) {
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 2 && t.size(0) == batch && t.is_contiguous() &&
                  t.device() == like.device(),
              name, ": ", what, " must be a contiguous Int [", batch, ", blocks] tensor on ",
              like.device(), ", got ", t.scalar_type(), " ", t.sizes(), " on ", t.device());
}

}  // namespace

std::tuple<at::Tensor, at::Tensor> add_rms_norm(const at::Tensor& x, const at::Tensor& weight,
                                                double eps,
                                                const c10::optional<at::Tensor>& residual) {
  const char* name = "add_rms_norm";
  const c10::cuda::OptionalCUDAGuard guard(x.is_cuda() ? c10::make_optional(x.device()) : c10::nullopt);
  const Norm n = check_norm(name, x, weight, residual);
  at::Tensor y = make(x.sizes(), x.scalar_type(), x);
  check_status(int4gemv_add_rms_norm(y.data_ptr(), n.h_out, x.data_ptr(), n.residual,
                                     weight.data_ptr(), static_cast<float>(eps), n.dtype, x.size(0),
                                     x.size(1), stream_of(x)));
  return {y, n.h};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> add_rms_norm_quant(
    const at::Tensor& x, const at::Tensor& weight, double eps,
    const c10::optional<at::Tensor>& residual) {
  const char* name = "add_rms_norm_quant";
  const c10::cuda::OptionalCUDAGuard guard(x.is_cuda() ? c10::make_optional(x.device()) : c10::nullopt);
  const Norm n = check_norm(name, x, weight, residual);
  at::Tensor y = make(x.sizes(), at::kFloat8_e4m3fn, x);
  at::Tensor scales = make({x.size(0)}, at::kFloat, x);
  check_status(int4gemv_add_rms_norm_quant(y.data_ptr(), scales.data_ptr<float>(), n.h_out,
                                           x.data_ptr(), n.residual, weight.data_ptr(),
                                           static_cast<float>(eps), n.dtype, x.size(0), x.size(1),
                                           stream_of(x)));
  return {y, scales, n.h};
}

at::Tensor paged_attention(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                           const at::Tensor& block_table, const at::Tensor& seq_lens, double scale,
                           const c10::optional<at::Tensor>& k, const c10::optional<at::Tensor>& v,
                           const c10::optional<at::Tensor>& weights) {
  const char* name = "paged_attention";
  const at::Tensor* w = weights.has_value() ? &*weights : nullptr;
  const int4gemv_paged_cache_t cache = check_cache(name, k_cache, v_cache, w);
  TORCH_CHECK(q.scalar_type() == k_cache.scalar_type() && q.dim() == 3 && q.size(2) == cache.head_dim &&
                  q.is_contiguous() && q.device() == k_cache.device(),
              name, ": q must be a contiguous ", k_cache.scalar_type(), " [batch, q_heads, ",
              cache.head_dim, "] tensor on ", k_cache.device(), ", got ", q.scalar_type(), " ", q.sizes(),
              " on ", q.device());
  const int64_t batch = q.size(0), q_heads = q.size(1);
  check_table(name, "block_table", block_table, batch, q);
  check_like(name, "seq_lens", seq_lens, at::kInt, {batch}, q);
  TORCH_CHECK(k.has_value() == v.has_value(), name, ": k and v come together");
  if (k.has_value()) {
    const std::array<int64_t, 3> sizes = {batch, cache.kv_heads, cache.head_dim};
    check_like(name, "k", *k, q.scalar_type(), sizes, q);
    check_like(name, "v", *v, q.scalar_type(), sizes, q);
  }
  const c10::cuda::CUDAGuard guard(q.device());
  const int64_t blocks = block_table.size(1);
  const int64_t bytes = int4gemv_paged_attention_workspace_size(&cache, batch, q_heads, blocks, w != nullptr);
  TORCH_CHECK(bytes >= 0, int4gemv_last_error());
  at::Tensor out = make(q.sizes(), q.scalar_type(), q);
  at::Tensor workspace;
  if (bytes > 0) workspace = make({bytes}, at::kByte, q);
  check_status(int4gemv_paged_attention(
      out.data_ptr(), q.data_ptr(), &cache, block_table.data_ptr<int>(), seq_lens.data_ptr<int>(),
      static_cast<float>(scale), k.has_value() ? k->data_ptr() : nullptr,
      v.has_value() ? v->data_ptr() : nullptr, w != nullptr, batch, q_heads, blocks,
      bytes > 0 ? workspace.data_ptr() : nullptr, bytes, stream_of(q)));
  return out;
}

std::tuple<at::Tensor, at::Tensor> paged_evict(const at::Tensor& k_cache, const at::Tensor& v_cache,
                                               const at::Tensor& weights,
                                               const at::Tensor& block_table,
                                               const at::Tensor& seq_lens, const at::Tensor& new_table,
                                               int64_t budget, int64_t recent) {
  const char* name = "paged_evict";
  const int4gemv_paged_cache_t cache = check_cache(name, k_cache, v_cache, &weights);
  TORCH_CHECK(seq_lens.dim() == 1, name, ": seq_lens must be 1-D");
  const int64_t batch = seq_lens.size(0);
  check_like(name, "seq_lens", seq_lens, at::kInt, {batch}, k_cache);
  check_table(name, "block_table", block_table, batch, k_cache);
  check_table(name, "new_table", new_table, batch, k_cache);
  TORCH_CHECK(budget > 0, name, ": budget ", budget, " must be positive");
  const c10::cuda::CUDAGuard guard(k_cache.device());
  at::Tensor kept = make({batch, cache.kv_heads, budget}, at::kInt, k_cache);
  at::Tensor new_lens = make({batch}, at::kInt, k_cache);
  check_status(int4gemv_paged_evict(kept.data_ptr<int>(), new_lens.data_ptr<int>(), &cache,
                                    block_table.data_ptr<int>(), seq_lens.data_ptr<int>(),
                                    new_table.data_ptr<int>(), budget, recent, batch,
                                    block_table.size(1), new_table.size(1), stream_of(k_cache)));
  return {kept, new_lens};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> token_logprobs(const at::Tensor& logits,
                                                                          const at::Tensor& tokens,
                                                                          int64_t top) {
  const char* name = "token_logprobs";
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2, name, ": logits must be a 2-D CUDA tensor");
  TORCH_CHECK(logits.size(1) > 0, name, ": logits have no columns");
  TORCH_CHECK(logits.stride(1) == 1 || logits.size(1) == 1 || logits.numel() == 0, name,
              ": the logits of a row must be contiguous");
  const int dtype = dtype_of(name, "logits", logits, true);
  const int64_t rows = logits.size(0), vocab = logits.size(1);
  check_like(name, "tokens", tokens, at::kLong, {rows}, logits);
  TORCH_CHECK(top >= 0 && top <= INT4GEMV_MAX_TOP && top <= vocab, name, ": top ", top,
              " must be in [0, ", INT4GEMV_MAX_TOP, "] and at most vocab = ", vocab);
  const c10::cuda::CUDAGuard guard(logits.device());
  at::Tensor logprobs = make({rows}, at::kFloat, logits), entropy = make({rows}, at::kFloat, logits);
  at::Tensor top_logprobs = make({rows, top}, at::kFloat, logits);
  at::Tensor top_ids = make({rows, top}, at::kLong, logits);
  check_status(int4gemv_token_logprobs(
      logprobs.data_ptr<float>(), entropy.data_ptr<float>(), top_logprobs.data_ptr<float>(),
      top_ids.data_ptr<int64_t>(), logits.data_ptr(), tokens.data_ptr<int64_t>(), dtype, rows, vocab,
      rows > 1 ? logits.stride(0) : vocab, top, stream_of(logits)));
  return {logprobs, entropy, top_logprobs, top_ids};
}

}  // namespace int4gemv
