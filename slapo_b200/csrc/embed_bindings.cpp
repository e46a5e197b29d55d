// torch bindings of the token table's lookup and gradient.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <limits>

#include "kernels.h"

namespace {

using at::Tensor;
using c10::optional;

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return 0;
    case at::kHalf: return 1;
    case at::kFloat: return 2;
    default: TORCH_CHECK(false, "embedding: a table of bf16, fp16 or fp32 required, not ", t.scalar_type());
  }
}

void check_ids(const Tensor& ids, const Tensor& other) {
  TORCH_CHECK(ids.is_cuda() && ids.get_device() == other.get_device(),
              "embedding: ids must be on the table's CUDA device");
  TORCH_CHECK(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt,
              "embedding: ids of int64 or int32 required, not ", ids.scalar_type());
}

Tensor embedding_fwd(const Tensor& ids_in, const Tensor& weight_in, int64_t start, double scale) {
  TORCH_CHECK(weight_in.is_cuda() && weight_in.dim() == 2, "embedding: a 2-D CUDA table required");
  check_ids(ids_in, weight_in);
  const int code = dtype_code(weight_in);
  c10::cuda::CUDAGuard guard(weight_in.device());
  const Tensor ids = ids_in.contiguous();
  const Tensor weight = weight_in.stride(1) == 1 ? weight_in : weight_in.contiguous();
  std::vector<int64_t> shape = ids.sizes().vec();
  shape.push_back(weight.size(1));
  Tensor out = at::empty(shape, weight.options().memory_format(at::MemoryFormat::Contiguous));
  const int rc = slapo::launch_embedding_fwd(
      ids.const_data_ptr(), ids.scalar_type() == at::kLong, weight.const_data_ptr(), out.data_ptr(), ids.numel(),
      weight.size(0), weight.size(1), weight.stride(0), start, static_cast<float>(scale), code,
      at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(rc == 0, "embedding_fwd: launch refused (code ", rc, ")");
  return out;
}

Tensor embedding_bwd(const Tensor& dy_in, const Tensor& ids_in, int64_t rows, int64_t start,
                     const optional<int64_t>& padding, double scale) {
  TORCH_CHECK(dy_in.is_cuda() && dy_in.dim() >= 1 && rows >= 0, "embedding: a CUDA gradient required");
  check_ids(ids_in, dy_in);
  const int code = dtype_code(dy_in);
  const int64_t cols = dy_in.size(-1), tokens = ids_in.numel();
  TORCH_CHECK(dy_in.numel() == tokens * cols, "embedding: one row of the gradient for each of the ", tokens,
              " ids required");
  TORCH_CHECK(tokens <= slapo::kEmbedGradTokens, "embedding: the gradient takes at most ", slapo::kEmbedGradTokens,
              " ids at a time, not ", tokens);
  c10::cuda::CUDAGuard guard(dy_in.device());
  const Tensor dy = dy_in.contiguous(), ids = ids_in.contiguous();
  Tensor dw = at::empty({rows, cols}, dy.options().memory_format(at::MemoryFormat::Contiguous));
  const slapo::EmbedGradPlan plan = slapo::embedding_bwd_plan(tokens, rows, cols);
  Tensor scratch = at::empty({plan.words()}, dy.options().dtype(at::kInt));
  const int rc = slapo::launch_embedding_bwd(
      ids.const_data_ptr(), ids.scalar_type() == at::kLong, dy.const_data_ptr(), dw.data_ptr(),
      scratch.data_ptr<int32_t>(), plan, tokens, rows, cols, start,
      padding.has_value() ? *padding : std::numeric_limits<int64_t>::min(), static_cast<float>(scale), code,
      at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(rc == 0, "embedding_bwd: launch refused (code ", rc, ")");
  return dw;
}

}  // namespace

void register_embed_ops(torch::Library& m) {
  m.def("embedding_fwd(Tensor ids, Tensor weight, int start, float scale) -> Tensor", &embedding_fwd);
  m.def("embedding_bwd(Tensor dy, Tensor ids, int rows, int start, int? padding, float scale) -> Tensor",
        &embedding_bwd);
}
