// torch binding of AdamW over many tensors.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <vector>

#include "kernels.h"

namespace {

using at::Tensor;
using c10::optional;
using List = at::TensorList;

constexpr int64_t kBlock = 256;       // values per factor of the 8-bit moments

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return 0;
    case at::kHalf: return 1;
    case at::kFloat: return 2;
    default: TORCH_CHECK(false, "multi_adamw: parameters of bf16, fp16 or fp32 required, not ", t);
  }
}

void check_one(const Tensor& t, const char* name, const Tensor& param, at::ScalarType type, int64_t n) {
  TORCH_CHECK(t.is_cuda() && t.layout() == at::kStrided && t.get_device() == param.get_device(), "multi_adamw: ",
              name, " must be CUDA tensors on the parameters' device");
  TORCH_CHECK(t.scalar_type() == type, "multi_adamw: ", name, " must be ", type, ", not ", t.scalar_type());
  TORCH_CHECK(t.is_contiguous(), "multi_adamw: ", name, " must be contiguous");
  TORCH_CHECK(t.numel() == n, "multi_adamw: ", name, ": ", n, " values required, not ", t.numel());
}

// No two of a list's tensors share memory: both would be written at the same time.
void check_apart(List list, const char* name) {
  using Range = std::pair<const char*, const char*>;
  std::vector<Range> r;
  r.reserve(list.size());
  bool sorted = true;
  for (const Tensor& t : list) {
    if (t.numel() == 0) continue;
    const char* at = static_cast<const char*>(t.const_data_ptr());
    r.emplace_back(at, at + t.nbytes());
    if (r.size() > 1) sorted = sorted && r[r.size() - 2].second <= at;
  }
  if (sorted) return;
  std::sort(r.begin(), r.end());
  for (size_t i = 1; i < r.size(); ++i)
    TORCH_CHECK(r[i - 1].second <= r[i].first, "multi_adamw: two of the ", name, " share memory");
}

bool on(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

void multi_adamw(List params, List grads, List masters, List exp_avgs, List exp_avg_sqs, List exp_avg_scales,
                 List exp_avg_sq_scales, at::ArrayRef<double> lrs, at::ArrayRef<double> weight_decays, double beta1,
                 double beta2, double eps, int64_t step, const optional<Tensor>& step_tensor,
                 const optional<Tensor>& grad_scale) {
  const size_t n = params.size();
  if (n == 0) return;
  const bool bits8 = !exp_avg_scales.empty();
  auto same = [&](size_t m, bool may_miss) { return m == n || (may_miss && m == 0); };
  TORCH_CHECK(same(grads.size(), false) && same(masters.size(), true) && same(exp_avgs.size(), false) &&
                  same(exp_avg_sqs.size(), false) && same(exp_avg_scales.size(), true) &&
                  exp_avg_sq_scales.size() == exp_avg_scales.size() && lrs.size() == n && weight_decays.size() == n,
              "multi_adamw: one entry for each of the ", n, " parameters required in every list");
  TORCH_CHECK(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0,
              "multi_adamw: betas in [0, 1) and eps >= 0 required");
  TORCH_CHECK(n <= INT_MAX, "multi_adamw: too many tensors");
  const Tensor& p0 = params[0];
  TORCH_CHECK(masters.empty() || p0.scalar_type() != at::kFloat, "multi_adamw: fp32 parameters are their own masters");
  TORCH_CHECK(p0.is_cuda(), "multi_adamw: parameters must be CUDA tensors");
  const at::ScalarType type = p0.scalar_type(), moments = bits8 ? at::kFloat8_e4m3fn : at::kFloat;
  slapo::AdamwScalars s{};
  s.beta1 = static_cast<float>(beta1);
  s.one_beta1 = static_cast<float>(1.0 - beta1);
  s.beta2 = static_cast<float>(beta2);
  s.one_beta2 = static_cast<float>(1.0 - beta2);
  s.eps = static_cast<float>(eps);
  s.beta1_d = beta1;
  s.beta2_d = beta2;
  if (step_tensor.has_value() && step_tensor->defined()) {
    check_one(*step_tensor, "the step", p0, at::kLong, 1);
    s.step = step_tensor->data_ptr<int64_t>();
  } else {
    TORCH_CHECK(step >= 1, "multi_adamw: steps count from 1, not ", step);
    s.inv_bc1 = static_cast<float>(1.0 / (1.0 - std::pow(beta1, static_cast<double>(step))));
    s.inv_sqrt_bc2 = static_cast<float>(1.0 / std::sqrt(1.0 - std::pow(beta2, static_cast<double>(step))));
  }
  if (grad_scale.has_value() && grad_scale->defined()) {
    check_one(*grad_scale, "grad_scale", p0, at::kFloat, 1);
    s.grad_scale = grad_scale->data_ptr<float>();
  }
  std::vector<slapo::AdamwTensor> table;
  table.reserve(n);
  for (size_t i = 0; i < n; ++i) {
    const int64_t count = params[i].numel();
    check_one(params[i], "parameters", p0, type, count);
    check_one(grads[i], "gradients", p0, type, count);
    if (!masters.empty()) check_one(masters[i], "masters", p0, at::kFloat, count);
    check_one(exp_avgs[i], "first moments", p0, moments, count);
    check_one(exp_avg_sqs[i], "second moments", p0, moments, count);
    slapo::AdamwTensor t{};
    t.param = params[i].data_ptr();
    t.grad = grads[i].const_data_ptr();
    t.master = masters.empty() ? nullptr : masters[i].data_ptr<float>();
    t.m = exp_avgs[i].data_ptr();
    t.v = exp_avg_sqs[i].data_ptr();
    if (bits8) {
      const int64_t blocks = (count + kBlock - 1) / kBlock;
      check_one(exp_avg_scales[i], "factors", p0, at::kFloat, blocks);
      check_one(exp_avg_sq_scales[i], "factors", p0, at::kFloat, blocks);
      t.m_scale = exp_avg_scales[i].data_ptr<float>();
      t.v_scale = exp_avg_sq_scales[i].data_ptr<float>();
    }
    t.n = count;
    t.lr = static_cast<float>(lrs[i]);
    t.weight_decay = static_cast<float>(weight_decays[i]);
    t.aligned = on(t.param, 32) && on(t.grad, 32) && on(t.master, 32) && on(t.m, 32) && on(t.v, 32);
    if (count > 0) table.push_back(t);
  }
  for (auto& [list, name] : {std::make_pair(params, "parameters"), std::make_pair(masters, "masters"),
                             std::make_pair(exp_avgs, "first moments"), std::make_pair(exp_avg_sqs, "second moments"),
                             std::make_pair(exp_avg_scales, "factors"), std::make_pair(exp_avg_sq_scales, "factors")})
    check_apart(list, name);
  c10::cuda::CUDAGuard guard(p0.device());
  const int rc = slapo::launch_adamw_multi(table.data(), static_cast<int>(table.size()), s, bits8, dtype_code(type),
                                           at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(rc == 0, "multi_adamw: launch refused (code ", rc, ")");
  // (autograd notices that a saved parameter has changed)
  for (const Tensor& p : params)
    if (!p.is_inference()) p.unsafeGetTensorImpl()->bump_version();
}

}  // namespace

void register_optim_ops(torch::Library& m) {
  m.def("multi_adamw(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] masters, Tensor(c!)[] exp_avgs, Tensor(d!)[] exp_avg_sqs, Tensor(e!)[] exp_avg_scales, Tensor(f!)[] exp_avg_sq_scales, float[] lrs, float[] weight_decays, float beta1, float beta2, float eps, int step, Tensor? step_tensor, Tensor? grad_scale) -> ()",
        &multi_adamw);
}
