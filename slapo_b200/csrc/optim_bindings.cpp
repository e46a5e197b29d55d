// torch binding of AdamW over many tensors.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <vector>

#include "kernels.h"
#include "py_entry.h"

namespace {

using at::Tensor;
using c10::optional;
using slapo::AdamwLists;
using List = AdamwLists::List;

constexpr int64_t kBlock = 256;       // values per factor of the 8-bit moments

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return 0;
    case at::kHalf: return 1;
    case at::kFloat: return 2;
    default: TORCH_CHECK(false, "multi_adamw: parameters of bf16, fp16 or fp32 required, not ", t);
  }
}

// A tensor of a list: a type, a length, contiguous, on the parameters' device; where its values are.
// (Some hundred nanoseconds a tensor are a step's host time: one condition, the message only when it fails.)
char* checked(const Tensor& t, const char* name, c10::Device device, caffe2::TypeMeta type, int64_t n) {
  c10::TensorImpl* impl = t.unsafeGetTensorImpl();
  if (C10_UNLIKELY(!t.defined() || impl->device() != device || impl->layout() != at::kStrided || impl->dtype() != type ||
                   impl->numel() != n || !impl->is_contiguous())) {
    TORCH_CHECK(t.defined() && impl->device() == device && impl->layout() == at::kStrided, "multi_adamw: ", name,
                " must be CUDA tensors on the parameters' device");
    TORCH_CHECK(impl->dtype() == type, "multi_adamw: ", name, " must be ", type, ", not ", impl->dtype());
    TORCH_CHECK(impl->numel() == n, "multi_adamw: ", name, ": ", n, " values required, not ", impl->numel());
    TORCH_CHECK(false, "multi_adamw: ", name, " must be contiguous");
  }
  char* const at = static_cast<char*>(impl->mutable_data());
  TORCH_CHECK(at != nullptr || n == 0, "multi_adamw: ", name, " have no memory");
  return at;
}

// No two of a list's tensors share memory: both would be written at the same time.
void check_apart(const std::vector<slapo::AdamwTensor>& table, char* (*at)(const slapo::AdamwTensor&), int64_t bytes,
                 int64_t per, const char* name) {
  using Range = std::pair<const char*, const char*>;
  auto range = [&](const slapo::AdamwTensor& t) {
    const char* begin = at(t);
    return Range(begin, begin + (t.n + per - 1) / per * bytes);
  };
  const char* end = nullptr;
  bool sorted = true;
  for (const auto& t : table) {
    const Range r = range(t);
    sorted = sorted && end <= r.first;
    end = r.second;
  }
  if (sorted) return;
  std::vector<Range> r;
  r.reserve(table.size());
  for (const auto& t : table) r.push_back(range(t));
  std::sort(r.begin(), r.end());
  for (size_t i = 1; i < r.size(); ++i)
    TORCH_CHECK(r[i - 1].second <= r[i].first, "multi_adamw: two of the ", name, " share memory");
}

bool on32(const slapo::AdamwTensor& t) {
  const auto bits = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  return ((bits(t.param) | bits(t.grad) | bits(t.master) | bits(t.m) | bits(t.v)) & 31) == 0;
}

void run(const AdamwLists& x) {
  const size_t n = x.params.size;
  if (n == 0) return;
  const bool bits8 = x.exp_avg_scales.size != 0, has_master = x.masters.size != 0;
  auto same = [&](const List& list, bool may_miss) { return list.size == n || (may_miss && list.size == 0); };
  TORCH_CHECK(same(x.grads, false) && same(x.masters, true) && same(x.exp_avgs, false) && same(x.exp_avg_sqs, false) &&
                  same(x.exp_avg_scales, true) && x.exp_avg_sq_scales.size == x.exp_avg_scales.size &&
                  x.n_lrs == n && x.n_weight_decays == n,
              "multi_adamw: one entry for each of the ", n, " parameters required in every list");
  TORCH_CHECK(x.beta1 >= 0.0 && x.beta1 < 1.0 && x.beta2 >= 0.0 && x.beta2 < 1.0 && x.eps >= 0.0,
              "multi_adamw: betas in [0, 1) and eps >= 0 required");
  // (8 bits: a second moment below 2^-126 counts as zero.  The root of its corrected value is below 2^-63 / sqrt(1 - beta2)
  // then; where eps is no less, leaving it out of the divisor makes a step at most twice as long.)
  TORCH_CHECK(!bits8 || x.eps * std::sqrt(1.0 - x.beta2) >= std::ldexp(1.0, -63),
              "multi_adamw: 8-bit moments need eps of at least 2^-63 / sqrt(1 - beta2), not ", x.eps);
  TORCH_CHECK(n <= INT_MAX, "multi_adamw: too many tensors");
  const Tensor& p0 = x.params[0];
  TORCH_CHECK(p0.is_cuda(), "multi_adamw: parameters must be CUDA tensors");
  const int code = dtype_code(p0.scalar_type());
  TORCH_CHECK(!has_master || p0.scalar_type() != at::kFloat, "multi_adamw: fp32 parameters are their own masters");
  const c10::Device device = p0.device();
  const caffe2::TypeMeta type = p0.dtype(), fp32 = caffe2::TypeMeta::Make<float>(),
                         moments = bits8 ? caffe2::TypeMeta::Make<c10::Float8_e4m3fn>() : fp32;
  slapo::AdamwScalars s{};
  s.beta1 = static_cast<float>(x.beta1);
  s.one_beta1 = static_cast<float>(1.0 - x.beta1);
  s.beta2 = static_cast<float>(x.beta2);
  s.one_beta2 = static_cast<float>(1.0 - x.beta2);
  s.eps = static_cast<float>(x.eps);
  s.beta1_d = x.beta1;
  s.beta2_d = x.beta2;
  if (x.step_tensor != nullptr) {
    s.step = reinterpret_cast<int64_t*>(
        checked(*x.step_tensor, "the step", device, caffe2::TypeMeta::Make<int64_t>(), 1));
  } else {
    TORCH_CHECK(x.step >= 1, "multi_adamw: steps count from 1, not ", x.step);
    const double t = static_cast<double>(x.step);
    s.inv_bc1 = static_cast<float>(1.0 / (1.0 - std::pow(x.beta1, t)));
    s.inv_sqrt_bc2 = static_cast<float>(1.0 / std::sqrt(1.0 - std::pow(x.beta2, t)));
  }
  if (x.grad_scale != nullptr)
    s.grad_scale = reinterpret_cast<float*>(checked(*x.grad_scale, "grad_scale", device, fp32, 1));
  std::vector<slapo::AdamwTensor> table;
  table.reserve(n);
  for (size_t i = 0; i < n; ++i) {
    const int64_t count = x.params[i].numel();
    slapo::AdamwTensor t{};
    t.param = checked(x.params[i], "parameters", device, type, count);
    t.grad = checked(x.grads[i], "gradients", device, type, count);
    if (has_master) t.master = reinterpret_cast<float*>(checked(x.masters[i], "masters", device, fp32, count));
    t.m = checked(x.exp_avgs[i], "first moments", device, moments, count);
    t.v = checked(x.exp_avg_sqs[i], "second moments", device, moments, count);
    if (bits8) {
      const int64_t blocks = (count + kBlock - 1) / kBlock;
      t.m_scale = reinterpret_cast<float*>(checked(x.exp_avg_scales[i], "factors", device, fp32, blocks));
      t.v_scale = reinterpret_cast<float*>(checked(x.exp_avg_sq_scales[i], "factors", device, fp32, blocks));
    }
    t.n = count;
    t.lr = static_cast<float>(x.lrs[i]);
    t.weight_decay = static_cast<float>(x.weight_decays[i]);
    t.aligned = on32(t);
    if (count > 0) table.push_back(t);
  }
  using Entry = slapo::AdamwTensor;
  const int64_t size = static_cast<int64_t>(type.itemsize()), moment = bits8 ? 1 : 4;
  check_apart(table, [](const Entry& t) { return static_cast<char*>(t.param); }, size, 1, "parameters");
  check_apart(table, [](const Entry& t) { return static_cast<char*>(t.m); }, moment, 1, "first moments");
  check_apart(table, [](const Entry& t) { return static_cast<char*>(t.v); }, moment, 1, "second moments");
  if (has_master)
    check_apart(table, [](const Entry& t) { return reinterpret_cast<char*>(t.master); }, 4, 1, "masters");
  if (bits8) {
    check_apart(table, [](const Entry& t) { return reinterpret_cast<char*>(t.m_scale); }, 4, kBlock, "factors");
    check_apart(table, [](const Entry& t) { return reinterpret_cast<char*>(t.v_scale); }, 4, kBlock, "factors");
  }
  c10::cuda::CUDAGuard guard(device);
  const int rc = slapo::launch_adamw_multi(table.data(), static_cast<int>(table.size()), s, bits8, code,
                                           at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(rc == 0, "multi_adamw: launch refused (code ", rc, ")");
  // (autograd notices that weights it has saved have changed.  Moments and factors, which nothing is computed from but the
  // next step, are not worth it: 67 us for 57 in a step of 300 small tensors in 8 bits.)
  for (const List* list : {&x.params, &x.masters})
    for (size_t i = 0; i < list->size; ++i)
      if (!(*list)[i].is_inference()) (*list)[i].unsafeGetTensorImpl()->bump_version();
}

using Ops = at::TensorList;

void multi_adamw(Ops params, Ops grads, Ops masters, Ops exp_avgs, Ops exp_avg_sqs, Ops exp_avg_scales,
                 Ops exp_avg_sq_scales, at::ArrayRef<double> lrs, at::ArrayRef<double> weight_decays, double beta1,
                 double beta2, double eps, int64_t step, const optional<Tensor>& step_tensor,
                 const optional<Tensor>& grad_scale) {
  std::vector<std::vector<const Tensor*>> at;
  at.reserve(7);
  auto list = [&](Ops tensors) {
    at.emplace_back();
    at.back().reserve(tensors.size());
    for (const Tensor& t : tensors) at.back().push_back(&t);
    return List{at.back().data(), at.back().size()};
  };
  AdamwLists x{list(params), list(grads), list(masters), list(exp_avgs), list(exp_avg_sqs), list(exp_avg_scales),
               list(exp_avg_sq_scales), lrs.data(), lrs.size(), weight_decays.data(), weight_decays.size(), beta1, beta2,
               eps, step, nullptr, nullptr};
  if (step_tensor.has_value() && step_tensor->defined()) x.step_tensor = &*step_tensor;
  if (grad_scale.has_value() && grad_scale->defined()) x.grad_scale = &*grad_scale;
  run(x);
}

}  // namespace

void register_optim_ops(torch::Library& m) {
  m.def("multi_adamw(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] masters, Tensor(c!)[] exp_avgs, Tensor(d!)[] exp_avg_sqs, Tensor(e!)[] exp_avg_scales, Tensor(f!)[] exp_avg_sq_scales, float[] lrs, float[] weight_decays, float beta1, float beta2, float eps, int step, Tensor? step_tensor, Tensor? grad_scale) -> ()",
        &multi_adamw);
  // for py_entry.cpp: where the function that takes the lists is
  m.def("multi_adamw_entry() -> int", []() -> int64_t { return reinterpret_cast<int64_t>(&run); });
}
