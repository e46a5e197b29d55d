// Functions of this extension that py_entry.cpp calls without the dispatcher in between.
#pragma once
#include <ATen/ATen.h>
#include <c10/core/impl/LocalDispatchKeySet.h>

#include <optional>
#include <tuple>

namespace slapo {

// Whether a function transform is at work: calls pass through its layer then.  (Whether the thread has a record of
// transforms says less: it stays behind once one was made.)
inline bool transforming() {
  return c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) ||
         c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerBackMode);
}

// What AdamW over many tensors takes, as lists of tensors that live elsewhere.
struct AdamwLists {
  struct List {
    const at::Tensor* const* at;
    size_t size;
    const at::Tensor& operator[](size_t i) const { return *at[i]; }
  };
  List params, grads, masters, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales;
  const double* lrs;
  size_t n_lrs;
  const double* weight_decays;
  size_t n_weight_decays;
  double beta1, beta2, eps;
  int64_t step;
  const at::Tensor* step_tensor;       // or null
  const at::Tensor* grad_scale;        // or null
};
using AdamwEntry = void (*)(const AdamwLists&);

// q, k, v, key bias, relative bias, causal, scale, dropout, window, sinks
using FlashEntry = at::Tensor (*)(const at::Tensor&, const std::optional<at::Tensor>&, const std::optional<at::Tensor>&,
                                  const std::optional<at::Tensor>&, const std::optional<at::Tensor>&, bool, double, double,
                                  int64_t, int64_t);
// ids, table, first row, padding id, scale
using EmbeddingEntry = at::Tensor (*)(const at::Tensor&, const at::Tensor&, int64_t, const std::optional<int64_t>&, double);

// q (or the packed projection), k, table, positions (or the first one), interleaved
using RotaryEntry = std::tuple<at::Tensor, at::Tensor> (*)(const at::Tensor&, const std::optional<at::Tensor>&,
                                                           const at::Tensor&, const std::optional<at::Tensor>&, int64_t, bool);
// pages, scales, k, v, block table, lengths, counts, q, rotation's table, interleaved
using PagedAppendEntry = at::Tensor (*)(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                        const at::Tensor&, const at::Tensor&, const std::optional<at::Tensor>&,
                                        const std::optional<at::Tensor>&, const std::optional<at::Tensor>&, bool);
// q, pages, scales, block table, lengths, counts, scale, window
using PagedAttentionEntry = at::Tensor (*)(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                           const at::Tensor&, const std::optional<at::Tensor>&, std::optional<double>, int64_t);
// A setting: one number, or one for each row
template <typename N>
struct Setting {
  N value;
  std::optional<at::Tensor> rows;
};
// logits, random numbers, temperature, top_k, top_p, min_p
using SampleEntry = at::Tensor (*)(const at::Tensor&, const at::Tensor&, const Setting<double>&, const Setting<int64_t>&,
                                   const Setting<double>&, const Setting<double>&);

}  // namespace slapo
