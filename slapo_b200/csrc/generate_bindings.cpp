// torch bindings of rotation by positions, the paged cache in 8 bits and sampling.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <climits>
#include <cmath>

#include "generate.h"
#include "kernels.h"
#include "py_entry.h"

namespace {

using at::Tensor;
using c10::optional;

// A new contiguous tensor on the current device, without the dispatcher (half a microsecond less)
Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt);
}

int dtype_code(const Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return 0;
    case at::kHalf: return 1;
    case at::kFloat: return 2;
    default: TORCH_CHECK_TYPE(false, what, ": bf16, fp16 or fp32 required, not ", t.scalar_type());
  }
}

void check_on(const Tensor& t, const Tensor& other, const char* what) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.device() == other.device(), what, " must be on ", other.device(), ", not on ", t.device());
}

// Generation: nothing here is differentiated
void check_no_gradient(std::initializer_list<const Tensor*> inputs, const char* what) {
  TORCH_CHECK(!slapo::transforming(), "slapo_b200's CUDA layers do not support functorch transforms (vmap, grad, jvp, ...)");
  for (const Tensor* t : inputs)
    TORCH_CHECK(!(at::GradMode::is_enabled() && t->requires_grad()) && !t->_fw_grad(/*level=*/0).defined(), what,
                " has no gradient: call it under torch.no_grad()");
}

// The table as the kernels read it, pair by pair: a copy where its pairs are not one after the other on 8 bytes
Tensor rotary_rows(const Tensor& table, const Tensor& x) {
  check_on(table, x, "rotary: the table");
  TORCH_CHECK_TYPE(table.scalar_type() == at::kFloat, "rotary: a table of fp32 required, not ", table.scalar_type());
  TORCH_CHECK_VALUE(table.dim() == 3 && table.size(2) == 2 && table.size(1) >= 1 && 2 * table.size(1) <= x.size(-1),
                    "rotary: a table [positions, rotated / 2, 2] of at most the head's ", x.size(-1), " values required, not ",
                    table.sizes());
  if (table.is_contiguous() && reinterpret_cast<uintptr_t>(table.const_data_ptr()) % 8 == 0) return table;
  c10::cuda::CUDAGuard guard(x.device());
  return table.clone(at::MemoryFormat::Contiguous);
}

Tensor heads_in_rows(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }

// The heads of a tensor, or the `slice`-th ones of a packed projection.  (Views of it would take a microsecond each.)
slapo::RotaryPart part(const Tensor& x, const Tensor& y, bool turn, int slice = 0) {
  slapo::RotaryPart p{};
  const int64_t e = x.element_size();
  const bool packed = x.dim() == 5;
  p.x = static_cast<const char*>(x.const_data_ptr()) + (packed ? slice * x.stride(3) * e : 0);
  p.y = static_cast<char*>(y.data_ptr()) + (packed ? slice * y.stride(3) * e : 0);
  for (int d = 0; d < 3; ++d) {
    p.x_stride[d] = x.stride(d);
    p.y_stride[d] = y.stride(d);
  }
  p.heads = static_cast<int>(x.size(2));
  p.turn = turn;
  return p;
}

// q [B, S, H, D] and k (heads of its own), or the packed projection [B, S, H, 3, D] alone; new tensors
std::tuple<Tensor, Tensor> rotary_fwd(const Tensor& q_in, const optional<Tensor>& k_in, const Tensor& table_in,
                                      const optional<Tensor>& positions, int64_t start, bool interleaved, bool transposed) {
  const bool packed = !k_in.has_value();
  TORCH_CHECK_VALUE(q_in.is_cuda() && q_in.dim() == (packed ? 5 : 4) && (!packed || q_in.size(3) == 3),
                    packed ? "rotary: a CUDA tensor [B, S, H, 3, D] required, not "
                           : "rotary: CUDA tensors [B, S, H, D] required, not ", q_in.sizes());
  const int code = dtype_code(q_in, "rotary");
  const Tensor table = rotary_rows(table_in, q_in);
  TORCH_CHECK_VALUE(q_in.size(-1) <= 256 && q_in.size(2) <= INT_MAX, "rotary: heads of at most 256 values required");
  c10::cuda::CUDAGuard guard(q_in.device());
  const Tensor q = heads_in_rows(q_in);
  Tensor k, out_q, out_k;
  slapo::RotaryCall c{};
  if (packed) {
    out_q = empty(q.sizes(), q.scalar_type(), q);
    for (int i = 0; i < 3; ++i) c.part[i] = part(q, out_q, i < 2, i);
    c.parts = 3;
  } else {
    check_on(*k_in, q, "rotary: k");
    TORCH_CHECK_TYPE(k_in->scalar_type() == q.scalar_type(), "rotary: q and k of one type required");
    TORCH_CHECK_VALUE(k_in->dim() == 4 && k_in->size(0) == q.size(0) && k_in->size(1) == q.size(1) && k_in->size(3) == q.size(3) &&
                          k_in->size(2) <= INT_MAX,
                      "rotary: k [B, S, heads, D] of q's tokens and width required: ", k_in->sizes(), " and ", q.sizes());
    k = heads_in_rows(*k_in);
    out_q = empty(q.sizes(), q.scalar_type(), q);
    out_k = empty(k.sizes(), k.scalar_type(), k);
    c.part[0] = part(q, out_q, true);
    c.part[1] = part(k, out_k, true);
    c.parts = 2;
  }
  c.table = table.const_data_ptr<float>();
  c.table_rows = table.size(0);
  c.B = q.size(0);
  c.S = q.size(1);
  c.D = static_cast<int>(q.size(-1));
  c.rotary = static_cast<int>(2 * table.size(1));
  c.interleaved = interleaved;
  c.transposed = transposed;
  c.dtype = code;
  c.at.start = start;
  if (positions.has_value()) {
    const Tensor& p = *positions;
    check_on(p, q, "rotary: positions");
    TORCH_CHECK_TYPE(p.scalar_type() == at::kLong || p.scalar_type() == at::kInt,
                     "rotary: positions of int64 or int32 required, not ", p.scalar_type());
    TORCH_CHECK_VALUE((p.dim() == 1 && p.size(0) == c.S) ||
                          (p.dim() == 2 && (p.size(0) == c.B || p.size(0) == 1) && p.size(1) == c.S),
                      "rotary: positions [S], [1, S] or [B, S] required, not ", p.sizes());
    c.at.ids = p.const_data_ptr();
    c.at.ids64 = p.scalar_type() == at::kLong;
    c.at.batch_stride = p.dim() == 2 && p.size(0) > 1 ? p.stride(0) : 0;
    c.at.token_stride = p.stride(-1);
  }
  const int rc = slapo::launch_rotary(c, at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(rc == 0, "rotary: launch refused (code ", rc, ")");
  return {out_q, out_k};
}

// What append and attention take alike; q_like: [B, n, heads, D]
slapo::PagedCache check_cache(const Tensor& pages, const Tensor& scales, const Tensor& block_table, const Tensor& lengths,
                              const optional<Tensor>& counts, const Tensor& q_like, const char* what) {
  TORCH_CHECK_VALUE(q_like.is_cuda() && q_like.dim() == 4, what, ": CUDA tensors [B, n, heads, D] required, not ", q_like.sizes());
  check_on(pages, q_like, "pages");
  check_on(scales, q_like, "scales");
  check_on(block_table, q_like, "block_table");
  check_on(lengths, q_like, "lengths");
  TORCH_CHECK_TYPE(pages.scalar_type() == at::kFloat8_e4m3fn, what, ": pages of float8_e4m3fn required, not ", pages.scalar_type());
  TORCH_CHECK_TYPE(scales.scalar_type() == at::kFloat, what, ": scales of fp32 required, not ", scales.scalar_type());
  TORCH_CHECK_VALUE(pages.dim() == 5 && pages.size(0) >= 1 && pages.size(1) == 2 && pages.is_contiguous() &&
                        reinterpret_cast<uintptr_t>(pages.const_data_ptr()) % 16 == 0,
                    what, ": contiguous pages [pages, 2, heads, tokens, width] on 16 bytes required, not ", pages.sizes());
  const int64_t d = q_like.size(3), t = pages.size(3);
  TORCH_CHECK_VALUE(d >= 8 && d <= 128 && d % 8 == 0, what, ": heads of 8 to 128 values, a multiple of 8, required, not ", d);
  TORCH_CHECK_VALUE(t == 16 || t == 32 || t == 64 || t == 128, what, ": pages of 16, 32, 64 or 128 tokens required, not ", t);
  TORCH_CHECK_VALUE(pages.size(4) == (d + 15) / 16 * 16, what, ": pages of ", (d + 15) / 16 * 16, " values a token for heads of ", d,
                    " required, not ", pages.size(4));
  TORCH_CHECK_VALUE(scales.dim() == 3 && scales.size(0) == pages.size(0) && scales.size(1) == 2 && scales.size(2) == pages.size(2) &&
                        scales.is_contiguous(),
                    what, ": contiguous scales [pages, 2, heads] required, not ", scales.sizes());
  const int64_t b = q_like.size(0);
  TORCH_CHECK_TYPE(block_table.scalar_type() == at::kInt && lengths.scalar_type() == at::kInt, what,
                   ": block_table and lengths of int32 required");
  TORCH_CHECK_VALUE(block_table.dim() == 2 && block_table.size(0) == b && block_table.is_contiguous(), what,
                    ": a contiguous block_table [", b, ", pages] required, not ", block_table.sizes());
  TORCH_CHECK_VALUE(lengths.dim() == 1 && lengths.size(0) == b && lengths.is_contiguous(), what, ": contiguous lengths [", b,
                    "] required, not ", lengths.sizes());
  if (counts.has_value()) {
    check_on(*counts, q_like, "counts");
    TORCH_CHECK_TYPE(counts->scalar_type() == at::kInt, what, ": counts of int32 required, not ", counts->scalar_type());
    TORCH_CHECK_VALUE(counts->dim() == 1 && counts->size(0) == b && counts->is_contiguous(), what, ": contiguous counts [", b,
                      "] required, not ", counts->sizes());
  }
  TORCH_CHECK_VALUE(block_table.size(1) * t <= INT_MAX - 256 && pages.size(0) <= INT_MAX && pages.size(2) <= 65535 && b <= INT_MAX &&
                        q_like.size(1) <= INT_MAX - 256 && q_like.size(2) <= 65535,
                    what, ": more tokens, pages or heads than have a number");
  slapo::PagedCache c{};
  c.pages = static_cast<uint8_t*>(pages.data_ptr());
  c.scales = scales.data_ptr<float>();
  c.n_pages = pages.size(0);
  c.heads = static_cast<int>(pages.size(2));
  c.page = static_cast<int>(t);
  c.dim = static_cast<int>(d);
  c.pitch = static_cast<int>(pages.size(4));
  c.table = block_table.const_data_ptr<int32_t>();
  c.table_pages = static_cast<int>(block_table.size(1));
  c.lengths = lengths.const_data_ptr<int32_t>();
  c.counts = counts.has_value() ? counts->const_data_ptr<int32_t>() : nullptr;
  c.B = static_cast<int>(b);
  c.n = static_cast<int>(q_like.size(1));
  return c;
}

// D contiguous, heads on 16 bytes, as vectors are read; else a copy
Tensor vectors(const Tensor& t) {
  const int64_t e = t.element_size();
  const bool fine = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0 && t.stride(0) * e % 16 == 0 &&
                    t.stride(1) * e % 16 == 0 && t.stride(2) * e % 16 == 0;
  return fine ? t : t.clone(at::MemoryFormat::Contiguous);
}

Tensor paged_append(const Tensor& pages, const Tensor& scales, const Tensor& k_in, const Tensor& v_in, const Tensor& block_table,
                    const Tensor& lengths, const optional<Tensor>& counts, const optional<Tensor>& q_in,
                    const optional<Tensor>& rot, bool interleaved) {
  slapo::PagedAppend a{};
  a.cache = check_cache(pages, scales, block_table, lengths, counts, k_in, "paged_append");
  check_no_gradient({&k_in, &v_in}, "paged_append");
  a.dtype = dtype_code(k_in, "paged_append");
  check_on(v_in, k_in, "paged_append: v");
  TORCH_CHECK_TYPE(v_in.scalar_type() == k_in.scalar_type(), "paged_append: k and v of one type required");
  TORCH_CHECK_VALUE(v_in.sizes() == k_in.sizes() && k_in.size(2) == pages.size(2), "paged_append: k and v [B, n, ", pages.size(2),
                    ", D] required, not ", k_in.sizes(), " and ", v_in.sizes());
  Tensor table;
  if (rot.has_value()) {
    table = rotary_rows(*rot, k_in);
    a.rot = table.const_data_ptr<float>();
    a.rot_rows = table.size(0);
    a.rotary = static_cast<int>(2 * table.size(1));
    a.interleaved = interleaved;
  }
  c10::cuda::CUDAGuard guard(k_in.device());
  const Tensor k = vectors(k_in), v = vectors(v_in);
  Tensor q, out;
  if (q_in.has_value()) {
    check_no_gradient({&*q_in}, "paged_append");
    check_on(*q_in, k_in, "paged_append: q");
    TORCH_CHECK_TYPE(q_in->scalar_type() == k_in.scalar_type(), "paged_append: q of k's type required");
    TORCH_CHECK_VALUE(q_in->dim() == 4 && q_in->size(0) == k_in.size(0) && q_in->size(1) == k_in.size(1) &&
                          q_in->size(3) == k_in.size(3) && q_in->size(2) <= 65535,
                      "paged_append: q [B, n, heads, D] of k's tokens and width required: ", q_in->sizes(), " and ", k_in.sizes());
    q = vectors(*q_in);
    out = empty(q.sizes(), q.scalar_type(), q);
    a.q = q.const_data_ptr();
    a.q_out = out.data_ptr();
    a.q_heads = static_cast<int>(q.size(2));
  } else {
    out = empty({0}, k.scalar_type(), k);
  }
  a.k = k.const_data_ptr();
  a.v = v.const_data_ptr();
  for (int d = 0; d < 3; ++d) {
    a.k_stride[d] = k.stride(d);
    a.v_stride[d] = v.stride(d);
    a.q_stride[d] = q.defined() ? q.stride(d) : 0;
  }
  const int rc = slapo::launch_paged_append(a, at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(rc == 0, "paged_append: launch refused (code ", rc, ")");
  for (const Tensor* t : {&pages, &scales})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  return out;
}

Tensor paged_attention(const Tensor& q_in, const Tensor& pages, const Tensor& scales, const Tensor& block_table,
                       const Tensor& lengths, const optional<Tensor>& counts, optional<double> scale, int64_t window) {
  slapo::PagedAttention a{};
  a.cache = check_cache(pages, scales, block_table, lengths, counts, q_in, "paged_attention");
  check_no_gradient({&q_in}, "paged_attention");
  TORCH_CHECK_TYPE(q_in.scalar_type() == at::kBFloat16 || q_in.scalar_type() == at::kHalf,
                   "paged_attention: queries of bf16 or fp16 required, not ", q_in.scalar_type());
  TORCH_CHECK_VALUE(pages.size(2) > 0 ? q_in.size(2) % pages.size(2) == 0 : q_in.size(2) == 0,
                    "paged_attention: a multiple of the cache's ", pages.size(2), " heads required, not ", q_in.size(2));
  TORCH_CHECK_VALUE(window >= 0, "a window is a number of keys, 1 and more, not ", window);
  TORCH_CHECK_VALUE(q_in.size(1) * std::max<int64_t>(q_in.size(2), 1) <= INT_MAX - 256, "paged_attention: too many queries");
  c10::cuda::CUDAGuard guard(q_in.device());
  const Tensor q = vectors(q_in);
  Tensor out = empty(q.sizes(), q.scalar_type(), q);
  a.q = q.const_data_ptr();
  for (int d = 0; d < 3; ++d) a.q_stride[d] = q.stride(d);
  a.q_heads = static_cast<int>(q.size(2));
  a.out = out.data_ptr();
  a.scale = static_cast<float>(scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(q.size(3))));
  a.window = static_cast<int>(std::min<int64_t>(window, INT_MAX));        // (positions are below that)
  a.bf16 = q.scalar_type() == at::kBFloat16;
  Tensor scratch;
  if (out.numel() > 0) {
    scratch = empty({slapo::paged_attention_words(a)}, at::kFloat, q);
    a.scratch = scratch.data_ptr<float>();
  }
  const int rc = slapo::launch_paged_attention(a, at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(rc == 0, "paged_attention: launch refused (code ", rc, ")");
  return out;
}

// (kept: a copy where rows are not one after the other, alive until the launch)
template <typename N, typename M>
slapo::PerRow<M> per_row(const slapo::Setting<N>& s, int64_t rows, at::ScalarType type, const Tensor& logits, const char* name,
                         Tensor& kept) {
  if (!s.rows.has_value()) return {nullptr, static_cast<M>(s.value)};
  check_on(*s.rows, logits, name);
  TORCH_CHECK_TYPE(s.rows->scalar_type() == type, "sample: ", name, " of ", type, " required, not ", s.rows->scalar_type());
  TORCH_CHECK_VALUE(s.rows->numel() == rows, "sample: one ", name, " for each of the ", rows, " rows required");
  if (s.rows->is_contiguous()) return {static_cast<const M*>(s.rows->const_data_ptr()), M()};
  kept = s.rows->contiguous();
  return {static_cast<const M*>(kept.const_data_ptr()), M()};
}

Tensor sample(const Tensor& logits_in, const Tensor& uniform_in, const slapo::Setting<double>& temperature,
              const slapo::Setting<int64_t>& top_k, const slapo::Setting<double>& top_p, const slapo::Setting<double>& min_p) {
  TORCH_CHECK_VALUE(logits_in.is_cuda() && logits_in.dim() >= 1, "sample: CUDA logits [..., vocabulary] required");
  slapo::SampleCall c{};
  c.dtype = dtype_code(logits_in, "sample");
  check_on(uniform_in, logits_in, "sample: random numbers");
  TORCH_CHECK_TYPE(uniform_in.scalar_type() == at::kFloat, "sample: random numbers of fp32 required, not ",
                   uniform_in.scalar_type());
  const int64_t vocab = logits_in.size(-1);
  TORCH_CHECK_VALUE(vocab >= 1 && vocab <= slapo::kSampleVocab, "sample: a vocabulary of 1 to ", slapo::kSampleVocab,
                    " tokens required, not ", vocab);
  const int64_t rows = logits_in.numel() / vocab;
  TORCH_CHECK_VALUE(uniform_in.numel() == rows, "sample: one random number for each of the ", rows, " rows required, not ",
                    uniform_in.sizes());
  TORCH_CHECK_VALUE(temperature.rows.has_value() || temperature.value >= 0.0, "sample: a temperature of 0 or more required, not ",
                    temperature.value);
  TORCH_CHECK_VALUE(top_k.rows.has_value() || top_k.value >= 0, "sample: top_k is a number of tokens, or 0, not ", top_k.value);
  TORCH_CHECK_VALUE(top_p.rows.has_value() || (top_p.value >= 0.0 && top_p.value <= 1.0), "sample: top_p between 0 and 1 required, not ",
                    top_p.value);
  TORCH_CHECK_VALUE(min_p.rows.has_value() || (min_p.value >= 0.0 && min_p.value <= 1.0), "sample: min_p between 0 and 1 required, not ",
                    min_p.value);
  c10::cuda::CUDAGuard guard(logits_in.device());
  const Tensor logits = logits_in.dim() == 2 && logits_in.stride(1) == 1 ? logits_in : logits_in.reshape({rows, vocab}).contiguous();
  const Tensor uniform = uniform_in.is_contiguous() ? uniform_in : uniform_in.contiguous();
  Tensor kept[4], out = empty(logits_in.sizes().slice(0, logits_in.dim() - 1), at::kLong, logits);
  c.logits = logits.const_data_ptr();
  c.row_stride = logits.stride(0);
  c.uniform = uniform.const_data_ptr<float>();
  c.temperature = per_row<double, float>(temperature, rows, at::kFloat, logits, "temperature", kept[0]);
  slapo::Setting<int64_t> most = top_k;
  most.value = std::min<int64_t>(most.value, INT_MAX);
  c.top_k = per_row<int64_t, int>(most, rows, at::kInt, logits, "top_k", kept[1]);
  c.top_p = per_row<double, float>(top_p, rows, at::kFloat, logits, "top_p", kept[2]);
  c.min_p = per_row<double, float>(min_p, rows, at::kFloat, logits, "min_p", kept[3]);
  c.out = out.data_ptr<int64_t>();
  c.rows = rows;
  c.vocab = static_cast<int>(vocab);
  const int rc = slapo::launch_sample(c, at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(rc == 0, "sample: launch refused (code ", rc, ")");
  return out;
}

}  // namespace

void register_generate_ops(torch::Library& m) {
  m.def("rotary_fwd(Tensor q, Tensor? k, Tensor table, Tensor? positions, int start, bool interleaved, bool transposed) -> (Tensor, Tensor)",
        &rotary_fwd);
  m.def("paged_append(Tensor(a!) pages, Tensor(b!) scales, Tensor k, Tensor v, Tensor block_table, Tensor lengths, Tensor? counts, Tensor? q, Tensor? rotary_table, bool interleaved) -> Tensor",
        &paged_append);
  m.def("paged_attention(Tensor q, Tensor pages, Tensor scales, Tensor block_table, Tensor lengths, Tensor? counts, float? scale, int window) -> Tensor",
        &paged_attention);
  m.def("sample(Tensor logits, Tensor uniform, float temperature, Tensor? temperatures, int top_k, Tensor? top_ks, float top_p, Tensor? top_ps, float min_p, Tensor? min_ps) -> Tensor",
        [](const Tensor& logits, const Tensor& uniform, double temperature, const optional<Tensor>& temperatures, int64_t top_k,
           const optional<Tensor>& top_ks, double top_p, const optional<Tensor>& top_ps, double min_p,
           const optional<Tensor>& min_ps) {
          return sample(logits, uniform, {temperature, temperatures}, {top_k, top_ks}, {top_p, top_ps}, {min_p, min_ps});
        });
  // for py_entry.cpp: where these functions are
  m.def("paged_append_entry() -> int",
        []() -> int64_t { return reinterpret_cast<int64_t>(static_cast<slapo::PagedAppendEntry>(&paged_append)); });
  m.def("paged_attention_entry() -> int",
        []() -> int64_t { return reinterpret_cast<int64_t>(static_cast<slapo::PagedAttentionEntry>(&paged_attention)); });
  m.def("sample_entry() -> int", []() -> int64_t { return reinterpret_cast<int64_t>(static_cast<slapo::SampleEntry>(&sample)); });
}
