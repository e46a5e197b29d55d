// slapo_b200._py: entry points for calls whose host time counts.
//
// Lists of tensors: a registered operator's lists are converted element by element, twice, on their way through the
// dispatcher: 0.1 us for each tensor, which for the two thousand of an optimizer step's lists (300 parameters, their
// gradients, moments and factors) was 190 us of host time around a kernel of 30.  This module reads the lists in place
// and calls the function behind the operator `multi_adamw`, whose address the operator `multi_adamw_entry` gives: 59 us
// there, and 14 instead of 40 for 60 tensors.
//
// Attention and lookup of a token of generation: arguments that are matched with an operator's schema, and checks that
// are made in Python before, cost as much as the launch.
//
// What the dispatcher has to see goes to the operators: each function here says so by its result, with nothing done.
#include <Python.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <vector>

#include "py_entry.h"

namespace {

using slapo::AdamwLists;

// Whether something watches calls that pass through the dispatcher: modes, function transforms, a tracer
bool watched() {
  return c10::impl::TorchDispatchModeTLS::any_modes_set() || at::impl::torch_function_mode_enabled() ||
         slapo::transforming() ||
         c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::Tracer);
}

// A tensor or a parameter, no subclass, that the dispatcher has not to see (fake ones, lazy signs); else null
const at::Tensor* plain(PyObject* item) {
  static const c10::DispatchKeySet others({c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot,
                                           c10::DispatchKey::Functionalize, c10::DispatchKey::FuncTorchBatched,
                                           c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Batched,
                                           c10::DispatchKey::Conjugate, c10::DispatchKey::Negative,
                                           c10::DispatchKey::ZeroTensor});
  if (!THPVariable_CheckExact(item)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(item);
  return t.defined() && !t.key_set().has_any(others) ? &t : nullptr;
}

// Other Python threads run while this one allocates and launches.
struct WithoutGil {
  PyThreadState* state = PyEval_SaveThread();
  ~WithoutGil() { PyEval_RestoreThread(state); }
};

bool tensors(PyObject* list, std::vector<const at::Tensor*>& to, AdamwLists::List& at, bool& all_plain) {
  if (!PyList_CheckExact(list)) {
    PyErr_SetString(PyExc_TypeError, "multi_adamw: lists of tensors required");
    return false;
  }
  const Py_ssize_t n = PyList_GET_SIZE(list);
  to.reserve(static_cast<size_t>(n));
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* item = PyList_GET_ITEM(list, i);
    const at::Tensor* t = plain(item);
    if (t == nullptr) {
      if (!THPVariable_Check(item)) {
        PyErr_SetString(PyExc_TypeError, "multi_adamw: lists of tensors required");
        return false;
      }
      all_plain = false;
    }
    to.push_back(t);
  }
  at = {to.data(), to.size()};
  return true;
}

bool numbers(PyObject* list, std::vector<double>& to) {
  if (!PyList_CheckExact(list)) {
    PyErr_SetString(PyExc_TypeError, "multi_adamw: lists of numbers required");
    return false;
  }
  const Py_ssize_t n = PyList_GET_SIZE(list);
  to.reserve(static_cast<size_t>(n));
  for (Py_ssize_t i = 0; i < n; ++i) {
    const double v = PyFloat_AsDouble(PyList_GET_ITEM(list, i));
    if (v == -1.0 && PyErr_Occurred()) return false;
    to.push_back(v);
  }
  return true;
}

bool maybe_tensor(PyObject* item, const at::Tensor*& to, bool& all_plain) {
  to = nullptr;
  if (item == Py_None) return true;
  if (!THPVariable_Check(item)) {
    PyErr_SetString(PyExc_TypeError, "multi_adamw: a tensor or None required");
    return false;
  }
  to = plain(item);
  all_plain = all_plain && to != nullptr;
  return true;
}

// multi_adamw(entry, params, grads, masters, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, lrs,
//             weight_decays, beta1, beta2, eps, step, step_tensor, grad_scale) -> whether it was done: False, with
// nothing done, where a tensor has to go through the dispatcher
PyObject* multi_adamw(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  if (n_args != 16) {
    PyErr_SetString(PyExc_TypeError, "multi_adamw takes 16 arguments");
    return nullptr;
  }
  HANDLE_TH_ERRORS
  const auto entry = reinterpret_cast<slapo::AdamwEntry>(PyLong_AsVoidPtr(args[0]));
  std::vector<const at::Tensor*> lists[7];
  std::vector<double> lrs, decays;
  AdamwLists x{};
  bool all_plain = true;
  AdamwLists::List* const to[7] = {&x.params,      &x.grads,          &x.masters, &x.exp_avgs,
                                   &x.exp_avg_sqs, &x.exp_avg_scales, &x.exp_avg_sq_scales};
  for (int i = 0; i < 7; ++i)
    if (!tensors(args[1 + i], lists[i], *to[i], all_plain)) return nullptr;
  if (!numbers(args[8], lrs) || !numbers(args[9], decays)) return nullptr;
  x.lrs = lrs.data();
  x.n_lrs = lrs.size();
  x.weight_decays = decays.data();
  x.n_weight_decays = decays.size();
  x.beta1 = PyFloat_AsDouble(args[10]);
  x.beta2 = PyFloat_AsDouble(args[11]);
  x.eps = PyFloat_AsDouble(args[12]);
  x.step = PyLong_AsLongLong(args[13]);
  if (PyErr_Occurred() || !maybe_tensor(args[14], x.step_tensor, all_plain) ||
      !maybe_tensor(args[15], x.grad_scale, all_plain))
    return nullptr;
  if (!all_plain || watched()) Py_RETURN_FALSE;
  {
    WithoutGil released;
    entry(x);
  }
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

bool count(PyObject* item, int64_t& to) {      // 0 for None
  to = item == Py_None ? 0 : PyLong_AsLongLong(item);
  return !(to == -1 && PyErr_Occurred());
}

// flash(entry, q, k, v, key_bias, causal, scale, window, sinks) -> output, or None where the kernels do not take it as it
// is.  key_bias, scale, window: or None.
PyObject* flash(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 9) {
    PyErr_SetString(PyExc_TypeError, "flash takes 9 arguments");
    return nullptr;
  }
  const at::Tensor* t[3];
  for (int i = 0; i < 3; ++i) {
    t[i] = plain(args[1 + i]);
    if (t[i] == nullptr || !t[i]->is_cuda() || t[i]->dim() != 4) Py_RETURN_NONE;
    const auto strides = t[i]->strides();
    if (strides[3] != 1 || ((strides[0] | strides[1] | strides[2]) & 7) != 0 ||
        (reinterpret_cast<uintptr_t>(t[i]->const_data_ptr()) & 15) != 0)
      Py_RETURN_NONE;
  }
  const auto type = t[0]->scalar_type();
  const int64_t d = t[0]->size(3);
  if ((type != at::kBFloat16 && type != at::kHalf) || d < 8 || d > 128 || d % 8 != 0 || watched()) Py_RETURN_NONE;
  std::optional<at::Tensor> bias;
  if (args[4] != Py_None) {
    const at::Tensor* b = plain(args[4]);
    if (b == nullptr || !b->is_cuda() || b->scalar_type() != at::kFloat || !b->is_contiguous()) Py_RETURN_NONE;
    bias = *b;
  }
  const int causal = PyObject_IsTrue(args[5]);
  const double scale = args[6] == Py_None ? 1.0 / std::sqrt(static_cast<double>(d)) : PyFloat_AsDouble(args[6]);
  int64_t window, sinks;
  const auto entry = reinterpret_cast<slapo::FlashEntry>(PyLong_AsVoidPtr(args[0]));
  if (causal < 0 || !count(args[7], window) || !count(args[8], sinks) || PyErr_Occurred()) return nullptr;
  at::Tensor out;
  {
    WithoutGil released;
    out = entry(*t[0], *t[1], *t[2], bias, std::nullopt, causal != 0, scale, 0.0, window, sinks);
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// embedding(entry, ids, weight, start, padding, scale) -> rows, or None where the kernels do not take it as it is.
// padding: or None.
PyObject* embedding(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 6) {
    PyErr_SetString(PyExc_TypeError, "embedding takes 6 arguments");
    return nullptr;
  }
  const at::Tensor *ids = plain(args[1]), *weight = plain(args[2]);
  if (ids == nullptr || weight == nullptr || !weight->is_cuda() || weight->dim() != 2 || watched()) Py_RETURN_NONE;
  const auto id = ids->scalar_type(), type = weight->scalar_type();
  if ((id != at::kLong && id != at::kInt) || (type != at::kBFloat16 && type != at::kHalf && type != at::kFloat))
    Py_RETURN_NONE;
  int64_t start, padding;
  const auto entry = reinterpret_cast<slapo::EmbeddingEntry>(PyLong_AsVoidPtr(args[0]));
  if (!count(args[3], start) || !count(args[4], padding)) return nullptr;
  const double scale = PyFloat_AsDouble(args[5]);
  if (PyErr_Occurred()) return nullptr;
  if (args[4] != Py_None && padding < 0) Py_RETURN_NONE;
  at::Tensor out;
  {
    WithoutGil released;
    out = entry(*ids, *weight, start, args[4] == Py_None ? std::nullopt : std::optional<int64_t>(padding), scale);
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

#define SLAPO_METHOD(NAME_, DOC_) \
  {#NAME_, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&NAME_)), METH_FASTCALL, DOC_}
PyMethodDef methods[] = {SLAPO_METHOD(multi_adamw, "One AdamW step on lists of tensors (see slapo_b200.ops.adamw)."),
                         SLAPO_METHOD(flash, "Attention (see slapo_b200.ops.functional.flash_attention)."),
                         SLAPO_METHOD(embedding, "Rows of a table (see slapo_b200.ops.functional.embedding)."),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_py", "Entry points for calls whose host time counts.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__py() { return PyModule_Create(&module); }
