// slapo_b200._py: entry points that take Python lists of tensors as they are.
//
// A registered operator's lists are converted element by element, twice, on their way through the dispatcher: 0.1 us
// for each tensor, which for the two thousand of an optimizer step's lists (300 parameters, their gradients, moments
// and factors) was 190 us of host time around a kernel of 30.  This module reads the lists in place and calls the
// function behind the operator `multi_adamw`, whose address the operator `multi_adamw_entry` gives: 59 us there, and
// 14 instead of 40 for 60 tensors.
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include <exception>
#include <vector>

#include "optim_entry.h"

namespace {

using slapo::AdamwLists;

// Tensors that the dispatcher has to see (subclasses with a dispatch of their own, fake ones, function transforms,
// lazy signs): for these the operator is called.
bool plain(const at::Tensor& t) {
  static const c10::DispatchKeySet others({c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot,
                                           c10::DispatchKey::Functionalize, c10::DispatchKey::FuncTorchBatched,
                                           c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Batched,
                                           c10::DispatchKey::Conjugate, c10::DispatchKey::Negative,
                                           c10::DispatchKey::ZeroTensor});
  return t.defined() && !t.key_set().has_any(others);
}

bool tensors(PyObject* list, std::vector<const at::Tensor*>& to, AdamwLists::List& at, bool& all_plain) {
  if (!PyList_CheckExact(list)) {
    PyErr_SetString(PyExc_TypeError, "multi_adamw: lists of tensors required");
    return false;
  }
  const Py_ssize_t n = PyList_GET_SIZE(list);
  to.reserve(static_cast<size_t>(n));
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* item = PyList_GET_ITEM(list, i);
    if (!THPVariable_Check(item)) {
      PyErr_SetString(PyExc_TypeError, "multi_adamw: lists of tensors required");
      return false;
    }
    to.push_back(&THPVariable_Unpack(item));
    all_plain = all_plain && plain(*to.back());
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
  to = &THPVariable_Unpack(item);
  all_plain = all_plain && plain(*to);
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
  try {
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
    if (!all_plain) Py_RETURN_FALSE;
    entry(x);
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
  Py_RETURN_TRUE;
}

PyMethodDef methods[] = {{"multi_adamw", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&multi_adamw)),
                          METH_FASTCALL, "One AdamW step on lists of tensors (see slapo_b200.ops.adamw)."},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_py", "Entry points that take Python lists of tensors.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__py() { return PyModule_Create(&module); }
