// The host's side of an AdamW step over many small tensors, as a Python module (libmuon_amd_python.so):
// what the optimizer's state holds for each parameter is looked up here and handed to the operator
// muonium_amd::adamw_ of libmuon_amd_torch.so at once.
//
// A step of 129 tensors of a few thousand values takes the GPU 15 us; walking the parameters in Python
// took 435 us, of which the lookups of gradients, states and layouts were most.
#include <Python.h>

#include <algorithm>
#include <map>
#include <vector>

#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/core/grad_mode.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

namespace {

using at::Tensor;

typedef void Step(at::TensorList, at::TensorList, at::TensorList, at::TensorList, at::TensorList,
                  at::TensorList, at::TensorList, int64_t, double, double, double, double, double, bool);

struct Lists {
  std::vector<Tensor> params, grads, avgs, sqs, steps;
};

// What everybody's path takes: a plain tensor on a device, nothing that traces or wraps.
bool plain(const Tensor& t) {
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided && !t.key_set().has(c10::DispatchKey::Python) &&
         t.has_storage();
}
bool like(const Tensor& t, const Tensor& p) {
  return plain(t) && t.device() == p.device() && t.sizes() == p.sizes() &&
         (p.numel() <= 1 || t.strides() == p.strides());
}
const Tensor* tensor_at(PyObject* dict, PyObject* key) {
  PyObject* value = PyDict_GetItemWithError(dict, key);
  return value && THPVariable_CheckExact(value) ? &THPVariable_Unpack(value) : nullptr;
}

struct Keys {
  PyObject *step, *avg, *sq;
  Keys()
      : step(PyUnicode_InternFromString("step")), avg(PyUnicode_InternFromString("exp_avg")),
        sq(PyUnicode_InternFromString("exp_avg_sq")) {}
};

// step(params, state, lr, beta1, beta2, eps, weight_decay, maximize): steps the parameters of the list that
// have a gradient and fp32 moments laid out like them, and returns the list of those whose moments are
// something else. None, and nothing done, where a parameter has no state yet, is laid out unlike its
// gradient or moments, is no plain tensor, or shares memory with another one.
PyObject* step(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  static const Keys keys;
  if (nargs != 8 || !PyList_Check(args[0]) || !PyDict_Check(args[1])) {
    PyErr_SetString(PyExc_TypeError, "step(params, state, lr, beta1, beta2, eps, weight_decay, maximize)");
    return nullptr;
  }
  double numbers[5];
  for (int i = 0; i < 5; ++i) {
    numbers[i] = PyFloat_AsDouble(args[2 + i]);
    if (numbers[i] == -1.0 && PyErr_Occurred()) return nullptr;
  }
  const bool maximize = PyObject_IsTrue(args[7]);
  const Py_ssize_t n = PyList_GET_SIZE(args[0]);
  std::map<std::pair<int, int>, Lists> calls;
  std::vector<std::pair<uintptr_t, uintptr_t>> spans;
  std::vector<PyObject*> others;
  spans.reserve(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* object = PyList_GET_ITEM(args[0], i);
    if (!THPVariable_CheckExact(object)) Py_RETURN_NONE;
    const Tensor& p = THPVariable_Unpack(object);
    const Tensor& grad = p.grad();
    if (!grad.defined()) continue;
    if (!plain(p) || !p.is_non_overlapping_and_dense()) Py_RETURN_NONE;
    PyObject* held = PyDict_GetItemWithError(args[1], object);
    if (!held || !PyDict_Check(held)) {
      if (PyErr_Occurred()) return nullptr;
      Py_RETURN_NONE;
    }
    if (p.numel()) {
      const uintptr_t at = (uintptr_t)p.const_data_ptr();
      spans.emplace_back(at, at + p.nbytes());
    }
    const Tensor* avg = tensor_at(held, keys.avg);
    if (!avg) {
      if (PyErr_Occurred()) return nullptr;
      if (!PyDict_GetItemWithError(held, keys.avg)) Py_RETURN_NONE;
      others.push_back(object);
      continue;
    }
    const Tensor *sq = tensor_at(held, keys.sq), *count = tensor_at(held, keys.step);
    if (PyErr_Occurred()) return nullptr;
    if (!sq || !count || !like(grad, p) || grad.scalar_type() != p.scalar_type() || !like(*avg, p) || !like(*sq, p) ||
        avg->scalar_type() != at::kFloat || sq->scalar_type() != at::kFloat || !plain(*count) ||
        count->device() != p.device() || count->numel() != 1 || count->scalar_type() != at::kFloat)
      Py_RETURN_NONE;
    Lists& l = calls[{p.device().index(), (int)p.scalar_type()}];
    if (l.params.empty())
      for (auto* v : {&l.params, &l.grads, &l.avgs, &l.sqs, &l.steps}) v->reserve(n - i);
    l.params.push_back(p);
    l.grads.push_back(grad);
    l.avgs.push_back(*avg);
    l.sqs.push_back(*sq);
    l.steps.push_back(*count);
  }
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    if (spans[i].first < spans[i - 1].second) Py_RETURN_NONE;
  {
    at::NoGradGuard no_grad;
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("muonium_amd::adamw_", "").typed<Step>();
    for (auto& call : calls) {
      Lists& l = call.second;
      op.call(l.params, l.grads, l.avgs, l.sqs, {}, {}, l.steps, 0, numbers[0], numbers[1], numbers[2],
              numbers[3], numbers[4], maximize);
    }
  }
  PyObject* rest = PyList_New((Py_ssize_t)others.size());
  for (size_t i = 0; rest && i < others.size(); ++i) {
    Py_INCREF(others[i]);
    PyList_SET_ITEM(rest, (Py_ssize_t)i, others[i]);
  }
  return rest;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"adamw_step", (PyCFunction)(void (*)(void))step, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "libmuon_amd_python", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_libmuon_amd_python() { return PyModule_Create(&module); }
