// Shared by the sources of the native torch front (_mq_torch.so).
#pragma once
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <initializer_list>
#include <vector>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <torch/csrc/autograd/python_variable.h>

namespace mq_front {

bool modes_set();                          // a dispatch or function mode is active
const at::Tensor* plain(PyObject* o);      // null where it is not an ordinary strided GPU tensor
inline PyObject* decline() { Py_RETURN_NONE; }

inline bool vec(const at::Tensor* t, c10::Device dev, at::ScalarType ty, int64_t n) {
  return t && t->device() == dev && t->scalar_type() == ty && t->dim() == 1 && t->size(0) == n && t->is_contiguous();
}

inline bool as_int(PyObject* o, int64_t* v) {
  if (!PyLong_CheckExact(o)) return false;
  int over = 0;
  *v = PyLong_AsLongLongAndOverflow(o, &over);
  return !over;
}
inline bool as_float(PyObject* o, float* v) {
  if (!PyFloat_CheckExact(o) && !PyLong_CheckExact(o)) return false;
  *v = (float)PyFloat_AsDouble(o);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

// Device of a call, and dispatch below Python's modes: what is allocated here
// is launched on at once and has to be memory.
struct Call {
  c10::DeviceGuard device;
  c10::impl::ExcludeDispatchKeyGuard modes;
  explicit Call(c10::Device d)
      : device(d), modes(c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot})) {}
};

// whether autograd follows one of them (null: not given), which has a tangent of forward
// mode or requires a gradient; the Python side then refuses, or marks the outputs
inline bool tracked(std::initializer_list<const at::Tensor*> ts) {
  const bool backward = c10::GradMode::is_enabled();
  for (const at::Tensor* t : ts)
    if (t && ((backward && t->requires_grad()) || t->_fw_grad(0).defined())) return true;
  return false;
}

inline PyObject* status(int rc) { return PyLong_FromLong(rc); }
inline PyObject* wrong_count(const char* what) {
  PyErr_SetString(PyExc_TypeError, what);
  return nullptr;
}
// a tuple of outputs
inline PyObject* packed(std::vector<at::Tensor> ts) {
  PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
  for (size_t i = 0; r && i < ts.size(); ++i) {
    PyObject* o = THPVariable_Wrap(std::move(ts[i]));
    if (!o) {
      Py_DECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, (Py_ssize_t)i, o);
  }
  return r;
}

PyObject* paged_rope_kv(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* paged_attention_mass(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* paged_ancestors(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* paged_tree_attention(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* paged_accept(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* sample(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* paged_evict(PyObject*, PyObject* const* a, Py_ssize_t n);

}  // namespace mq_front
