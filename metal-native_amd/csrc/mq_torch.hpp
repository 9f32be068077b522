// Shared by the sources of the native torch front (_mq_torch.so).
#pragma once
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>

namespace mq_front {

bool modes_set();                          // a dispatch or function mode is active
const at::Tensor* plain(PyObject* o);      // null where it is not an ordinary strided GPU tensor
inline PyObject* decline() { Py_RETURN_NONE; }

PyObject* paged_rope_kv(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* paged_attention_mass(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* paged_evict(PyObject*, PyObject* const* a, Py_ssize_t n);

}  // namespace mq_front
