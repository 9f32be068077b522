// Native front of the paged-cache operators: checks, allocation and launch as
// one CPython call.  Every function returns None for what it does not take as
// it is (paged.py then names the fault, or copies and calls again), an int for
// a status of the library, else the outputs.  Function and dispatch modes (a
// default device is one) make no difference: nothing here is theirs to change,
// and the outputs are allocated below them.
#include "mq_torch.hpp"

#include <algorithm>
#include <initializer_list>
#include <utility>

#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/metal_native_amd.h"

namespace mq_front {
namespace {

bool aligned16(const at::Tensor& t) { return ((uintptr_t)t.const_data_ptr() & 15) == 0; }

// [b, w] int32 rows of unit stride that do not overlap
bool index_rows(const at::Tensor& t, c10::Device dev) {
  return t.device() == dev && t.scalar_type() == at::kInt && t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1) &&
         (t.size(0) <= 1 || t.stride(0) >= t.size(1));
}
bool vec(const at::Tensor* t, c10::Device dev, at::ScalarType ty, int64_t n) {
  return t && t->device() == dev && t->scalar_type() == ty && t->dim() == 1 && t->size(0) == n && t->is_contiguous();
}

// no two elements share memory: each stride reaches past all smaller dimensions
bool distinct(const at::Tensor& t) {
  std::pair<int64_t, int64_t> d[4];
  int n = 0;
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1) d[n++] = {t.stride(i), t.size(i)};
  std::sort(d, d + n);
  int64_t span = 1;
  for (int i = 0; i < n; ++i) {
    if (d[i].first < span) return false;
    span = d[i].first * d[i].second;
  }
  return true;
}

struct Cache {
  mq_paged_cache c{};
  c10::Device dev = c10::Device(c10::kCPU);
  at::ScalarType ty = at::kHalf;

  bool one(const at::Tensor& t, int64_t* page, int64_t* head, int64_t* slot, bool write) const {
    if (t.dim() != 4 || t.stride(3) != 1 || !aligned16(t)) return false;
    *page = t.size(0) > 1 ? t.stride(0) : 0;
    *head = t.size(1) > 1 ? t.stride(1) : 0;
    *slot = t.stride(2);
    return *page % 8 == 0 && *head % 8 == 0 && *slot % 8 == 0 && *page >= 0 && *head >= 0 && *slot >= t.size(3) &&
           (!write || distinct(t));
  }
  // v null: keys alone
  bool take(PyObject* ko, PyObject* vo, PyObject* table, PyObject* lens, bool write) {
    const at::Tensor *k = plain(ko), *v = vo ? plain(vo) : k, *t = plain(table), *l = plain(lens);
    if (!k || !v || !t || !l) return false;
    dev = k->device();
    ty = k->scalar_type();
    if ((ty != at::kHalf && ty != at::kBFloat16) || v->scalar_type() != ty || v->device() != dev) return false;
    if (!one(*k, &c.k_page, &c.k_head, &c.k_slot, write) || !one(*v, &c.v_page, &c.v_head, &c.v_slot, write)) return false;
    if (k->sizes() != v->sizes() || !index_rows(*t, dev) || !vec(l, dev, at::kInt, t->size(0))) return false;
    if (t->size(0) < 1 || t->size(1) < 1 || k->numel() == 0) return false;
    if (k->size(1) > INT32_MAX || k->size(2) > INT32_MAX || k->size(3) > INT32_MAX) return false;
    c.k = const_cast<void*>(k->const_data_ptr());
    c.v = const_cast<void*>(v->const_data_ptr());
    c.pages = k->size(0);
    c.kv_heads = (int32_t)k->size(1);
    c.page_size = (int32_t)k->size(2);
    c.head_dim = (int32_t)k->size(3);
    c.dtype = ty == at::kHalf ? MQ_PAGED_F16 : MQ_PAGED_BF16;
    c.table = t->const_data_ptr<int32_t>();
    c.ld_table = t->size(0) > 1 ? t->stride(0) : t->size(1);
    c.width = t->size(1);
    c.batch = t->size(0);
    c.lens = l->const_data_ptr<int32_t>();
    return true;
  }
};

bool as_int(PyObject* o, int64_t* v) {
  if (!PyLong_CheckExact(o)) return false;
  int over = 0;
  *v = PyLong_AsLongLongAndOverflow(o, &over);
  return !over;
}
bool as_float(PyObject* o, float* v) {
  if (!PyFloat_CheckExact(o) && !PyLong_CheckExact(o)) return false;
  *v = (float)PyFloat_AsDouble(o);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}
bool chunks(PyObject* o, const Cache& k, int64_t rows, const int32_t** cu) {
  *cu = nullptr;
  if (o == Py_None) return rows == k.c.batch;
  const at::Tensor* t = plain(o);
  if (!vec(t, k.dev, at::kInt, k.c.batch + 1)) return false;
  *cu = t->const_data_ptr<int32_t>();
  return true;
}

// queries [rows, heads, dim]
struct Query {
  const at::Tensor* t = nullptr;
  int64_t rows = 0, heads = 0, s_t = 0, s_h = 0;
  bool take(PyObject* o, const Cache& k) {
    t = plain(o);
    if (!t || t->dim() != 3 || t->device() != k.dev || t->scalar_type() != k.ty || t->size(2) != k.c.head_dim ||
        t->stride(2) != 1)
      return false;
    rows = t->size(0);
    heads = t->size(1);
    s_t = rows > 1 ? t->stride(0) : 0;
    s_h = heads > 1 ? t->stride(1) : 0;
    return heads >= 1 && heads <= INT32_MAX && s_t % 8 == 0 && s_h % 8 == 0 && s_t >= 0 && s_h >= 0 && s_t <= 1 << 22 &&
           s_h <= 1 << 22 && (rows == 0 || aligned16(*t));
  }
};

// (cu, scale, softcap, slopes, window, prefix_lens, max_q)
bool mask(PyObject* const* a, const Cache& k, const Query& q, mq_paged_mask* m) {
  if (!chunks(a[0], k, q.rows, &m->cu_q) || !as_float(a[1], &m->scale) || !as_float(a[2], &m->softcap)) return false;
  m->slopes = nullptr;
  m->prefix_lens = nullptr;
  if (a[3] != Py_None) {
    const at::Tensor* t = plain(a[3]);
    if (!vec(t, k.dev, at::kFloat, q.heads)) return false;
    m->slopes = t->const_data_ptr<float>();
  }
  if (!as_int(a[4], &m->window)) return false;
  if (a[5] != Py_None) {
    const at::Tensor* t = plain(a[5]);
    if (!vec(t, k.dev, at::kInt, k.c.batch)) return false;
    m->prefix_lens = t->const_data_ptr<int32_t>();
  }
  return as_int(a[6], &m->max_q);
}

// Device of a call, and dispatch below Python's modes: what is allocated here
// is launched on at once and has to be memory.
struct Call {
  c10::DeviceGuard device;
  c10::impl::ExcludeDispatchKeyGuard modes;
  explicit Call(c10::Device d)
      : device(d), modes(c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot})) {}
};

// whether autograd follows one of them (null: not given); paged.py then marks
// the outputs as having no gradient
bool tracked(std::initializer_list<const at::Tensor*> ts) {
  if (!c10::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : ts)
    if (t && t->requires_grad()) return true;
  return false;
}
// a cache that the call wrote
void written(PyObject* o) {
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

PyObject* status(int rc) { return PyLong_FromLong(rc); }
PyObject* wrong_count(const char* what) {
  PyErr_SetString(PyExc_TypeError, what);
  return nullptr;
}

}  // namespace

// (qkv, cos, sin, pos, k, v, table, lens, cu, sections tuple | None, stream)
PyObject* paged_rope_kv(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 11) return wrong_count("paged_rope_kv: 11 arguments");
  Cache k;
  const at::Tensor *x = plain(a[0]), *co = plain(a[1]), *si = plain(a[2]), *pos = plain(a[3]);
  if (!x || !co || !si || !pos || !k.take(a[4], a[5], a[6], a[7], true) || tracked({x, co, si, plain(a[4]), plain(a[5])}))
    return decline();
  const int64_t D = k.c.head_dim, KVH = k.c.kv_heads;
  if (x->dim() != 2 || x->device() != k.dev || x->scalar_type() != k.ty || x->size(1) % D || x->size(1) / D <= 2 * KVH ||
      x->size(1) / D > INT32_MAX || x->stride(1) != 1)
    return decline();
  const int64_t rows = x->size(0), heads = x->size(1) / D - 2 * KVH, ld = rows > 1 ? x->stride(0) : x->size(1);
  if (ld % 8 || ld < x->size(1) || (rows > 0 && !aligned16(*x))) return decline();
  for (const at::Tensor* t : {co, si})
    if (t->device() != k.dev || t->scalar_type() != at::kFloat || t->dim() != 2 || t->size(1) != D || t->stride(1) != 1 ||
        t->size(0) < 1 || t->stride(0) % 4 || t->stride(0) < 0 || !aligned16(*t))
      return decline();
  if (co->size(0) != si->size(0)) return decline();
  int32_t sec[8];
  int axes = 1;
  if (a[9] != Py_None) {
    if (!PyTuple_CheckExact(a[9]) || PyTuple_GET_SIZE(a[9]) < 1 || PyTuple_GET_SIZE(a[9]) > 8) return decline();
    axes = (int)PyTuple_GET_SIZE(a[9]);
    for (int i = 0; i < axes; ++i) {
      int64_t v;
      if (!as_int(PyTuple_GET_ITEM(a[9], i), &v) || v < 0 || v > D / 2) return decline();
      sec[i] = (int32_t)v;
    }
  }
  if (pos->device() != k.dev || pos->scalar_type() != at::kLong || pos->dim() < 1 || pos->dim() > 2 ||
      (pos->dim() == 1 ? axes != 1 : pos->size(0) != axes) || pos->size(-1) != rows || (rows > 1 && pos->stride(-1) != 1))
    return decline();
  const int64_t ld_pos = pos->dim() == 2 && axes > 1 ? pos->stride(0) : rows;
  const int32_t* cu;
  if (!chunks(a[8], k, rows, &cu)) return decline();
  void* stream = PyLong_AsVoidPtr(a[10]);
  if (PyErr_Occurred()) return nullptr;
  HANDLE_TH_ERRORS
  const Call guard(k.dev);
  at::Tensor out = at::empty({rows, heads, D}, x->options());
  if (rows == 0) return THPVariable_Wrap(std::move(out));
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = mq_paged_rope_kv(&k.c, x->const_data_ptr(), ld, co->const_data_ptr<float>(), co->stride(0),
                        si->const_data_ptr<float>(), si->stride(0), co->size(0), pos->const_data_ptr<int64_t>(), ld_pos,
                        axes, a[9] == Py_None ? nullptr : sec, cu, rows, (int32_t)heads, out.mutable_data_ptr(), stream);
  Py_END_ALLOW_THREADS
  if (rc == MQ_SUCCESS) written(a[4]), written(a[5]);
  return rc == MQ_SUCCESS ? THPVariable_Wrap(std::move(out)) : status(rc);
  END_HANDLE_TH_ERRORS
}

// (q, k, v, table, lens, cu, scale, softcap, slopes, window, prefix_lens, max_q, return_lse, stream)
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 14) return wrong_count("paged_attention: 14 arguments");
  Cache k;
  Query q;
  mq_paged_mask m{};
  if (!k.take(a[1], a[2], a[3], a[4], false) || !q.take(a[0], k) || !mask(a + 5, k, q, &m) ||
      tracked({q.t, plain(a[1]), plain(a[2]), plain(a[8])}))
    return decline();
  const int want_lse = PyObject_IsTrue(a[12]);
  if (want_lse < 0) return nullptr;
  void* stream = PyLong_AsVoidPtr(a[13]);
  if (PyErr_Occurred()) return nullptr;
  HANDLE_TH_ERRORS
  const Call guard(k.dev);
  const int64_t wsb = mq_paged_attention_workspace_size(&k.c, &m, q.rows, (int32_t)q.heads);
  if (wsb < 0) return status(MQ_INVALID_ARGUMENT);
  at::Tensor out = at::empty({q.rows, q.heads, q.t->size(2)}, q.t->options());
  at::Tensor lse, ws;
  if (want_lse) lse = at::empty({q.rows, q.heads}, q.t->options().dtype(at::kFloat));
  if (wsb) ws = at::empty({wsb}, q.t->options().dtype(at::kByte));
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = mq_paged_attention(&k.c, &m, q.t->const_data_ptr(), q.s_t, q.s_h, q.rows, (int32_t)q.heads, out.mutable_data_ptr(),
                          want_lse ? lse.mutable_data_ptr<float>() : nullptr, wsb ? ws.mutable_data_ptr() : nullptr, wsb,
                          stream);
  Py_END_ALLOW_THREADS
  if (rc != MQ_SUCCESS) return status(rc);
  PyObject* o = THPVariable_Wrap(std::move(out));
  if (!want_lse || !o) return o;
  PyObject* l = THPVariable_Wrap(std::move(lse));
  if (!l) {
    Py_DECREF(o);
    return nullptr;
  }
  PyObject* r = PyTuple_Pack(2, o, l);
  Py_DECREF(o);
  Py_DECREF(l);
  return r;
  END_HANDLE_TH_ERRORS
}

// (q, k, table, lens, lse, cu, scale, softcap, slopes, window, prefix_lens, max_q, stream)
PyObject* paged_attention_mass(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 13) return wrong_count("paged_attention_mass: 13 arguments");
  Cache k;
  Query q;
  mq_paged_mask m{};
  const at::Tensor* lse = plain(a[4]);
  if (!lse || !k.take(a[1], nullptr, a[2], a[3], false) || !q.take(a[0], k) || !mask(a + 5, k, q, &m) ||
      tracked({q.t, plain(a[1]), lse, plain(a[8])}))
    return decline();
  if (lse->device() != k.dev || lse->scalar_type() != at::kFloat || lse->dim() != 2 || lse->size(0) != q.rows ||
      lse->size(1) != q.heads || !lse->is_contiguous())
    return decline();
  void* stream = PyLong_AsVoidPtr(a[12]);
  if (PyErr_Occurred()) return nullptr;
  HANDLE_TH_ERRORS
  const Call guard(k.dev);
  const int64_t wsb = mq_paged_attention_mass_workspace_size(&k.c, &m, q.rows, (int32_t)q.heads);
  if (wsb < 0) return status(MQ_INVALID_ARGUMENT);
  at::Tensor mass = at::empty({k.c.batch, k.c.kv_heads, k.c.width * k.c.page_size}, lse->options());
  at::Tensor ws;
  if (wsb) ws = at::empty({wsb}, lse->options().dtype(at::kByte));
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = mq_paged_attention_mass(&k.c, &m, q.t->const_data_ptr(), q.s_t, q.s_h, q.rows, (int32_t)q.heads,
                               lse->const_data_ptr<float>(), mass.mutable_data_ptr<float>(),
                               wsb ? ws.mutable_data_ptr() : nullptr, wsb, stream);
  Py_END_ALLOW_THREADS
  return rc == MQ_SUCCESS ? THPVariable_Wrap(std::move(mass)) : status(rc);
  END_HANDLE_TH_ERRORS
}

// (k, v, table, lens, mass, to, budget, recent, stream)
PyObject* paged_evict(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 9) return wrong_count("paged_evict: 9 arguments");
  Cache k;
  const at::Tensor *mass = plain(a[4]), *to = plain(a[5]);
  int64_t budget, recent;
  if (!mass || !to || !k.take(a[0], a[1], a[2], a[3], true) || !index_rows(*to, k.dev) || to->size(0) != k.c.batch ||
      to->size(1) < 1 || !as_int(a[6], &budget) || !as_int(a[7], &recent) || tracked({plain(a[0]), plain(a[1]), mass}))
    return decline();
  if (mass->device() != k.dev || mass->scalar_type() != at::kFloat || mass->dim() != 3 || mass->size(0) != k.c.batch ||
      mass->size(1) != k.c.kv_heads || mass->size(2) != k.c.width * k.c.page_size || mass->stride(2) != 1)
    return decline();
  if (budget < 1 || recent < 0 || recent > budget || budget > to->size(1) * (int64_t)k.c.page_size) return decline();
  void* stream = PyLong_AsVoidPtr(a[8]);
  if (PyErr_Occurred()) return nullptr;
  HANDLE_TH_ERRORS
  const Call guard(k.dev);
  const auto ints = mass->options().dtype(at::kInt);
  at::Tensor kept = at::empty({k.c.batch, k.c.kv_heads, budget}, ints), lens = at::empty({k.c.batch}, ints);
  at::Tensor left = at::empty({k.c.batch, k.c.kv_heads, to->size(1) * k.c.page_size}, mass->options());
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = mq_paged_evict(&k.c, mass->const_data_ptr<float>(), mass->stride(0), mass->stride(1), to->const_data_ptr<int32_t>(),
                      to->size(0) > 1 ? to->stride(0) : to->size(1), to->size(1), budget, recent,
                      kept.mutable_data_ptr<int32_t>(), lens.mutable_data_ptr<int32_t>(), left.mutable_data_ptr<float>(),
                      stream);
  Py_END_ALLOW_THREADS
  if (rc != MQ_SUCCESS) return status(rc);
  written(a[0]), written(a[1]);
  PyObject* o[3] = {THPVariable_Wrap(std::move(kept)), THPVariable_Wrap(std::move(lens)), THPVariable_Wrap(std::move(left))};
  PyObject* r = o[0] && o[1] && o[2] ? PyTuple_Pack(3, o[0], o[1], o[2]) : nullptr;
  for (PyObject* x : o) Py_XDECREF(x);
  return r;
  END_HANDLE_TH_ERRORS
}

}  // namespace mq_front
