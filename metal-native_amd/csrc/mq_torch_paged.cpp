// Native front of the paged-cache operators: checks, allocation and launch as
// one CPython call.  Every function returns None for what it does not take as
// it is (paged.py then names the fault, or copies and calls again), an int for
// a status of the library, else the outputs.  Function and dispatch modes (a
// default device is one) make no difference: nothing here is theirs to change,
// and the outputs are allocated below them.
#include "mq_torch.hpp"

#include <algorithm>
#include <utility>

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
// no two elements share memory: each stride reaches past all smaller dimensions
bool distinct(const at::Tensor& t) {
  if (t.dim() > 8) return false;
  std::pair<int64_t, int64_t> d[8];
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

  // l: dimensions in front of the pages'
  bool one(const at::Tensor& t, int l, int64_t* page, int64_t* head, int64_t* slot, bool write) const {
    if (t.dim() != l + 4 || t.stride(l + 3) != 1 || !aligned16(t)) return false;
    *page = t.size(l) > 1 ? t.stride(l) : 0;
    *head = t.size(l + 1) > 1 ? t.stride(l + 1) : 0;
    *slot = t.stride(l + 2);
    return *page % 8 == 0 && *head % 8 == 0 && *slot % 8 == 0 && *page >= 0 && *head >= 0 && *slot >= t.size(l + 3) &&
           (!write || distinct(t));
  }
  // v null: keys alone
  bool take(PyObject* ko, PyObject* vo, PyObject* table, PyObject* lens, bool write) {
    const at::Tensor* k = plain(ko);
    return take(k, vo ? plain(vo) : k, table, lens, write);
  }
  bool take(const at::Tensor* k, const at::Tensor* v, PyObject* table, PyObject* lens, bool write, int l = 0) {
    const at::Tensor *t = plain(table), *n = plain(lens);
    if (!k || !v || !t || !n) return false;
    dev = k->device();
    ty = k->scalar_type();
    if ((ty != at::kHalf && ty != at::kBFloat16) || v->scalar_type() != ty || v->device() != dev) return false;
    if (!one(*k, l, &c.k_page, &c.k_head, &c.k_slot, write) || !one(*v, l, &c.v_page, &c.v_head, &c.v_slot, write)) return false;
    if (k->sizes() != v->sizes() || !index_rows(*t, dev) || !vec(n, dev, at::kInt, t->size(0))) return false;
    if (t->size(0) < 1 || t->size(1) < 1 || k->numel() == 0) return false;
    if (k->size(l + 1) > INT32_MAX || k->size(l + 2) > INT32_MAX || k->size(l + 3) > INT32_MAX) return false;
    c.k = const_cast<void*>(k->const_data_ptr());
    c.v = const_cast<void*>(v->const_data_ptr());
    c.pages = k->size(l);
    c.kv_heads = (int32_t)k->size(l + 1);
    c.page_size = (int32_t)k->size(l + 2);
    c.head_dim = (int32_t)k->size(l + 3);
    c.dtype = ty == at::kHalf ? MQ_PAGED_F16 : MQ_PAGED_BF16;
    c.table = t->const_data_ptr<int32_t>();
    c.ld_table = t->size(0) > 1 ? t->stride(0) : t->size(1);
    c.width = t->size(1);
    c.batch = t->size(0);
    c.lens = n->const_data_ptr<int32_t>();
    return true;
  }
};

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

// a cache that the call wrote
void written(PyObject* o) {
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
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

// (parents, cu, words, stream)
PyObject* paged_ancestors(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 4) return wrong_count("paged_ancestors: 4 arguments");
  const at::Tensor *p = plain(a[0]), *cu = a[1] == Py_None ? nullptr : plain(a[1]);
  int64_t words;
  if (!p || p->dim() != 1 || !vec(p, p->device(), at::kInt, p->size(0)) || !as_int(a[2], &words) || words < 1 || words > INT32_MAX / 64)
    return decline();
  if (a[1] != Py_None && (!cu || cu->dim() != 1 || cu->size(0) < 2 || !vec(cu, p->device(), at::kInt, cu->size(0)))) return decline();
  const int64_t rows = p->size(0);
  void* stream = PyLong_AsVoidPtr(a[3]);
  if (PyErr_Occurred()) return nullptr;
  HANDLE_TH_ERRORS
  const Call guard(p->device());
  at::Tensor out = at::empty({rows, words}, p->options().dtype(at::kLong));
  if (rows == 0) return THPVariable_Wrap(std::move(out));
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = mq_paged_ancestors(p->const_data_ptr<int32_t>(), cu ? cu->const_data_ptr<int32_t>() : nullptr, cu ? cu->size(0) - 1 : rows,
                          rows, words, out.mutable_data_ptr<int64_t>(), stream);
  Py_END_ALLOW_THREADS
  return rc == MQ_SUCCESS ? THPVariable_Wrap(std::move(out)) : status(rc);
  END_HANDLE_TH_ERRORS
}

// (q, k, v, table, lens, tree, cu, scale, softcap, slopes, window, prefix_lens, max_q, return_lse, stream)
PyObject* paged_tree_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 15) return wrong_count("paged_tree_attention: 15 arguments");
  Cache k;
  Query q;
  mq_paged_mask m{};
  const at::Tensor* bits = plain(a[5]);
  if (!bits || !k.take(a[1], a[2], a[3], a[4], false) || !q.take(a[0], k) || !mask(a + 6, k, q, &m) ||
      tracked({q.t, plain(a[1]), plain(a[2]), plain(a[9])}))
    return decline();
  if (bits->device() != k.dev || bits->scalar_type() != at::kLong || bits->dim() != 2 || bits->size(0) != q.rows || bits->size(1) < 1 ||
      bits->size(1) > INT32_MAX / 64 || (bits->size(1) > 1 && bits->stride(1) != 1) || bits->stride(0) < 0)
    return decline();
  const int want_lse = PyObject_IsTrue(a[13]);
  if (want_lse < 0) return nullptr;
  void* stream = PyLong_AsVoidPtr(a[14]);
  if (PyErr_Occurred()) return nullptr;
  HANDLE_TH_ERRORS
  const Call guard(k.dev);
  const int64_t wsb = mq_paged_tree_attention_workspace_size(&k.c, &m, q.rows, (int32_t)q.heads);
  if (wsb < 0) return status(MQ_INVALID_ARGUMENT);
  at::Tensor out = at::empty({q.rows, q.heads, q.t->size(2)}, q.t->options());
  at::Tensor lse, ws;
  if (want_lse) lse = at::empty({q.rows, q.heads}, q.t->options().dtype(at::kFloat));
  if (wsb) ws = at::empty({wsb}, q.t->options().dtype(at::kByte));
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = mq_paged_tree_attention(&k.c, &m, bits->const_data_ptr<int64_t>(), bits->stride(0), bits->size(1), q.t->const_data_ptr(), q.s_t,
                               q.s_h, q.rows, (int32_t)q.heads, out.mutable_data_ptr(),
                               want_lse ? lse.mutable_data_ptr<float>() : nullptr, wsb ? ws.mutable_data_ptr() : nullptr, wsb, stream);
  Py_END_ALLOW_THREADS
  if (rc != MQ_SUCCESS) return status(rc);
  return want_lse ? packed({out, lse}) : THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// (k, v, table, lens, drawn, drafted, parents, cu, steps, stream); k and v with or without a dimension of layers
PyObject* paged_accept(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 10) return wrong_count("paged_accept: 10 arguments");
  Cache k;
  const at::Tensor *kt = plain(a[0]), *vt = plain(a[1]), *drawn = plain(a[4]), *drafted = plain(a[5]), *parents = plain(a[6]);
  int64_t steps;
  if (!kt || !vt || !drawn || drawn->dim() != 1 || !as_int(a[8], &steps) || steps < 1 || steps > INT32_MAX - 64 || tracked({kt, vt}))
    return decline();
  const int64_t rows = drawn->size(0);
  const int32_t* cu;
  int64_t layers = 1, kl = 0, vl = 0;
  void* stream = PyLong_AsVoidPtr(a[9]);
  if (PyErr_Occurred()) return nullptr;
  HANDLE_TH_ERRORS
  const Call guard(kt->device());
  const bool deep = kt->dim() == 5;
  if (!k.take(kt, vt, a[2], a[3], true, deep) || kt->const_data_ptr() == vt->const_data_ptr()) return decline();
  if (deep && kt->size(0) > 1) {
    layers = kt->size(0);
    kl = kt->stride(0);
    vl = vt->stride(0);
    if (kl % 8 || vl % 8 || kl < 0 || vl < 0) return decline();
  }
  if (!vec(drawn, k.dev, at::kLong, rows) || !vec(drafted, k.dev, at::kLong, rows) || !vec(parents, k.dev, at::kInt, rows) ||
      !chunks(a[7], k, rows, &cu))
    return decline();
  const auto ints = drawn->options().dtype(at::kInt);
  at::Tensor path = at::empty({k.c.batch, steps}, ints), tokens = at::empty({k.c.batch, steps}, drawn->options());
  at::Tensor count = at::empty({k.c.batch}, ints), lens = at::empty({k.c.batch}, ints);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = mq_paged_accept(&k.c, layers, kl, vl, drawn->const_data_ptr<int64_t>(), drafted->const_data_ptr<int64_t>(),
                       parents->const_data_ptr<int32_t>(), cu, rows, steps, path.mutable_data_ptr<int32_t>(),
                       tokens.mutable_data_ptr<int64_t>(), count.mutable_data_ptr<int32_t>(), lens.mutable_data_ptr<int32_t>(), stream);
  Py_END_ALLOW_THREADS
  if (rc != MQ_SUCCESS) return status(rc);
  written(a[0]), written(a[1]);
  return packed({path, tokens, count, lens});
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
