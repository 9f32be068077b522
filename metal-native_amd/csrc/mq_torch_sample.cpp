// Native front of sampling.sample: checks, allocation and launch as one CPython
// call, in the manner of mq_torch_paged.cpp.
#include "mq_torch.hpp"

#include <torch/csrc/Exceptions.h>

#include "../../include/metal_native_amd.h"

namespace mq_front {
namespace {

// One number, or a tensor with one for each row.
bool setting(PyObject* o, const at::Tensor& x, float* one, const float** each) {
  if (as_float(o, one)) return true;
  const at::Tensor* t = plain(o);
  if (!vec(t, x.device(), at::kFloat, x.size(0))) return false;
  *each = t->const_data_ptr<float>();
  return true;
}

}  // namespace

// (logits, u, temperature, top_k, top_p, min_p, return_logprob, stream)
PyObject* sample(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 8) return wrong_count("sample: 8 arguments");
  const at::Tensor *x = plain(a[0]), *u = plain(a[1]);
  if (!x || x->dim() != 2 || x->size(1) < 1 || x->size(1) > 1 << 22 || (x->size(1) > 1 && x->stride(1) != 1) || x->stride(0) < 0) return decline();
  const at::ScalarType ty = x->scalar_type();
  if ((ty != at::kHalf && ty != at::kBFloat16 && ty != at::kFloat) || !vec(u, x->device(), at::kFloat, x->size(0))) return decline();
  mq_sampling how{};
  if (!setting(a[2], *x, &how.temperature, &how.temperatures) || !setting(a[4], *x, &how.top_p, &how.top_ps) ||
      !setting(a[5], *x, &how.min_p, &how.min_ps))
    return decline();
  int64_t k;
  const at::Tensor* ks = nullptr;
  if (as_int(a[3], &k)) {
    how.top_k = (int32_t)(k < 0 ? 0 : (k > INT32_MAX ? INT32_MAX : k));
  } else {
    ks = plain(a[3]);
    if (!vec(ks, x->device(), at::kInt, x->size(0))) return decline();
    how.top_ks = ks->const_data_ptr<int32_t>();
  }
  const at::Tensor *t0 = how.temperatures ? plain(a[2]) : nullptr, *t1 = how.top_ps ? plain(a[4]) : nullptr, *t2 = how.min_ps ? plain(a[5]) : nullptr;
  if (tracked({x, u, t0, t1, t2})) return decline();
  const int want = PyObject_IsTrue(a[6]);
  if (want < 0) return nullptr;
  void* stream = PyLong_AsVoidPtr(a[7]);
  if (PyErr_Occurred()) return nullptr;
  HANDLE_TH_ERRORS
  const Call guard(x->device());
  const int64_t rows = x->size(0), vocab = x->size(1);
  const int32_t dtype = ty == at::kHalf ? MQ_SAMPLE_F16 : (ty == at::kBFloat16 ? MQ_SAMPLE_BF16 : MQ_SAMPLE_F32);
  const int64_t wsb = mq_sample_workspace_size(rows, vocab, dtype, &how);
  if (wsb < 0) return status(MQ_INVALID_ARGUMENT);
  at::Tensor token = at::empty({rows}, x->options().dtype(at::kLong)), logprob, ws;
  if (want) logprob = at::empty({rows}, x->options().dtype(at::kFloat));
  if (wsb) ws = at::empty({wsb}, x->options().dtype(at::kByte));
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = mq_sample(x->const_data_ptr(), rows > 1 ? x->stride(0) : vocab, rows, vocab, dtype, u->const_data_ptr<float>(), &how,
                 token.mutable_data_ptr<int64_t>(), want ? logprob.mutable_data_ptr<float>() : nullptr,
                 wsb ? ws.mutable_data_ptr() : nullptr, wsb, stream);
  Py_END_ALLOW_THREADS
  if (rc != MQ_SUCCESS) return status(rc);
  return want ? packed({token, logprob}) : THPVariable_Wrap(std::move(token));
  END_HANDLE_TH_ERRORS
}

}  // namespace mq_front
