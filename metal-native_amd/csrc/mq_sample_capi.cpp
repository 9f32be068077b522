// C entries that draw tokens from logits: argument checks and launch.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstdio>

#include "../../include/metal_native_amd.h"
#include "mq_sample.hpp"

namespace {

int refuse(const char* what) {
  char msg[256];
  std::snprintf(msg, sizeof msg, "sampling.sample: %s", what);
  return mq::fail_with(MQ_INVALID_ARGUMENT, msg);
}

// null, or what is wrong
const char* sample_args(mq::SampleArgs& a, int64_t rows, int64_t vocab, int32_t dtype, const mq_sampling* how) {
  if (!how) return "null settings";
  if (dtype != MQ_SAMPLE_F16 && dtype != MQ_SAMPLE_BF16 && dtype != MQ_SAMPLE_F32) return "unknown dtype";
  if (rows < 0 || rows > INT_MAX || vocab < 1 || vocab > 1 << 22) return "rows must be below 2^31, the vocabulary 1 to 2^22";
  a = mq::SampleArgs{};
  a.rows = (int)rows;
  a.vocab = (int)vocab;
  a.dtype = dtype;
  a.temperatures = how->temperatures;
  a.top_ps = how->top_ps;
  a.min_ps = how->min_ps;
  a.top_ks = how->top_ks;
  a.temperature = how->temperature;
  a.top_p = how->top_p;
  a.min_p = how->min_p;
  a.top_k = how->top_k;
  return nullptr;
}

}  // namespace

extern "C" {

MQ_API int64_t mq_sample_workspace_size(int64_t rows, int64_t vocab, int32_t dtype, const mq_sampling* how) {
  mq::SampleArgs a;
  if (const char* bad = sample_args(a, rows, vocab, dtype, how)) {
    refuse(bad);
    return -1;
  }
  return (int64_t)mq::sample_workspace(a, mq::current_num_cus());
}

MQ_API int mq_sample(const void* logits, int64_t ld, int64_t rows, int64_t vocab, int32_t dtype, const float* u,
                     const mq_sampling* how, int64_t* token, float* logprob, void* ws, int64_t ws_bytes, void* stream) {
  mq::SampleArgs a;
  if (const char* bad = sample_args(a, rows, vocab, dtype, how)) return refuse(bad);
  if (rows == 0) return MQ_SUCCESS;
  if (!logits || !u || !token) return refuse("null pointer argument");
  const uintptr_t size = dtype == MQ_SAMPLE_F32 ? 4 : 2;
  if ((uintptr_t)logits % size || ld < 0 || ld > LLONG_MAX / 8 / rows) return refuse("logits misaligned, or their row stride out of range");
  a.logits = logits;
  a.ld = ld;
  a.u = u;
  a.token = token;
  a.logprob = logprob;
  const int cus = mq::current_num_cus();
  const size_t need = mq::sample_workspace(a, cus);
  if (need && (!ws || ((uintptr_t)ws & 15) || ws_bytes < (int64_t)need)) return refuse("workspace too small or not 16-byte aligned");
  const hipError_t e = mq::sample_launch(a, cus, ws, (hipStream_t)stream);
  return e == hipSuccess ? MQ_SUCCESS : mq::hip_fail_with(e, "sampling.sample: kernel launch failed");
}

}  // extern "C"
