// Drawing tokens from logits: arguments (mq_sample.hip).
#pragma once
#include "mq_launch.hpp"

namespace mq {

struct SampleArgs {
  const void* logits;   // [rows, vocab], row stride ld elements
  int64_t ld;
  int rows, vocab, dtype;   // enum mq_sample_dtype
  const float* u;           // [rows]
  // a setting is the array's value of the row, or where there is none the number
  const float *temperatures, *top_ps, *min_ps;
  const int32_t* top_ks;
  float temperature, top_p, min_p;
  int32_t top_k;
  int64_t* token;
  float* logprob;   // or null
};
size_t sample_workspace(const SampleArgs& a, int num_cus);
hipError_t sample_launch(const SampleArgs& a, int num_cus, void* ws, hipStream_t s);

}  // namespace mq
