// Attention of trees of drafted tokens over a paged cache: the kernels of
// mq_pattn_dev.hpp for chunks whose rows see what their ancestor bits say.
#include "mq_pattn_dev.hpp"

namespace mq {

PagedPlan ptattn_plan(const PagedArgs& a, int num_cus) {
  if (many_rows(a)) return {kRowsP, rows_plan(a, num_cus).parts};
  return {kRowsS, split_plan(a, num_cus).parts};
}

size_t ptattn_workspace(const PagedArgs& a, int num_cus) {
  return many_rows(a) ? rows_plan(a, num_cus).ws_bytes : split_plan(a, num_cus).ws_bytes;
}

hipError_t ptattn_launch(const PagedArgs& a, int num_cus, void* ws, hipStream_t s) { return launch<true>(a, num_cus, ws, s); }

}  // namespace mq
