// Attention of new tokens over a paged cache: the kernels of mq_pattn_dev.hpp for
// chunks whose tokens stand in order.
#include "mq_pattn_dev.hpp"

namespace mq {

PagedPlan pattn_plan(const PagedArgs& a, int num_cus) {
  if (many_rows(a)) return {kRowsP, rows_plan(a, num_cus).parts};
  return {kRowsS, split_plan(a, num_cus).parts};
}

size_t pattn_workspace(const PagedArgs& a, int num_cus) {
  return many_rows(a) ? rows_plan(a, num_cus).ws_bytes : split_plan(a, num_cus).ws_bytes;
}

hipError_t pattn_launch(const PagedArgs& a, int num_cus, void* ws, hipStream_t s) { return launch<false>(a, num_cus, ws, s); }

}  // namespace mq
