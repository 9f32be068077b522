// Attention of trees of drafted tokens over a paged cache: the kernels of
// mq_pattn_dev.hpp for chunks whose rows see what their ancestor bits say.
//
// Only the newest slots differ by row, so a tile in front of the chunk costs what it
// does for chunks in order; of the chunk's own tiles a row's 64 bits are two words, read
// where they are needed.  Beside `attention` of the same shapes (us): 16 nodes behind 512
// slots 14.8 and 14.6, 24 trees of 4 to 26 behind 200 to 8000 slots 88 and 86 (memory:
// 255 MB, a floor of 50; the longest sequence's parts end the call), 4 of 64 behind 90 to
// 131 thousand 494 (0.87 PFLOP/s, the matrix units).  With a window or a bias a row counts
// bits for its distances: 5 trees of 60 to 257 nodes, cap, bias, window and prefix, 43 and 35.
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
