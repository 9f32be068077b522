// Attention of trees of drafted tokens over a paged cache: the kernels of
// mq_pattn_dev.hpp for chunks whose rows see what their ancestor bits say.
//
// Only the newest slots differ by row, so a tile in front of the chunk costs what it
// does for chunks in order; of the chunk's own tiles a row's 64 bits are two words, read
// where they are needed.  Beside `attention` of the same shapes, called in turn (us): 16
// nodes behind 512 slots 14.6 and 14.3, 24 trees of 4 to 26 behind 200 to 8000 slots 83
// and 81 (memory: 255 MB, a floor of 50; the longest sequence's parts end the call), 4 of
// 64 behind 90 to 131 thousand 491 and 493 (0.87 PFLOP/s, the matrix units), 5 of 60 to
// 257, 64 wide, cap, bias, window and prefix, 42.5 and 33.1, as many 128 wide with a cap
// 112 and 100.  With a window or a bias a row counts bits for its distances, and what it
// keeps of its bits takes registers in the main loop.  Registers in memory, in order and
// here: blocks of 256 rows, 128 wide, 6 and 12, with cap or bias 8 and 98, 64 wide with cap
// or bias 0 and 6; blocks of 32, 128 wide with cap or bias, 9 and 32.  Blocks of 32, 64
// wide, have 162 and 169 (cap or bias 166 and 189): three waves on a SIMD and two.
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
