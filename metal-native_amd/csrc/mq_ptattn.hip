// Attention of trees of drafted tokens over a paged cache: the kernels of
// mq_pattn_dev.hpp for chunks whose rows see what their ancestor bits say.
#include "mq_pattn_dev.hpp"

namespace mq {

hipError_t ptattn_launch(const PagedArgs& a, int num_cus, void* ws, hipStream_t s) { return launch<true>(a, num_cus, ws, s); }

}  // namespace mq
