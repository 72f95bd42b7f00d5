// lm_expert.hip -- the workspace of the experts' products (the kernels: lm_expert_kernel.h).
#include "lm_expert.h"

namespace lm {

// Gathered rows: dx of the sorted rows in fp32, which their tokens' sums are formed from.
int64_t product_workspace(const ProductArgs &a) { return a.k && a.dx ? a.slots * a.in * 4 : 0; }

}  // namespace lm
