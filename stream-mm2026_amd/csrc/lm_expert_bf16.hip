// lm_expert_bf16.hip -- the experts' products for bf16.
#include "lm_expert_kernel.h"

namespace lm {
template hipError_t product_forward<DT_BF16>(const ProductArgs &, hipStream_t);
template hipError_t product_backward<DT_BF16>(const ProductArgs &, hipStream_t);
}
