// lm_expert_f16.hip -- the experts' products for fp16.
#include "lm_expert_kernel.h"

namespace lm {
template hipError_t product_forward<DT_F16>(const ProductArgs &, hipStream_t);
template hipError_t product_backward<DT_F16>(const ProductArgs &, hipStream_t);
}
