// lm_attn_bf16.hip -- the attention kernels for bf16.
#include "lm_attn_kernel.h"

namespace lm {
template hipError_t attn_forward<DT_BF16>(const AttnArgs &, hipStream_t);
template hipError_t attn_backward<DT_BF16>(const AttnArgs &, hipStream_t);
}
