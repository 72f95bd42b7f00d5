// lm_attn_f16.hip -- the attention kernels for f16.
#include "lm_attn_kernel.h"

namespace lm {
template hipError_t attn_forward<DT_F16>(const AttnArgs &, hipStream_t);
template hipError_t attn_backward<DT_F16>(const AttnArgs &, hipStream_t);
}
