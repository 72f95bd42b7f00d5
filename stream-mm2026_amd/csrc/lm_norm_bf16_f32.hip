// lm_norm_bf16_f32.hip -- the residual norms' row kernels for bf16 rows and fp32 weights.
#include "lm_norm_kernel.h"

namespace lm {
template hipError_t norm_run<DT_BF16, true>(const NormArgs &, const NormSplit &, bool, bool, hipStream_t);
}
