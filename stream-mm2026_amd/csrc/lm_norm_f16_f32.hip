// lm_norm_f16_f32.hip -- the residual norms' row kernels for f16 rows and fp32 weights.
#include "lm_norm_kernel.h"

namespace lm {
template hipError_t norm_run<DT_F16, true>(const NormArgs &, const NormSplit &, bool, bool, hipStream_t);
}
