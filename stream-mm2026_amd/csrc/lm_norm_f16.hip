// lm_norm_f16.hip -- the residual norms' row kernels for f16 rows and weights.
#include "lm_norm_kernel.h"

namespace lm {
template hipError_t norm_run<DT_F16, false>(const NormArgs &, const NormSplit &, bool, bool, hipStream_t);
}
