// lm_norm_bf16.hip -- the residual norms' row kernels for bf16 rows and weights.
#include "lm_norm_kernel.h"

namespace lm {
template hipError_t norm_run<DT_BF16, false>(const NormArgs &, const NormSplit &, bool, bool, hipStream_t);
}
