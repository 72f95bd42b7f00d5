// lm_norm_bf16.hip -- the residual norms' row kernels for bf16 rows.
#include "lm_norm_kernel.h"

namespace lm {
template hipError_t norm_run<DT_BF16>(const NormArgs &, const NormSplit &, bool, bool, hipStream_t);
}
