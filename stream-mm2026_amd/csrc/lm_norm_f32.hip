// lm_norm_f32.hip -- the residual norms' row kernels for f32 rows.
#include "lm_norm_kernel.h"

namespace lm {
template hipError_t norm_run<DT_F32, true>(const NormArgs &, const NormSplit &, bool, bool, hipStream_t);
}
