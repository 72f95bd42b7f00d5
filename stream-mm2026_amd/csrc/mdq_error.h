// mdq_error.h -- the C entry points' error reports (stq_last_error()).
#pragma once
#include <hip/hip_runtime.h>

namespace mdq {

// Keeps the message for stq_last_error() on this thread and returns `code`.
int fail(int code, const char *fmt, ...);
int hip_fail(hipError_t e, const char *what);
const char *dtype_name(int dt);

}  // namespace mdq
