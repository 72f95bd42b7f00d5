// lm_clip.h -- launches of the gradient norm and clipping kernels (lm_clip.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace lm {

struct ClipTensor {
    const void *grad;
    void *out;                           // null where only the norm is asked for; may be grad
    int64_t numel;
    int dt;
};

// Elements of a tensor at most.
constexpr int64_t CLIP_MAX_NUMEL = (int64_t)1 << 36;
// The workspace in bytes: a double for each workgroup that adds squares.
int64_t clip_workspace(int64_t count);
// norm = sqrt(sum of all squares) into *norm (a float on the device); workspace as above.
hipError_t clip_norm(const ClipTensor *t, int64_t count, double *partial, float *norm, hipStream_t stream);
// out = grad min(1, max_norm / (norm + 1e-6)), the norm computed and written, or where `given` read from there.
hipError_t clip_scale(const ClipTensor *t, int64_t count, double max_norm, const float *given, double *partial, float *norm, hipStream_t stream);

}  // namespace lm
