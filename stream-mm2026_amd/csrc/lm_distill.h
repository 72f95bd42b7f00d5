// lm_distill.h -- launches of the distillation loss kernels (lm_distill.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace lm {

constexpr int DISTILL_MAX_K = 1024;

struct DistillArgs {
    const void *logits;          // [n, vocab], rows `stride` elements apart
    int dt;
    int64_t n, vocab, stride;
    const void *teacher;         // [n, k] dense
    int teacher_dt;
    const void *ids;             // [n, k] dense, int64 or int32
    int id_bytes;
    int k;
    const void *labels;          // [n] or null
    int label_bytes;
    float temperature, alpha;
    float *loss;                 // [n], or null
    float *stats;                // [n, 4] or null: max, log sum exp((z - max) / T), log sum exp(z - max), unused
    const float *drow;           // [n]: the gradient of each row's loss (read where dlogits is written)
    void *dlogits;               // [n, vocab] or null; may be the logits themselves
    int64_t dstride;
};

// The loss alone, or the loss and its gradient from one read of the logits.
hipError_t distill_forward(const DistillArgs &a, hipStream_t stream);
// The gradient from the stats of an earlier forward call.
hipError_t distill_backward(const DistillArgs &a, hipStream_t stream);

}  // namespace lm
