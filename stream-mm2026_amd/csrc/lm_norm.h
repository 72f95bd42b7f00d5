// lm_norm.h -- launches of the residual-norm kernels (lm_norm.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace lm {

constexpr int NORM_MIN_DIM = 8, NORM_MAX_DIM = 8192;

struct NormArgs {
    int64_t n, dim;
    int dt;                        // of x, block, r, h and their gradients
    int weight_dt;                 // of the weights, biases, gates and their gradients
    const void *x, *block;         // [n, dim], rows x_stride / block_stride elements apart
    int64_t x_stride, block_stride;
    const void *pre_weight, *pre_bias, *post_weight, *post_bias;   // [dim]; pre_weight always, a bias or null, post_weight or null
    const void *gate;              // [groups, dim] dense or null; row i takes gate[i / (n / groups)]
    int64_t groups;
    float residual_scale, eps;
    int layer;                     // 0: RMS norms, 1: layer norms
    float *stats;                  // [n, 4]: mean and 1/deviation of block, of r
    void *r, *h;                   // forward: [n, dim] dense
    // backward
    const void *dr, *dh;           // dr may be null (zeros); rows dr_stride / dh_stride apart
    int64_t dr_stride, dh_stride;
    void *dx, *dblock;             // [n, dim] dense
    void *dpre_weight, *dpre_bias, *dpost_weight, *dpost_bias, *dgate;   // null where the operand is
    float *workspace;
};

// How the rows are shared out.  `waves` a row (1 and 2: several rows of a workgroup of four waves;
// more: a workgroup's).  Backward: with few groups of gates `per_group` workgroups to a group, with
// many (per_group 0) each row's threads take whole groups.
struct NormSplit {
    int wgs, per_group, waves, fwd_wgs;
};

// The row kernels of one element type, with weights of that type or fp32 (lm_norm_*.hip).
template <int DT, bool WF32>
hipError_t norm_run(const NormArgs &a, const NormSplit &sp, bool ragged, bool backward, hipStream_t stream);

hipError_t norm_forward(const NormArgs &a, hipStream_t stream);
int64_t norm_backward_workspace(int64_t n, int64_t dim, int64_t groups);
hipError_t norm_backward(const NormArgs &a, hipStream_t stream);

}  // namespace lm
