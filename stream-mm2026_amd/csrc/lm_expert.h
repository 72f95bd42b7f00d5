// lm_expert.h -- launches of the routing, planning and combining kernels (lm_route.hip) and of the experts' products
// (lm_expert_kernel.h, lm_expert_bf16.hip, lm_expert_f16.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace lm {

constexpr int EXPERT_MAX = 512;          // experts: a plan's histograms lie in LDS
constexpr int ROUTE_MAX_K = 64;          // experts a row may choose
constexpr int64_t SLOT_MAX = 1 << 30;

struct RouteArgs {
    const void *logits;                  // [n, experts], rows `stride` elements apart
    int dt;
    int64_t n, stride;
    int experts, k, renormalize;
    float *weights;                      // [n, k]
    int32_t *ids;                        // [n, k]
    float *load;                         // [experts] or null
    float *partial;                      // workspace: the workgroups' sums of probabilities
    const float *dweights, *dload;       // [n, k], [experts]; either may be null
    void *dlogits;
    int64_t dstride;
};
int64_t route_workspace(int64_t n, int experts);
hipError_t route_forward(const RouteArgs &a, hipStream_t stream);
hipError_t route_backward(const RouteArgs &a, hipStream_t stream);

struct PlanArgs {
    const void *ids;                     // [slots], int64 or int32
    int id_bytes;
    int64_t slots;
    int experts;
    int32_t *rows, *places, *offsets;
    int32_t *hist;                       // workspace
};
int64_t plan_workspace(int64_t slots, int experts);
hipError_t expert_plan(const PlanArgs &a, hipStream_t stream);

struct CombineArgs {
    int64_t n;
    int k, experts;
    int64_t dim;
    const void *y;                       // [n k, dim], rows y_stride apart
    int y_dt;
    int64_t y_stride;
    const float *weights;                // [n, k] or null: ones
    const int32_t *places, *offsets;
    void *out;                           // [n, dim], rows out_stride apart, y's type or 16 bits of fp32 rows
    int out_dt;
    int64_t out_stride;
    const void *dout;                    // backward: y's type
    int64_t dout_stride;
    void *dy;                            // [n k, dim] dense
    float *dweights;                     // [n, k] or null
};
hipError_t combine_forward(const CombineArgs &a, hipStream_t stream);
hipError_t combine_backward(const CombineArgs &a, hipStream_t stream);

struct ProductArgs {
    int64_t slots;
    int experts, in, out;
    int k;                               // > 0: row r is token rows[r] / k of x (and of dx), 0: row r of x
    uint32_t k_inverse;                  // (2^32 - 1) / k
    int64_t tokens;                      // k > 0: rows of x
    const void *x;
    int64_t x_stride;
    const void *weight;                  // [experts, out, in], 16-bit
    int64_t weight_expert_stride, weight_row_stride;
    void *y;                             // [slots, out] dense
    const int32_t *rows, *places, *offsets;
    const void *dy;                      // [slots, out]
    int64_t dy_stride;
    void *dx;                            // [slots, in] (k > 0: [tokens, in]) dense, or null
    float *scratch;                      // k > 0, where dx is wanted: [slots, in]
    void *dweight;                       // [experts, out, in] dense, or null
    int dweight_f32;
};
int64_t product_workspace(const ProductArgs &a);
template <int DT>
hipError_t product_forward(const ProductArgs &a, hipStream_t stream);
template <int DT>
hipError_t product_backward(const ProductArgs &a, hipStream_t stream);

}  // namespace lm
