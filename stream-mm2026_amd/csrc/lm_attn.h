// lm_attn.h -- launches of the attention kernels (lm_attn_kernel.h, lm_attn_bf16.hip, lm_attn_f16.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace lm {

// A [batch, heads, positions, dim] array: elements between batches, heads and positions; dim is dense.
struct AttnTensor {
    void *p;
    int64_t b, h, t;
};

struct AttnArgs {
    AttnTensor q, k, v, o, dout, dq, dk, dv;
    const uint8_t *key_mask;       // [batch, keys] (0: hidden), rows mask_stride apart, or null
    int64_t mask_stride;
    float *lse;                    // [batch, heads, rows]: log sum exp of the scaled scores
    float *delta;                  // backward's workspace, as lse: rowsum(dout * out)
    float *partial;                // forward's workspace where the keys are split
    int batch, heads, key_heads, group;   // heads = key_heads * group
    int rows, keys, dim;           // row i stands at position keys - rows + i
    int window, sinks;             // row at p sees key j <= p if p - j < window or j < sinks
    float scale;
    int splits;
};

template <int DT>
hipError_t attn_forward(const AttnArgs &a, hipStream_t stream);
template <int DT>
hipError_t attn_backward(const AttnArgs &a, hipStream_t stream);

// How many parts the keys are split into where there are few rows, and the floats of workspace that takes.
constexpr int MAX_SPLITS = 512;
int attn_splits(const AttnArgs &a);
int64_t attn_forward_workspace(const AttnArgs &a);

// Where the work on the keys' gradients is cut: blocks of 128 keys, and either (few blocks) the walk of
// each over its positions in `shares` parts, or (sinks) for the first `sink_blocks` of them `far` more
// workgroups of `step` positions each, which lie behind the window of the block's keys.
struct DkvSplit {
    int blocks, sink_blocks, far, step, shares;
    __host__ __device__ int parts() const { return shares > 1 ? shares : far + 1; }
    // the keys whose gradients come in parts
    __host__ __device__ int keys(const AttnArgs &a) const { return shares > 1 ? a.keys : far ? a.sinks : 0; }
    // the partial sums of part f: dk and dv of those keys
    __host__ __device__ float *sums(const AttnArgs &a, int head, int f) const
    {
        return a.partial + ((int64_t)head * parts() + f) * 2 * keys(a) * a.dim;
    }
};
DkvSplit dkv_split(const AttnArgs &a);
// The floats of workspace: delta, then the partial sums.
int64_t attn_backward_delta(const AttnArgs &a);
int64_t attn_backward_workspace(const AttnArgs &a);

}  // namespace lm
