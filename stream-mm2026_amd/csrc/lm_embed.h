// lm_embed.h -- launches of the embedding kernels (lm_embed.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace lm {

struct EmbedArgs {
    const void *tokens;      // int64 or int32 [n]
    int token_bytes;
    int64_t n;
    int64_t vocab, dim;
    float scale;
};

// out[i] = scale * weight[tokens[i]]; rows of the table `weight_stride` elements apart.
hipError_t embed_forward(const EmbedArgs &a, const void *weight, int weight_dt, int64_t weight_stride, void *out, int out_dt,
                         hipStream_t stream);

// The gradient's kernels count tokens and rows in 32 bits and step past the last of them by up to a grid's surplus
// (2^21 tokens, 512 rows), so that both stay below 2^31 up to here.
constexpr int64_t EMBED_GRAD_MAX = 1 << 30;
// Bytes of workspace that embed_backward needs.
int64_t embed_backward_workspace(int64_t n, int64_t vocab, int64_t dim);

// dweight[v] (+)= scale * sum of grad[i] over tokens[i] == v, in the order of i; token `padding`
// (negative: none) takes none.  Every row is written, or with `accumulate` only those of tokens.
hipError_t embed_backward(const EmbedArgs &a, const void *grad, int grad_dt, int64_t grad_stride, void *dweight, int dweight_dt,
                          int64_t dweight_stride, int64_t padding, bool accumulate, void *workspace, hipStream_t stream);

}  // namespace lm
