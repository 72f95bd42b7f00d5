/*
 * stquant_lm.h -- C ABI of the transformer operators of libstquant_hip.so: embedding lookup,
 * residual norms, windowed attention, the distillation loss, routing to experts, their products and
 * the products' combination, each with its gradient, and the clipping of gradients to a global norm.
 *
 * Every call takes one argument struct (read before the call returns) and a hipStream_t, queues
 * its kernels on that stream and returns; nothing is allocated, copied or kept, so calls can be
 * captured into a HIP graph.  Workspaces belong to the caller and are free again once the stream
 * has passed the call.  Device pointers address memory of the current HIP device, aligned to their
 * element size; sizes and strides count elements.  Element types are stq_dtype codes
 * (stquant_hip.h).  Return values and stq_last_error() are those of stquant_hip.h; argument errors
 * are reported before anything is queued.  Results do not depend on the order in which workgroups
 * run: the same call gives the same bits.
 */
#ifndef STQUANT_LM_H
#define STQUANT_LM_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Of the structs below and what their calls mean; added structs and entries leave it as it is.  (2 was the same as 1
 * with more entries: the next is 3.) */
#define STQ_LM_ABI_VERSION 1

/*
 * out[i, :] = scale * weight[tokens[i], :]; a token outside [0, vocab) gives a row of NaN.
 * weight: Float, BFloat16 or Half, rows weight_stride apart; out: [n, dim] dense, any of the three.
 * n and vocab < 2^31, dim up to 2^24.
 */
typedef struct stq_embedding {
    const void *tokens; /* [n], token_dtype STQ_LONG or STQ_INT */
    int64_t token_dtype, n, vocab, dim;
    const void *weight;
    int64_t weight_dtype, weight_stride;
    void *out;
    int64_t out_dtype;
    double scale; /* rounded to float */
} stq_embedding;

int stq_embedding_forward(const stq_embedding *a, void *stream);

/*
 * dweight[v, :] = scale * sum of grad[i, :] over tokens[i] == v, added in the order of i in fp32;
 * tokens outside [0, vocab) and `padding` (negative: none) add nothing.  accumulate: added to what
 * dweight holds (rows of no token are then left alone); otherwise every row is written.
 * n and vocab up to 2^30.  workspace: stq_embedding_grad_workspace(a) bytes, 16-byte aligned.
 */
typedef struct stq_embedding_grad {
    const void *tokens;
    int64_t token_dtype, n, vocab, dim;
    const void *grad;
    int64_t grad_dtype, grad_stride;
    void *dweight;
    int64_t dweight_dtype, dweight_stride;
    int64_t padding, accumulate;
    void *workspace;
    int64_t workspace_bytes;
    double scale;
} stq_embedding_grad;

int64_t stq_embedding_grad_workspace(const stq_embedding_grad *a);
int stq_embedding_backward(const stq_embedding_grad *a, void *stream);

/*
 * n1 = norm(block; post_weight, post_bias), or block where post_weight is null
 * r  = residual_scale * x + gate * n1      (gate null: 1)
 * h  = norm(r; pre_weight, pre_bias)       r and h rounded once, h from the unrounded r
 * norm(y; w, c) = (y - mean) / sqrt(mean((y - mean)^2) + eps) * w + c; layer = 0: no mean is taken off,
 * and there are no biases.
 * Rows of `dim` elements, 8 <= dim <= 8192; x, block, dr, dh strided, the others dense.  gate:
 * [groups, dim], row i takes gate[i / (n / groups)], groups divides n (0: up to 2^30 of them).
 * weight_dtype: Float or dtype.
 * stats: [n, 4] floats that the forward call writes and the backward call reads.
 */
typedef struct stq_norm_residual {
    int64_t n, dim, dtype, weight_dtype;
    const void *x, *block;
    int64_t x_stride, block_stride;
    const void *pre_weight, *pre_bias, *post_weight, *post_bias, *gate;
    int64_t groups, layer;
    double residual_scale, eps;
    float *stats;
    void *r, *h;
    /* backward: dr may be null (zeros); a gradient is null exactly where its operand is */
    const void *dr, *dh;
    int64_t dr_stride, dh_stride;
    void *dx, *dblock, *dpre_weight, *dpre_bias, *dpost_weight, *dpost_bias, *dgate;
    void *workspace;
    int64_t workspace_bytes;
} stq_norm_residual;

int64_t stq_norm_residual_workspace(const stq_norm_residual *a);
int stq_norm_residual_forward(const stq_norm_residual *a, void *stream);
int stq_norm_residual_backward(const stq_norm_residual *a, void *stream);

/* A [batch, heads, positions, dim] array: strides between batches, heads, positions; dim dense. */
typedef struct stq_tensor4 {
    void *p;
    int64_t batch_stride, head_stride, row_stride;
} stq_tensor4;

/*
 * Causal attention of `rows` positions, the last ones of `keys`: row i stands at p = keys - rows + i
 * and sees key j <= p if p - j < window (window 0: no limit) or j < sinks, and key_mask[batch, j] is
 * nonzero.  A row that sees nothing gives zeros, and zero gradients; what masked keys hold does not
 * matter.  BFloat16 or Half; dim a multiple of 8 up to 128; heads a multiple of key_heads, consecutive
 * heads sharing one; scale 1e-30 to 1e30.  Pointers are 16-byte aligned, strides multiples of 8.
 * Limits: keys and rows * (heads / key_heads) up to 2^22, batch * key_heads up to 65535, row_stride 0 to
 * 2^22, head_stride >= 0 and of q and dout, times heads / key_heads, up to 2^29.
 * out is rounded once; softmax weights and the gradients of the scores are rounded to dtype before the
 * products with them (those of Half times a power of two that keeps them among its normal numbers).
 * A weight carries fp32's error of its score and of lse, 2^-24 of their size: scores should stay below 2^24.
 * lse: [batch, heads, rows] floats, written forward, read backward.
 */
typedef struct stq_attention {
    int64_t dtype, batch, heads, key_heads, rows, keys, dim, window, sinks;
    double scale;
    stq_tensor4 q, k, v, out;
    const uint8_t *key_mask; /* [batch, keys], rows key_mask_stride apart, or null */
    int64_t key_mask_stride;
    float *lse;
    stq_tensor4 dout, dq, dk, dv; /* backward */
    void *workspace;
    int64_t workspace_bytes;
} stq_attention;

int64_t stq_attention_forward_workspace(const stq_attention *a);
int64_t stq_attention_backward_workspace(const stq_attention *a);
int stq_attention_forward(const stq_attention *a, void *stream);
int stq_attention_backward(const stq_attention *a, void *stream);

/*
 * Per row, with p the softmax of the teacher's logits / temperature over the row's entries, q the
 * softmax of logits / temperature and s that of logits:
 *   loss = alpha temperature^2 sum p (log p - log q) + (1 - alpha) (-log s[label])
 *   dlogits = drow (alpha temperature (q - p) + (1 - alpha) (s - [label]))
 * An entry whose id lies outside [0, vocab) is absent, a label outside it or a null `labels` too; a
 * row without entries has no first term, one without label no second, and one with neither is 0.  An
 * entry with a weight whose logit lies more than 3.4e38 temperature below the row's largest gives an infinite loss.
 * logits, dlogits: [n, vocab] of one type, rows strided; dlogits may be logits itself.  teacher, ids:
 * [n, k] dense, 0 <= k <= 1024.  temperature: 1e-15 to 1e15; alpha: 0 to 1.  loss: [n] floats or null.  stats: [n, 4] floats.
 * forward: dlogits null: loss and stats; dlogits given: loss and dlogits from one read of the logits.
 * backward: dlogits from the stats of a forward call.
 */
typedef struct stq_distill {
    int64_t n, vocab, dtype;
    const void *logits;
    int64_t stride;
    const void *teacher;
    int64_t teacher_dtype;
    const void *ids;
    int64_t id_dtype, k; /* STQ_LONG or STQ_INT */
    const void *labels;
    int64_t label_dtype;
    double temperature, alpha;
    float *loss, *stats;
    const float *drow;
    void *dlogits;
    int64_t dlogits_stride;
} stq_distill;

int stq_distill_forward(const stq_distill *a, void *stream);
int stq_distill_backward(const stq_distill *a, void *stream);

/*
 * Routing: per row p = softmax(logits) over the experts, and the k largest logits, ties to the lowest
 * expert; one of -inf is never chosen.  weights[j] = p of the j-th choice (renormalize: divided by the
 * choices' sum), ids[j] its expert; a row with fewer than k choices ends with weight 0 and id -1.
 * load[e] (or null) = sum of p[e] over the rows.  A row that holds a NaN or +inf has NaN for its p.
 *   dlogits = p (dload - <p, dload> - [not renormalize] <weights, dweights>)
 *           + [chosen] weights (dweights - [renormalize] <weights, dweights>)
 * logits: [n, experts] rows strided, Float, BFloat16 or Half, dlogits the same type; the others dense floats and
 * 32-bit ids.  experts 1 to 512, k 1 to min(experts, 64), n k up to 2^30.  dweights or dload may be null (zeros).
 * backward reads weights and ids of the forward call.  workspace: forward with load, stq_route_workspace(a) bytes.
 */
typedef struct stq_route {
    int64_t n, experts, k, dtype, renormalize;
    const void *logits;
    int64_t stride;
    float *weights;
    int32_t *ids;
    float *load;
    const float *dweights, *dload; /* backward */
    void *dlogits;
    int64_t dlogits_stride;
    void *workspace;
    int64_t workspace_bytes;
} stq_route;

int64_t stq_route_workspace(const stq_route *a);
int stq_route_forward(const stq_route *a, void *stream);
int stq_route_backward(const stq_route *a, void *stream);

/*
 * The slots sorted by expert, those of one expert in their order: rows[r] is the slot at place r, places[s]
 * where slot s stands, and expert e owns the places offsets[e] to offsets[e + 1] (experts + 1 offsets).  Slots
 * whose id lies outside [0, experts) come last.  slots up to 2^30, experts 1 to 512.
 */
typedef struct stq_expert_plan {
    const void *ids; /* [slots], STQ_LONG or STQ_INT */
    int64_t id_dtype, slots, experts;
    int32_t *rows, *places, *offsets;
    void *workspace;
    int64_t workspace_bytes;
} stq_expert_plan;

int64_t stq_expert_plan_workspace(const stq_expert_plan *a);
int stq_expert_plan_sort(const stq_expert_plan *a, void *stream);

/*
 * Products of each expert's run of rows with its weight [out, in]:
 *   y[r, :] = W[e] x[r, :],  dx[r, :] = W[e]^T dy[r, :],  dW[e] = sum over its rows of dy[r, :] x[r, :]^T
 * k > 0: row r reads x[rows[r] / k] of the `tokens` = slots / k rows of x, and dx is the sum over a token's k rows
 * (in fp32, rounded once); k = 0: row r is row r of x and dx.  Rows of no expert give y = dx = 0 and add nothing to dW,
 * an expert without rows gets dW = 0.  Sums are fp32, results rounded once.
 * BFloat16 or Half; in and out multiples of 8 up to 2^20; x, weight, dy: rows strided, 16-byte aligned, strides multiples
 * of 8; y, dx, dweight dense and aligned likewise.  dweight_dtype: dtype or Float.  backward: dx or dweight may be null (not wanted).
 * slots up to 2^30.  In tiles of 128 x 128, the rows that a pass writes (slots / 128, rounded down, times the tiles of out,
 * or of in for dx) and the weights have up to 2^23 each.
 * workspace: backward with dx and k > 0, stq_expert_product_workspace(a) bytes.
 */
typedef struct stq_expert_product {
    int64_t dtype, slots, experts, in, out, k, tokens;
    const void *x;
    int64_t x_stride;
    const void *weight;
    int64_t weight_expert_stride, weight_row_stride;
    const int32_t *rows, *places, *offsets; /* of a plan; rows and places with k > 0 */
    void *y;
    const void *dy; /* backward */
    int64_t dy_stride;
    void *dx, *dweight;
    int64_t dweight_dtype;
    void *workspace;
    int64_t workspace_bytes;
} stq_expert_product;

int64_t stq_expert_product_workspace(const stq_expert_product *a);
int stq_expert_product_forward(const stq_expert_product *a, void *stream);
int stq_expert_product_backward(const stq_expert_product *a, void *stream);

/*
 * out[t, :] = sum over j of weights[t, j] y[places[t, j], :] in fp32, slots of no expert left out (weights null: ones).
 *   dy[places[t, j], :] = weights[t, j] dout[t, :] (0 for slots of no expert),  dweights[t, j] = <y[places[t, j], :], dout[t, :]>
 * Float, BFloat16 or Half; y and dout rows strided, the others dense.  k 1 to 64, n k up to 2^30, dim up to 2^24.
 * dweights null: not wanted (y is then not read).
 */
typedef struct stq_expert_combine {
    int64_t n, k, experts, dim, dtype;
    const void *y;
    int64_t y_stride;
    const float *weights;
    const int32_t *places, *offsets;
    void *out;
    const void *dout; /* backward */
    int64_t dout_stride;
    void *dy;
    float *dweights;
} stq_expert_combine;

int stq_expert_combine_forward(const stq_expert_combine *a, void *stream);
int stq_expert_combine_backward(const stq_expert_combine *a, void *stream);

/*
 * The 2-norm of all tensors together, and out = grad min(1, max_norm / (norm + 1e-6)), of which a NaN norm makes NaN and
 * an infinite one 0 (NaN where the gradient is infinite, or max_norm).  Squares are added in double.  norm: one float on the
 * device.  given (or null): a norm to scale by in place of theirs, e.g. one summed over ranks; norm is then not written.
 * out may be grad; otherwise it lies apart from every grad and out of the list.  numel up to 2^36,
 * count to 2^24.  workspace: stq_clip_workspace(a) bytes (from count alone), 16-byte aligned.  The list is read before the call returns.
 */
typedef struct stq_grad {
    const void *grad; /* dense, Float, BFloat16 or Half */
    void *out; /* the same type; not read by stq_grad_norm */
    int64_t numel, dtype;
} stq_grad;
typedef struct stq_clip {
    const stq_grad *grads;
    int64_t count;
    double max_norm; /* >= 0 */
    const float *given;
    float *norm;
    void *workspace;
    int64_t workspace_bytes;
} stq_clip;

int64_t stq_clip_workspace(const stq_clip *a);
int stq_grad_norm(const stq_clip *a, void *stream);
int stq_clip_grads(const stq_clip *a, void *stream);

/* STQ_LM_ABI_VERSION the library was built with. */
int stq_lm_abi_version(void);

#ifdef __cplusplus
}
#endif

#endif /* STQUANT_LM_H */
