/*
 * stquant_lm.h -- C ABI of the transformer operators of libstquant_hip.so: embedding lookup,
 * residual norms, windowed attention and the distillation loss, each with its gradient.
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

/* STQ_LM_ABI_VERSION the library was built with. */
int stq_lm_abi_version(void);

#ifdef __cplusplus
}
#endif

#endif /* STQUANT_LM_H */
