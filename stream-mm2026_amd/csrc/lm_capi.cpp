// lm_capi.cpp -- C ABI of the transformer operators (declared in include/stquant_lm.h): argument
// checks and the launches' arguments.
#include <hip/hip_runtime.h>

#include <climits>
#include <cmath>

#include "../../include/stquant_hip.h"
#include "../../include/stquant_lm.h"
#include "lm_attn.h"
#include "lm_common.h"
#include "lm_distill.h"
#include "lm_embed.h"
#include "lm_norm.h"
#include "mdq_error.h"

namespace {

using mdq::dtype_name;
using mdq::fail;
using mdq::hip_fail;

bool is_float(int64_t dt) { return dt == STQ_FLOAT || dt == STQ_BFLOAT16 || dt == STQ_HALF; }
bool is_index(int64_t dt) { return dt == STQ_LONG || dt == STQ_INT; }
int size_of(int64_t dt) { return dt == STQ_LONG ? 8 : dt == STQ_FLOAT || dt == STQ_INT ? 4 : 2; }

int bad(const char *what) { return fail(STQ_ERR_INVALID, "%s", what); }

int bad_type(const char *name, int64_t dt, const char *want)
{
    return fail(STQ_ERR_INVALID, "%s must be %s, got %s", name, want, dtype_name((int)dt));
}
constexpr const char *FLOATS = "Float, BFloat16 or Half", *INDEXES = "Long or Int";

// p holds elements of `bytes`: given and aligned to them.
int check_ptr(const char *name, const void *p, int bytes)
{
    if (!p) return fail(STQ_ERR_INVALID, "%s: null data pointer", name);
    if ((uintptr_t)p % bytes) return fail(STQ_ERR_INVALID, "%s must be aligned to %d bytes", name, bytes);
    return STQ_OK;
}

int check_size(const char *name, int64_t v, int64_t lo, int64_t hi)
{
    if (v < lo || v > hi)
        return fail(STQ_ERR_INVALID, "%s must be %lld to %lld, got %lld", name, (long long)lo, (long long)hi, (long long)v);
    return STQ_OK;
}

int done(hipError_t e, const char *what) { return e == hipSuccess ? STQ_OK : hip_fail(e, what); }

#define CHECK(x)                     \
    do {                             \
        const int rc_ = (x);         \
        if (rc_ != STQ_OK) return rc_; \
    } while (0)

int check_tokens(const void *tokens, int64_t dt, int64_t n, int64_t vocab, int64_t dim, double scale)
{
    if (!is_index(dt)) return bad_type("tokens", dt, INDEXES);
    CHECK(check_size("n", n, 0, INT_MAX));
    CHECK(check_size("vocab", vocab, 1, INT_MAX));
    CHECK(check_size("dim", dim, 1, 1 << 24));
    if (n) CHECK(check_ptr("tokens", tokens, size_of(dt)));
    if (!std::isfinite(scale)) return bad("scale must be finite");
    return STQ_OK;
}

int check_embedding_grad(const stq_embedding_grad *a)
{
    if (!a) return bad("null arguments");
    CHECK(check_tokens(a->tokens, a->token_dtype, a->n, a->vocab, a->dim, a->scale));
    CHECK(check_size("n", a->n, 0, lm::EMBED_GRAD_MAX));
    CHECK(check_size("vocab", a->vocab, 1, lm::EMBED_GRAD_MAX));
    if (!is_float(a->grad_dtype)) return bad_type("grad", a->grad_dtype, FLOATS);
    if (!is_float(a->dweight_dtype)) return bad_type("dweight", a->dweight_dtype, FLOATS);
    return STQ_OK;
}

int check_norm(const stq_norm_residual *a, bool backward)
{
    if (!a) return bad("null arguments");
    if (!is_float(a->dtype)) return bad_type("x", a->dtype, FLOATS);
    if (a->weight_dtype != a->dtype && a->weight_dtype != STQ_FLOAT) return bad_type("weights", a->weight_dtype, "Float or the type of x");
    CHECK(check_size("n", a->n, 0, INT_MAX));
    CHECK(check_size("dim", a->dim, lm::NORM_MIN_DIM, lm::NORM_MAX_DIM));
    if (a->layer != 0 && a->layer != 1) return bad("layer must be 0 or 1");
    if (!(a->eps >= 0.0) || !std::isfinite(a->eps)) return bad("eps must be finite and >= 0");
    if (!std::isfinite(a->residual_scale)) return bad("residual_scale must be finite");
    if (!a->pre_weight) return bad("pre_weight: null data pointer");
    if (a->post_bias && !a->post_weight) return bad("post_bias needs post_weight");
    if (!a->layer && (a->pre_bias || a->post_bias)) return bad("biases need layer norms (layer = 1)");
    if (a->gate) {
        CHECK(check_size("gate rows", a->groups, 1, a->n > 0 ? a->n : 1 << 30));
        if (a->n % a->groups)
            return fail(STQ_ERR_INVALID, "gate rows (%lld) must divide the rows (%lld)", (long long)a->groups, (long long)a->n);
    }
    const int z = size_of(a->dtype), wz = size_of(a->weight_dtype);
    const void *const weights[5] = {a->pre_weight, a->pre_bias, a->post_weight, a->post_bias, a->gate};
    void *const grads[5] = {a->dpre_weight, a->dpre_bias, a->dpost_weight, a->dpost_bias, a->dgate};
    static const char *const names[5] = {"pre_weight", "pre_bias", "post_weight", "post_bias", "gate"};
    for (int i = 0; i < 5; i++) {
        if (weights[i]) CHECK(check_ptr(names[i], weights[i], wz));
        if (!backward) continue;
        if (!weights[i] != !grads[i]) return fail(STQ_ERR_INVALID, "the gradient of %s goes with it", names[i]);
        if (grads[i]) CHECK(check_ptr(names[i], grads[i], wz));
    }
    if (a->n == 0) return STQ_OK;
    CHECK(check_ptr("x", a->x, z));
    CHECK(check_ptr("block", a->block, z));
    CHECK(check_ptr("stats", a->stats, 16));
    if (a->x_stride < 0 || a->block_stride < 0) return bad("row strides must be >= 0");
    if (!backward) {
        CHECK(check_ptr("r", a->r, z));
        return check_ptr("h", a->h, z);
    }
    CHECK(check_ptr("dh", a->dh, z));
    if (a->dr) CHECK(check_ptr("dr", a->dr, z));
    if (a->dh_stride < 0 || a->dr_stride < 0) return bad("row strides must be >= 0");
    CHECK(check_ptr("dx", a->dx, z));
    return check_ptr("dblock", a->dblock, z);
}

lm::NormArgs norm_args(const stq_norm_residual *a)
{
    lm::NormArgs o;
    o.n = a->n;
    o.dim = a->dim;
    o.dt = (int)a->dtype;
    o.weight_dt = (int)a->weight_dtype;
    o.x = a->x;
    o.block = a->block;
    o.x_stride = a->x_stride;
    o.block_stride = a->block_stride;
    o.pre_weight = a->pre_weight;
    o.pre_bias = a->pre_bias;
    o.post_weight = a->post_weight;
    o.post_bias = a->post_bias;
    o.gate = a->gate;
    o.groups = a->gate ? a->groups : 1;
    o.residual_scale = (float)a->residual_scale;
    o.eps = (float)a->eps;
    o.layer = (int)a->layer;
    o.stats = a->stats;
    o.r = a->r;
    o.h = a->h;
    o.dr = a->dr;
    o.dh = a->dh;
    o.dr_stride = a->dr_stride;
    o.dh_stride = a->dh_stride;
    o.dx = a->dx;
    o.dblock = a->dblock;
    o.dpre_weight = a->dpre_weight;
    o.dpre_bias = a->dpre_bias;
    o.dpost_weight = a->dpost_weight;
    o.dpost_bias = a->dpost_bias;
    o.dgate = a->dgate;
    o.workspace = (float *)a->workspace;
    return o;
}

int check_tensor4(const char *name, const stq_tensor4 &t)
{
    CHECK(check_ptr(name, t.p, 16));
    if (t.batch_stride % 8 || t.head_stride % 8 || t.row_stride % 8)
        return fail(STQ_ERR_INVALID, "%s: strides must be multiples of 8 elements", name);
    // a tile of 64 rows and the heads that share a key head are addressed by 31 bits of bytes
    if (t.row_stride < 0 || t.row_stride > 1 << 22 || t.head_stride < 0) return fail(STQ_ERR_INVALID, "%s: row_stride must be 0 to 2^22, head_stride >= 0", name);
    return STQ_OK;
}

// The sizes alone (what the workspaces follow from).
int check_attention_sizes(const stq_attention *a)
{
    if (!a) return bad("null arguments");
    if (a->dtype != STQ_BFLOAT16 && a->dtype != STQ_HALF) return bad_type("q, k and v", a->dtype, "BFloat16 or Half");
    CHECK(check_size("batch", a->batch, 0, 65535));
    CHECK(check_size("key_heads", a->key_heads, 1, 65535));
    CHECK(check_size("heads", a->heads, 1, 65535));
    if (a->heads % a->key_heads)
        return fail(STQ_ERR_INVALID, "heads (%lld) must be a multiple of key_heads (%lld)", (long long)a->heads, (long long)a->key_heads);
    CHECK(check_size("batch * key_heads", a->batch * a->key_heads, 0, 65535));
    // (a launch has at most 65535 tiles of 128 rows, or 128 keys and their shares)
    CHECK(check_size("keys", a->keys, 0, 1 << 22));
    CHECK(check_size("rows", a->rows, 0, a->keys));
    CHECK(check_size("rows * heads / key_heads", a->rows * (a->heads / a->key_heads), 0, 1 << 22));
    CHECK(check_size("dim", a->dim, 8, 128));
    if (a->dim % 8) return fail(STQ_ERR_INVALID, "dim must be a multiple of 8, got %lld", (long long)a->dim);
    if (a->window < 0 || a->sinks < 0) return bad("window and sinks must be >= 0");
    return STQ_OK;
}

int check_attention(const stq_attention *a, bool backward)
{
    CHECK(check_attention_sizes(a));
    // (a float of 0 would turn hidden scores, -inf, into NaN, an infinite one scores of 0)
    if (!(a->scale >= 1e-30 && a->scale <= 1e30)) return bad("scale must be finite and > 0 (1e-30 to 1e30)");
    if (a->batch == 0 || a->keys == 0 || (a->rows == 0 && !backward)) return STQ_OK;
    const int64_t group = a->heads / a->key_heads;
    if (a->rows && (group * a->q.head_stride > 1 << 29 || (backward && group * a->dout.head_stride > 1 << 29)))
        return bad("q and dout: the heads of a key head must lie within 2^29 elements");
    if (a->key_mask && a->key_mask_stride < 0) return bad("key_mask_stride must be >= 0");
    CHECK(check_tensor4("k", a->k));
    CHECK(check_tensor4("v", a->v));
    if (a->rows) {
        CHECK(check_tensor4("q", a->q));
        CHECK(check_tensor4("out", a->out));
        CHECK(check_ptr("lse", a->lse, 4));
    }
    if (!backward) return STQ_OK;
    if (a->rows) {
        CHECK(check_tensor4("dout", a->dout));
        CHECK(check_tensor4("dq", a->dq));
    }
    CHECK(check_tensor4("dk", a->dk));
    return check_tensor4("dv", a->dv);
}

lm::AttnTensor tensor4(const stq_tensor4 &t) { return {t.p, t.batch_stride, t.head_stride, t.row_stride}; }

lm::AttnArgs attn_args(const stq_attention *a)
{
    lm::AttnArgs o;
    o.q = tensor4(a->q);
    o.k = tensor4(a->k);
    o.v = tensor4(a->v);
    o.o = tensor4(a->out);
    o.dout = tensor4(a->dout);
    o.dq = tensor4(a->dq);
    o.dk = tensor4(a->dk);
    o.dv = tensor4(a->dv);
    o.key_mask = a->key_mask;
    o.mask_stride = a->key_mask_stride;
    o.lse = a->lse;
    o.delta = (float *)a->workspace;
    o.partial = (float *)a->workspace;
    o.batch = (int)a->batch;
    o.heads = (int)a->heads;
    o.key_heads = (int)a->key_heads;
    o.group = (int)(a->heads / a->key_heads);
    o.rows = (int)a->rows;
    o.keys = (int)a->keys;
    o.dim = (int)a->dim;
    // a window of all keys and more is one of all keys; sinks behind the last key are none
    o.window = (int)(a->window == 0 || a->window > a->keys ? a->keys : a->window);
    o.sinks = (int)(a->sinks > a->keys ? a->keys : a->sinks);
    o.scale = (float)a->scale;
    o.splits = lm::attn_splits(o);
    return o;
}

int check_distill(const stq_distill *a)
{
    if (!a) return bad("null arguments");
    if (!is_float(a->dtype)) return bad_type("logits", a->dtype, FLOATS);
    if (!is_float(a->teacher_dtype)) return bad_type("teacher logits", a->teacher_dtype, FLOATS);
    if (!is_index(a->id_dtype)) return bad_type("teacher ids", a->id_dtype, INDEXES);
    if (a->labels && !is_index(a->label_dtype)) return bad_type("labels", a->label_dtype, INDEXES);
    CHECK(check_size("n", a->n, 0, INT_MAX));
    CHECK(check_size("vocab", a->vocab, 1, 1 << 30));
    CHECK(check_size("teacher entries", a->k, 0, lm::DISTILL_MAX_K));
    // (its square and its reciprocal are floats)
    if (!(a->temperature >= 1e-15 && a->temperature <= 1e15)) return bad("temperature must be finite and > 0 (1e-15 to 1e15)");
    if (!(a->alpha >= 0.0 && a->alpha <= 1.0)) return bad("alpha must be 0 to 1");
    if (a->n == 0) return STQ_OK;
    CHECK(check_ptr("logits", a->logits, size_of(a->dtype)));
    if (a->k) {
        CHECK(check_ptr("teacher logits", a->teacher, size_of(a->teacher_dtype)));
        CHECK(check_ptr("teacher ids", a->ids, size_of(a->id_dtype)));
    }
    if (a->labels) CHECK(check_ptr("labels", a->labels, size_of(a->label_dtype)));
    if (a->stride < 0 || (a->dlogits && a->dlogits_stride < a->vocab)) return bad("rows of logits must not overlap");
    if (a->dlogits) {
        CHECK(check_ptr("dlogits", a->dlogits, size_of(a->dtype)));
        CHECK(check_ptr("drow", a->drow, 4));
        // in place, or apart: a row is written while others are still read
        const char *z0 = (const char *)a->logits, *d0 = (const char *)a->dlogits;
        const int64_t z = size_of(a->dtype), zn = ((a->n - 1) * a->stride + a->vocab) * z, dn = ((a->n - 1) * a->dlogits_stride + a->vocab) * z;
        if (!(z0 == d0 && a->stride == a->dlogits_stride) && z0 < d0 + dn && d0 < z0 + zn) return bad("dlogits must be the logits or lie apart from them");
    }
    return STQ_OK;
}

lm::DistillArgs distill_args(const stq_distill *a)
{
    lm::DistillArgs o;
    o.logits = a->logits;
    o.dt = (int)a->dtype;
    o.n = a->n;
    o.vocab = a->vocab;
    o.stride = a->stride;
    o.teacher = a->teacher;
    o.teacher_dt = (int)a->teacher_dtype;
    o.ids = a->ids;
    o.id_bytes = size_of(a->id_dtype);
    o.k = (int)a->k;
    o.labels = a->labels;
    o.label_bytes = size_of(a->label_dtype);
    o.temperature = (float)a->temperature;
    o.alpha = (float)a->alpha;
    o.loss = a->loss;
    o.stats = a->stats;
    o.drow = a->drow;
    o.dlogits = a->dlogits;
    o.dstride = a->dlogits_stride;
    return o;
}

}  // namespace

extern "C" {

int stq_lm_abi_version(void) { return STQ_LM_ABI_VERSION; }

int stq_embedding_forward(const stq_embedding *a, void *stream)
{
    if (!a) return bad("null arguments");
    CHECK(check_tokens(a->tokens, a->token_dtype, a->n, a->vocab, a->dim, a->scale));
    if (!is_float(a->weight_dtype)) return bad_type("weight", a->weight_dtype, FLOATS);
    if (!is_float(a->out_dtype)) return bad_type("out", a->out_dtype, FLOATS);
    if (a->n == 0) return STQ_OK;
    CHECK(check_ptr("weight", a->weight, size_of(a->weight_dtype)));
    CHECK(check_ptr("out", a->out, size_of(a->out_dtype)));
    if (a->weight_stride < 0) return bad("weight_stride must be >= 0");
    const lm::EmbedArgs e = {a->tokens, size_of(a->token_dtype), a->n, a->vocab, a->dim, (float)a->scale};
    return done(lm::embed_forward(e, a->weight, (int)a->weight_dtype, a->weight_stride, a->out, (int)a->out_dtype, (hipStream_t)stream),
                "embedding forward");
}

int64_t stq_embedding_grad_workspace(const stq_embedding_grad *a)
{
    if (check_embedding_grad(a) != STQ_OK) return -1;
    return lm::embed_backward_workspace(a->n, a->vocab, a->dim);
}

int stq_embedding_backward(const stq_embedding_grad *a, void *stream)
{
    CHECK(check_embedding_grad(a));
    if (a->n) CHECK(check_ptr("grad", a->grad, size_of(a->grad_dtype)));
    CHECK(check_ptr("dweight", a->dweight, size_of(a->dweight_dtype)));
    if (a->grad_stride < 0 || a->dweight_stride < a->dim) return bad("rows of dweight must not overlap");
    CHECK(check_ptr("workspace", a->workspace, 16));
    const int64_t need = lm::embed_backward_workspace(a->n, a->vocab, a->dim);
    if (a->workspace_bytes < need)
        return fail(STQ_ERR_INVALID, "workspace needs %lld bytes, got %lld", (long long)need, (long long)a->workspace_bytes);
    const lm::EmbedArgs e = {a->tokens, size_of(a->token_dtype), a->n, a->vocab, a->dim, (float)a->scale};
    return done(lm::embed_backward(e, a->grad, (int)a->grad_dtype, a->grad_stride, a->dweight, (int)a->dweight_dtype, a->dweight_stride,
                                   a->padding < 0 ? -1 : a->padding, a->accumulate != 0, a->workspace, (hipStream_t)stream),
                "embedding backward");
}

int64_t stq_norm_residual_workspace(const stq_norm_residual *a)
{
    if (!a) return bad("null arguments"), -1;
    if (check_size("n", a->n, 0, INT_MAX) != STQ_OK || check_size("dim", a->dim, lm::NORM_MIN_DIM, lm::NORM_MAX_DIM) != STQ_OK) return -1;
    return lm::norm_backward_workspace(a->n, a->dim, a->gate && a->groups > 0 ? a->groups : 1);
}

int stq_norm_residual_forward(const stq_norm_residual *a, void *stream)
{
    CHECK(check_norm(a, false));
    return done(lm::norm_forward(norm_args(a), (hipStream_t)stream), "norm_residual forward");
}

int stq_norm_residual_backward(const stq_norm_residual *a, void *stream)
{
    CHECK(check_norm(a, true));
    CHECK(check_ptr("workspace", a->workspace, 16));
    const int64_t need = stq_norm_residual_workspace(a);
    if (a->workspace_bytes < need)
        return fail(STQ_ERR_INVALID, "workspace needs %lld bytes, got %lld", (long long)need, (long long)a->workspace_bytes);
    return done(lm::norm_backward(norm_args(a), (hipStream_t)stream), "norm_residual backward");
}

int64_t stq_attention_forward_workspace(const stq_attention *a)
{
    if (check_attention_sizes(a) != STQ_OK) return -1;
    return a->batch && a->rows ? 4 * lm::attn_forward_workspace(attn_args(a)) : 0;
}

int64_t stq_attention_backward_workspace(const stq_attention *a)
{
    if (check_attention_sizes(a) != STQ_OK) return -1;
    return a->batch && a->keys ? 4 * lm::attn_backward_workspace(attn_args(a)) : 0;
}

int stq_attention_forward(const stq_attention *a, void *stream)
{
    CHECK(check_attention(a, false));
    if (a->batch == 0 || a->rows == 0) return STQ_OK;
    const int64_t need = stq_attention_forward_workspace(a);
    if (need) CHECK(check_ptr("workspace", a->workspace, 16));
    if (a->workspace_bytes < need)
        return fail(STQ_ERR_INVALID, "workspace needs %lld bytes, got %lld", (long long)need, (long long)a->workspace_bytes);
    const lm::AttnArgs o = attn_args(a);
    return done(a->dtype == STQ_BFLOAT16 ? lm::attn_forward<lm::DT_BF16>(o, (hipStream_t)stream) : lm::attn_forward<lm::DT_F16>(o, (hipStream_t)stream),
                "attention forward");
}

int stq_attention_backward(const stq_attention *a, void *stream)
{
    CHECK(check_attention(a, true));
    if (a->batch == 0 || a->keys == 0) return STQ_OK;
    const int64_t need = stq_attention_backward_workspace(a);
    if (need) CHECK(check_ptr("workspace", a->workspace, 16));
    if (a->workspace_bytes < need)
        return fail(STQ_ERR_INVALID, "workspace needs %lld bytes, got %lld", (long long)need, (long long)a->workspace_bytes);
    lm::AttnArgs o = attn_args(a);
    o.partial = o.delta + lm::attn_backward_delta(o);
    return done(a->dtype == STQ_BFLOAT16 ? lm::attn_backward<lm::DT_BF16>(o, (hipStream_t)stream) : lm::attn_backward<lm::DT_F16>(o, (hipStream_t)stream),
                "attention backward");
}

int stq_distill_forward(const stq_distill *a, void *stream)
{
    CHECK(check_distill(a));
    if (a->n == 0) return STQ_OK;
    if (a->loss) CHECK(check_ptr("loss", a->loss, 4));
    if (!a->dlogits) CHECK(check_ptr("stats", a->stats, 4));
    lm::DistillArgs o = distill_args(a);
    if (o.dlogits) o.stats = nullptr;
    return done(lm::distill_forward(o, (hipStream_t)stream), "distill forward");
}

int stq_distill_backward(const stq_distill *a, void *stream)
{
    CHECK(check_distill(a));
    if (a->n == 0) return STQ_OK;
    CHECK(check_ptr("stats", a->stats, 4));
    if (!a->dlogits) return bad("dlogits: null data pointer");
    return done(lm::distill_backward(distill_args(a), (hipStream_t)stream), "distill backward");
}

}  // extern "C"
