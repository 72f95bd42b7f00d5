// lm_capi.cpp -- C ABI of the transformer operators (declared in include/stquant_lm.h): argument
// checks and the launches' arguments.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <new>
#include <vector>

#include "../../include/stquant_hip.h"
#include "../../include/stquant_lm.h"
#include "lm_attn.h"
#include "lm_clip.h"
#include "lm_common.h"
#include "lm_distill.h"
#include "lm_embed.h"
#include "lm_expert.h"
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

int check_workspace(const void *p, int64_t bytes, int64_t need)
{
    if (need) CHECK(check_ptr("workspace", p, 16));
    if (bytes < need)
        return fail(STQ_ERR_INVALID, "workspace needs %lld bytes, got %lld", (long long)need, (long long)bytes);
    return STQ_OK;
}

// The sizes alone (what the workspaces follow from).
int check_route_sizes(const stq_route *a)
{
    if (!a) return bad("null arguments");
    if (!is_float(a->dtype)) return bad_type("logits", a->dtype, FLOATS);
    CHECK(check_size("experts", a->experts, 1, lm::EXPERT_MAX));
    CHECK(check_size("k", a->k, 1, a->experts < lm::ROUTE_MAX_K ? a->experts : lm::ROUTE_MAX_K));
    return check_size("n", a->n, 0, lm::SLOT_MAX / a->k);
}

int check_route(const stq_route *a, bool backward)
{
    CHECK(check_route_sizes(a));
    if (a->renormalize != 0 && a->renormalize != 1) return bad("renormalize must be 0 or 1");
    if (!backward && a->load) {
        CHECK(check_ptr("load", a->load, 4));
        CHECK(check_workspace(a->workspace, a->workspace_bytes, lm::route_workspace(a->n, (int)a->experts)));
    }
    if (a->n == 0) return STQ_OK;
    CHECK(check_ptr("logits", a->logits, size_of(a->dtype)));
    if (a->stride < 0) return bad("rows of logits: the stride must be >= 0");
    CHECK(check_ptr("weights", a->weights, 4));
    CHECK(check_ptr("ids", a->ids, 4));
    if (!backward) return STQ_OK;
    if (a->dweights) CHECK(check_ptr("dweights", a->dweights, 4));
    if (a->dload) CHECK(check_ptr("dload", a->dload, 4));
    CHECK(check_ptr("dlogits", a->dlogits, size_of(a->dtype)));
    if (a->dlogits_stride < a->experts) return bad("rows of dlogits must not overlap");
    return STQ_OK;
}

lm::RouteArgs route_args(const stq_route *a)
{
    lm::RouteArgs o;
    o.logits = a->logits;
    o.dt = (int)a->dtype;
    o.n = a->n;
    o.stride = a->stride;
    o.experts = (int)a->experts;
    o.k = (int)a->k;
    o.renormalize = (int)a->renormalize;
    o.weights = a->weights;
    o.ids = a->ids;
    o.load = a->load;
    o.partial = (float *)a->workspace;
    o.dweights = a->dweights;
    o.dload = a->dload;
    o.dlogits = a->dlogits;
    o.dstride = a->dlogits_stride;
    return o;
}

int check_plan_sizes(const stq_expert_plan *a)
{
    if (!a) return bad("null arguments");
    if (!is_index(a->id_dtype)) return bad_type("ids", a->id_dtype, INDEXES);
    CHECK(check_size("experts", a->experts, 1, lm::EXPERT_MAX));
    return check_size("slots", a->slots, 0, lm::SLOT_MAX);
}

// Rows of 16-byte pieces.
int check_pieces(const char *name, const void *p, int64_t stride)
{
    CHECK(check_ptr(name, p, 16));
    if (stride < 0 || stride % 8) return fail(STQ_ERR_INVALID, "%s: strides must be multiples of 8 elements, >= 0", name);
    return STQ_OK;
}

// Kernels count tiles in 32 bits.  2^23 of 128 x 128 are results of 256 GiB in 16 bits; those that are not full (one an expert,
// and one of the rows of none, for each of up to 2^13 columns of tiles) come on top and stay below 2^23 too.
constexpr int64_t PRODUCT_TILES = 1 << 23;

int check_product_sizes(const stq_expert_product *a)
{
    if (!a) return bad("null arguments");
    if (a->dtype != STQ_BFLOAT16 && a->dtype != STQ_HALF) return bad_type("x and weight", a->dtype, "BFloat16 or Half");
    CHECK(check_size("experts", a->experts, 1, lm::EXPERT_MAX));
    CHECK(check_size("slots", a->slots, 0, lm::SLOT_MAX));
    CHECK(check_size("in", a->in, 8, 1 << 20));
    CHECK(check_size("out", a->out, 8, 1 << 20));
    if (a->in % 8 || a->out % 8) return bad("in and out must be multiples of 8");
    CHECK(check_size("k", a->k, 0, lm::ROUTE_MAX_K));
    if (a->k) CHECK(check_size("tokens", a->tokens, 0, lm::SLOT_MAX));
    if (a->k && a->tokens * a->k != a->slots)
        return fail(STQ_ERR_INVALID, "slots (%lld) must be tokens (%lld) times k (%lld)", (long long)a->slots, (long long)a->tokens, (long long)a->k);
    return check_size("tiles of weights", a->experts * ((a->in + 127) / 128) * ((a->out + 127) / 128), 0, PRODUCT_TILES);
}

// The full tiles of the rows that a pass writes: y of `out` columns, dx of `in` (dweight writes none).
int check_product_rows(const stq_expert_product *a, bool backward)
{
    if (backward && !a->dx) return STQ_OK;
    return check_size("tiles of rows", a->slots / 128 * (((backward ? a->in : a->out) + 127) / 128), 0, PRODUCT_TILES);
}

int check_product(const stq_expert_product *a, bool backward)
{
    CHECK(check_product_sizes(a));
    CHECK(check_product_rows(a, backward));
    CHECK(check_ptr("offsets", a->offsets, 4));
    CHECK(check_ptr("weight", a->weight, 16));
    if (a->weight_expert_stride % 8 || a->weight_row_stride % 8 || a->weight_expert_stride < 0 || a->weight_row_stride < 0)
        return bad("weight: strides must be multiples of 8 elements, >= 0");
    if (a->slots) {
        if (a->k) {
            CHECK(check_ptr("rows", a->rows, 4));
            CHECK(check_ptr("places", a->places, 4));
        }
        CHECK(check_pieces("x", a->x, a->x_stride));
        if (backward) CHECK(check_pieces("dy", a->dy, a->dy_stride));
        else CHECK(check_ptr("y", a->y, 16));
        if (backward && a->dx) CHECK(check_ptr("dx", a->dx, 16));
    }
    if (backward && a->dweight) {
        if (a->dweight_dtype != a->dtype && a->dweight_dtype != STQ_FLOAT) return bad_type("dweight", a->dweight_dtype, "Float or the type of x");
        CHECK(check_ptr("dweight", a->dweight, 16));
    }
    return STQ_OK;
}

lm::ProductArgs product_args(const stq_expert_product *a)
{
    lm::ProductArgs o;
    o.slots = a->slots;
    o.experts = (int)a->experts;
    o.in = (int)a->in;
    o.out = (int)a->out;
    o.k = (int)a->k;
    o.k_inverse = a->k ? 0xffffffffu / (uint32_t)a->k : 0;
    o.tokens = a->tokens;
    o.x = a->x;
    o.x_stride = a->x_stride;
    o.weight = a->weight;
    o.weight_expert_stride = a->weight_expert_stride;
    o.weight_row_stride = a->weight_row_stride;
    o.y = a->y;
    o.rows = a->rows;
    o.places = a->places;
    o.offsets = a->offsets;
    o.dy = a->dy;
    o.dy_stride = a->dy_stride;
    o.dx = a->dx;
    o.scratch = a->k ? (float *)a->workspace : nullptr;
    o.dweight = a->dweight;
    o.dweight_f32 = a->dweight_dtype == STQ_FLOAT;
    return o;
}

int check_combine(const stq_expert_combine *a, bool backward)
{
    if (!a) return bad("null arguments");
    if (!is_float(a->dtype)) return bad_type("y", a->dtype, FLOATS);
    CHECK(check_size("experts", a->experts, 1, lm::EXPERT_MAX));
    CHECK(check_size("k", a->k, 1, lm::ROUTE_MAX_K));
    CHECK(check_size("n", a->n, 0, lm::SLOT_MAX / a->k));
    CHECK(check_size("dim", a->dim, 1, 1 << 24));
    if (a->n == 0) return STQ_OK;
    const int z = size_of(a->dtype);
    if (a->weights) CHECK(check_ptr("weights", a->weights, 4));
    CHECK(check_ptr("places", a->places, 4));
    CHECK(check_ptr("offsets", a->offsets, 4));
    if (!backward || a->dweights) {
        CHECK(check_ptr("y", a->y, z));
        if (a->y_stride < 0) return bad("y_stride must be >= 0");
    }
    if (!backward) return check_ptr("out", a->out, z);
    CHECK(check_ptr("dout", a->dout, z));
    if (a->dout_stride < 0) return bad("dout_stride must be >= 0");
    if (a->dweights) CHECK(check_ptr("dweights", a->dweights, 4));
    return check_ptr("dy", a->dy, z);
}

lm::CombineArgs combine_args(const stq_expert_combine *a)
{
    lm::CombineArgs o;
    o.n = a->n;
    o.k = (int)a->k;
    o.experts = (int)a->experts;
    o.dim = a->dim;
    o.y = a->y;
    o.y_dt = o.out_dt = (int)a->dtype;
    o.y_stride = a->y_stride;
    o.weights = a->weights;
    o.places = a->places;
    o.offsets = a->offsets;
    o.out = a->out;
    o.out_stride = a->dim;
    o.dout = a->dout;
    o.dout_stride = a->dout_stride;
    o.dy = a->dy;
    o.dweights = a->dweights;
    return o;
}

int check_clip_list(const stq_clip *a)
{
    if (!a) return bad("null arguments");
    CHECK(check_size("count", a->count, 0, 1 << 24));
    if (a->count && !a->grads) return bad("grads: null data pointer");
    for (int64_t i = 0; i < a->count; i++) {
        const stq_grad &g = a->grads[i];
        if (!is_float(g.dtype)) return bad_type("gradients", g.dtype, FLOATS);
        CHECK(check_size("elements of a gradient", g.numel, 0, lm::CLIP_MAX_NUMEL));
        if (g.numel) CHECK(check_ptr("grad", g.grad, size_of(g.dtype)));
    }
    return STQ_OK;
}

// What is written lies apart from everything else in the list, but for a gradient in place.
int check_clip_apart(const stq_clip *a)
{
    struct Span {
        const char *from, *to;
        int64_t of;                       // the tensor; < 0: written, ~tensor
    };
    std::vector<Span> spans;
    spans.reserve(2 * a->count + 1);
    for (int64_t i = 0; i < a->count; i++) {
        const stq_grad &g = a->grads[i];
        if (g.numel == 0) continue;
        CHECK(check_ptr("out", g.out, size_of(g.dtype)));
        const int64_t bytes = g.numel * size_of(g.dtype);
        spans.push_back({(const char *)g.out, (const char *)g.out + bytes, ~i});
        if (g.out != g.grad) spans.push_back({(const char *)g.grad, (const char *)g.grad + bytes, i});
    }
    if (a->given) spans.push_back({(const char *)a->given, (const char *)(a->given + 1), a->count});
    std::sort(spans.begin(), spans.end(), [](const Span &x, const Span &y) { return x.from < y.from; });
    // the farthest ends so far, of all spans and of those written
    const char *any = nullptr, *written = nullptr;
    for (const Span &s : spans) {
        if ((s.of < 0 && any > s.from) || written > s.from) return bad("gradients that are written must not overlap others, or the given norm");
        any = std::max(any, s.to);
        if (s.of < 0) written = std::max(written, s.to);
    }
    return STQ_OK;
}

std::vector<lm::ClipTensor> clip_tensors(const stq_clip *a)
{
    std::vector<lm::ClipTensor> t(a->count);
    for (int64_t i = 0; i < a->count; i++) t[i] = {a->grads[i].grad, a->grads[i].out, a->grads[i].numel, (int)a->grads[i].dtype};
    return t;
}

// No exception leaves a C entry.
template <typename F>
auto guarded(F f, decltype(f()) failed) -> decltype(f())
{
    try {
        return f();
    } catch (const std::bad_alloc &) {
        return bad("out of host memory"), failed;
    }
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

int64_t stq_route_workspace(const stq_route *a)
{
    if (check_route_sizes(a) != STQ_OK) return -1;
    return lm::route_workspace(a->n, (int)a->experts);
}

int stq_route_forward(const stq_route *a, void *stream)
{
    CHECK(check_route(a, false));
    if (a->n == 0 && !a->load) return STQ_OK;
    return done(lm::route_forward(route_args(a), (hipStream_t)stream), "route forward");
}

int stq_route_backward(const stq_route *a, void *stream)
{
    CHECK(check_route(a, true));
    if (a->n == 0) return STQ_OK;
    return done(lm::route_backward(route_args(a), (hipStream_t)stream), "route backward");
}

int64_t stq_expert_plan_workspace(const stq_expert_plan *a)
{
    if (check_plan_sizes(a) != STQ_OK) return -1;
    return lm::plan_workspace(a->slots, (int)a->experts);
}

int stq_expert_plan_sort(const stq_expert_plan *a, void *stream)
{
    CHECK(check_plan_sizes(a));
    CHECK(check_ptr("offsets", a->offsets, 4));
    if (a->slots) {
        CHECK(check_ptr("ids", a->ids, size_of(a->id_dtype)));
        CHECK(check_ptr("rows", a->rows, 4));
        CHECK(check_ptr("places", a->places, 4));
    }
    CHECK(check_workspace(a->workspace, a->workspace_bytes, lm::plan_workspace(a->slots, (int)a->experts)));
    const lm::PlanArgs p = {a->ids, size_of(a->id_dtype), a->slots, (int)a->experts, a->rows, a->places, a->offsets, (int32_t *)a->workspace};
    return done(lm::expert_plan(p, (hipStream_t)stream), "expert plan");
}

int64_t stq_expert_product_workspace(const stq_expert_product *a)
{
    if (check_product_sizes(a) != STQ_OK || check_product_rows(a, true) != STQ_OK) return -1;
    return lm::product_workspace(product_args(a));
}

int stq_expert_product_forward(const stq_expert_product *a, void *stream)
{
    CHECK(check_product(a, false));
    if (a->slots == 0) return STQ_OK;
    const lm::ProductArgs o = product_args(a);
    return done(a->dtype == STQ_BFLOAT16 ? lm::product_forward<lm::DT_BF16>(o, (hipStream_t)stream) : lm::product_forward<lm::DT_F16>(o, (hipStream_t)stream),
                "expert product forward");
}

int stq_expert_product_backward(const stq_expert_product *a, void *stream)
{
    CHECK(check_product(a, true));
    lm::ProductArgs o = product_args(a);
    if (a->slots == 0) o.dx = nullptr;
    CHECK(check_workspace(a->workspace, a->workspace_bytes, lm::product_workspace(o)));
    return done(a->dtype == STQ_BFLOAT16 ? lm::product_backward<lm::DT_BF16>(o, (hipStream_t)stream) : lm::product_backward<lm::DT_F16>(o, (hipStream_t)stream),
                "expert product backward");
}

int stq_expert_combine_forward(const stq_expert_combine *a, void *stream)
{
    CHECK(check_combine(a, false));
    return done(lm::combine_forward(combine_args(a), (hipStream_t)stream), "expert combine forward");
}

int stq_expert_combine_backward(const stq_expert_combine *a, void *stream)
{
    CHECK(check_combine(a, true));
    return done(lm::combine_backward(combine_args(a), (hipStream_t)stream), "expert combine backward");
}

int64_t stq_clip_workspace(const stq_clip *a)
{
    if (!a) return bad("null arguments"), -1;
    if (check_size("count", a->count, 0, 1 << 24) != STQ_OK) return -1;
    return lm::clip_workspace(a->count);
}

int stq_grad_norm(const stq_clip *a, void *stream)
{
    return guarded([&]() -> int {
        CHECK(check_clip_list(a));
        CHECK(check_ptr("norm", a->norm, 4));
        const auto t = clip_tensors(a);
        CHECK(check_workspace(a->workspace, a->workspace_bytes, lm::clip_workspace(a->count)));
        return done(lm::clip_norm(t.data(), (int64_t)t.size(), (double *)a->workspace, a->norm, (hipStream_t)stream), "gradient norm");
    }, STQ_ERR_INVALID);
}

int stq_clip_grads(const stq_clip *a, void *stream)
{
    return guarded([&]() -> int {
        CHECK(check_clip_list(a));
        if (!(a->max_norm >= 0.0)) return bad("max_norm must be >= 0");
        CHECK(check_clip_apart(a));
        const auto t = clip_tensors(a);
        if (a->given) CHECK(check_ptr("given norm", a->given, 4));
        else {
            CHECK(check_ptr("norm", a->norm, 4));
            CHECK(check_workspace(a->workspace, a->workspace_bytes, lm::clip_workspace(a->count)));
        }
        return done(lm::clip_scale(t.data(), (int64_t)t.size(), a->max_norm, a->given, (double *)a->workspace, a->given ? nullptr : a->norm, (hipStream_t)stream),
                    "gradient clipping");
    }, STQ_ERR_INVALID);
}

}  // extern "C"
