// lm_distill.hip -- distillation from a teacher's top logits, mixed with the labels' cross-entropy.
//
//   p = softmax over the row's teacher entries of t / T,  q = softmax(z / T),  s = softmax(z)
//   loss = a T^2 sum_k p_k (log p_k - log q_{id_k}) + (1 - a) (-log s_label)
//   dloss/dz_j = a T (q_j - sum_{k : id_k = j} p_k) + (1 - a) (s_j - [j = label])
//
// An entry whose id lies outside the vocabulary is absent, a label outside it too; a row with
// neither has loss 0 and gradient 0 whatever its logits hold.
//
// Bound by memory: N V logits read, and N V gradients written where they are asked for.  One
// workgroup owns a row and keeps it in registers between the maximum, the sums and the gradient,
// so that the logits are read once; a row too long for that is read again (from the last-level
// cache, mostly).  Rows start anywhere: the 16-byte pieces of a row are those of memory, and the
// few elements before the first and behind the last whole piece go one by one.
#include "lm_common.h"
#include "lm_distill.h"

namespace lm {
namespace {

constexpr float LOG2E = 1.44269504088896340736f;

__device__ __forceinline__ int64_t index_at(const void *p, int bytes, int64_t i)
{
    return bytes == 8 ? ((const int64_t *)p)[i] : (int64_t)((const int32_t *)p)[i];
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

struct RowLds {
    float buf[4][16];
    int ids[DISTILL_MAX_K];
    float p[DISTILL_MAX_K];
};

// How a row lies in memory: `head` single elements, `pieces` whole 16-byte pieces, `tail` single ones.
struct RowShape {
    const char *row;
    int head, pieces, tail;
};

template <int DT>
__device__ __forceinline__ RowShape row_shape(const void *base, int64_t first, int vocab)
{
    using E = Elem<DT>;
    RowShape s;
    s.row = (const char *)base + first * E::SIZE;
    const int off = (int)((uintptr_t)s.row & 15) / E::SIZE;
    s.head = min(vocab, off ? E::PER16 - off : 0);
    s.pieces = (vocab - s.head) / E::PER16;
    s.tail = vocab - s.head - s.pieces * E::PER16;
    return s;
}

// MODE 0: loss (and stats); 1: loss and gradient; 2: gradient from stats.  NC: pieces a thread
// keeps in registers (0: none, the row is read again).
template <int DT, int MODE, int THREADS, int NC>
__global__ __launch_bounds__(THREADS) void distill_kernel(DistillArgs a)
{
    using E = Elem<DT>;
    constexpr int W = THREADS / 64, P = E::PER16;
    __shared__ RowLds s;
    const int tid = threadIdx.x;
    const int64_t n = blockIdx.x;
    const int vocab = (int)a.vocab;
    const RowShape sh = row_shape<DT>(a.logits, n * a.stride, vocab);
    const u32x4 *body = (const u32x4 *)(sh.row + sh.head * E::SIZE);
    const float invT = 1.0f / a.temperature;
    const bool has_label = a.labels != nullptr;

    // the teacher's entries: one a thread where there are as many threads
    int any = 0;
    for (int k = tid; k < a.k; k += THREADS) {
        const int64_t id = index_at(a.ids, a.id_bytes, n * a.k + k);
        const bool there = id >= 0 && id < vocab;
        s.ids[k] = there ? (int)id : -1;
        s.p[k] = there ? load_any(a.teacher_dt, a.teacher, n * a.k + k) * invT : -__builtin_inff();
        any |= there;
    }
    const bool taught = __syncthreads_or(any) && a.alpha != 0.0f;
    int64_t label = has_label ? index_at(a.labels, a.label_bytes, n) : -1;
    const bool named = label >= 0 && label < vocab && a.alpha != 1.0f;
    const float wd = taught ? a.alpha : 0.0f, wl = named ? 1.0f - a.alpha : 0.0f;

    // dlogits' pieces are those of the logits where both rows start alike in their 16 bytes
    char *drow = MODE == 0 ? nullptr : (char *)a.dlogits + n * a.dstride * E::SIZE;
    const bool alike = MODE != 0 && (((uintptr_t)drow ^ (uintptr_t)sh.row) & 15) == 0;
    u32x4 *dbody = (u32x4 *)(drow + sh.head * E::SIZE);

    if (!taught && !named) {
        if (tid == 0) {
            if (MODE != 2 && a.loss) a.loss[n] = 0.0f;
            if (MODE == 0 && a.stats)
                for (int j = 0; j < 4; j++) a.stats[n * 4 + j] = 0.0f;
        }
        if (MODE != 0) {
            for (int i = tid; i < sh.pieces; i += THREADS) {
                if (alike) dbody[i] = u32x4{0, 0, 0, 0};
                else
                    for (int j = 0; j < P; j++) E::store(drow, sh.head + i * P + j, 0.0f);
            }
            for (int i = tid; i < sh.head + sh.tail; i += THREADS)
                E::store(drow, i < sh.head ? i : vocab - sh.tail + (i - sh.head), 0.0f);
        }
        return;
    }

    // the row
    u32x4 reg[NC ? NC : 1];
    if constexpr (NC > 0) {
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const int i = tid + c * THREADS;
            if (i < sh.pieces) reg[c] = body[i];
        }
    }
    // each single element of head and tail is one thread's (there are fewer than 2 P of them)
    const int edge = tid < sh.head ? tid : tid < sh.head + sh.tail ? vocab - sh.tail + (tid - sh.head) : -1;
    const float zedge = edge >= 0 ? E::load(sh.row, edge) : -__builtin_inff();
    // the logits at the teacher's entries and the label, read before a gradient may overwrite them
    constexpr int KPT = (DISTILL_MAX_K + THREADS - 1) / THREADS;
    float zk[KPT];
#pragma unroll
    for (int u = 0; u < KPT; u++) {
        const int k = tid + u * THREADS;
        zk[u] = k < a.k && s.ids[k] >= 0 ? E::load(sh.row, s.ids[k]) : 0.0f;
    }
    const float zl = named ? E::load(sh.row, label) : 0.0f;

    auto each = [&](auto f) {            // f(value index of the piece, its values)
        float v[P];
        if constexpr (NC > 0) {
#pragma unroll
            for (int c = 0; c < NC; c++) {
                const int i = tid + c * THREADS;
                if (i < sh.pieces) {
                    E::unpack(reg[c], v);
                    f(i, v);
                }
            }
        } else {
            for (int i = tid; i < sh.pieces; i += THREADS) {
                E::unpack(body[i], v);
                f(i, v);
            }
        }
    };

    float top, lse_t, lse_1;             // the row's maximum and the two log-sums below it
    const float cT = invT * LOG2E;
    if constexpr (MODE == 2) {
        top = a.stats[n * 4];
        lse_t = a.stats[n * 4 + 1];
        lse_1 = a.stats[n * 4 + 2];
    } else {
        float m = zedge;
        each([&](int, float *v) {
#pragma unroll
            for (int j = 0; j < P; j++) m = Max()(m, v[j]);
        });
        top = group_reduce<W>(m, Max(), s.buf[0]);
        float st = 0.0f, s1 = 0.0f;
        if (taught) {
            st = edge >= 0 ? exp2_hw((zedge - top) * cT) : 0.0f;
            each([&](int, float *v) {
#pragma unroll
                for (int j = 0; j < P; j++) st += exp2_hw((v[j] - top) * cT);
            });
        }
        if (named) {
            s1 = edge >= 0 ? exp2_hw((zedge - top) * LOG2E) : 0.0f;
            each([&](int, float *v) {
#pragma unroll
                for (int j = 0; j < P; j++) s1 += exp2_hw((v[j] - top) * LOG2E);
            });
        }
        lse_t = taught ? logf(group_reduce<W>(st, Add(), s.buf[1])) : 0.0f;
        lse_1 = named ? logf(group_reduce<W>(s1, Add(), s.buf[2])) : 0.0f;
    }

    // the teacher's distribution (every wave forms it: k values in LDS)
    float logz = 0.0f, tmax = -__builtin_inff();
    if (taught) {
        float m = -__builtin_inff();
        for (int k = tid & 63; k < a.k; k += 64)
            if (s.ids[k] >= 0) m = Max()(m, s.p[k]);
        tmax = wave_reduce(m, Max());
        const float ref = tmax == -__builtin_inff() ? 0.0f : tmax;
        float z = 0.0f;
        for (int k = tid & 63; k < a.k; k += 64)
            if (s.ids[k] >= 0) z += expf(s.p[k] - ref);
        z = wave_reduce(z, Add());
        tmax = ref;
        logz = z > 0.0f || z != z ? logf(z) : __builtin_inff();      // every entry at -inf: all weights 0
    }
    if (MODE != 2 && (a.loss || a.stats)) {
        float kd = 0.0f;
        if (taught) {
#pragma unroll
            for (int u = 0; u < KPT; u++) {
                const int k = tid + u * THREADS;
                if (k < a.k && s.ids[k] >= 0) {
                    const float lp = s.p[k] - tmax - logz, p = expf(lp);
                    const float lq = (zk[u] - top) * invT - lse_t;
                    if (p != 0.0f) kd += p * (lp - lq);
                }
            }
            kd = group_reduce<W>(kd, Add(), s.buf[3]);
        }
        if (tid == 0) {
            float loss = 0.0f;
            if (taught) loss += wd * a.temperature * a.temperature * kd;
            if (named) loss += wl * (lse_1 - (zl - top));
            if (a.loss) a.loss[n] = loss;
            if (a.stats) {
                a.stats[n * 4] = top;
                a.stats[n * 4 + 1] = lse_t;
                a.stats[n * 4 + 2] = lse_1;
                a.stats[n * 4 + 3] = 0.0f;
            }
        }
    }
    if constexpr (MODE == 0) return;

    // the gradient: q and s from the log-sums, then the entries and the label set again
    const float g = a.drow[n];
    const float gd = g * wd * a.temperature, gl = g * wl;
    const float bt = lse_t * LOG2E, b1 = lse_1 * LOG2E;
    auto base = [&](float z) {
        float d = 0.0f;
        if (taught) d = gd * exp2_hw((z - top) * cT - bt);
        if (named) d += gl * exp2_hw((z - top) * LOG2E - b1);
        return d;
    };
    each([&](int i, float *v) {
        float d[P];
#pragma unroll
        for (int j = 0; j < P; j++) d[j] = base(v[j]);
        if (alike) dbody[i] = E::pack(d);
        else
#pragma unroll
            for (int j = 0; j < P; j++) E::store(drow, sh.head + i * P + j, d[j]);
    });
    if (edge >= 0) E::store(drow, edge, base(zedge));
    __syncthreads();                     // the row is written: what follows replaces some of it
#pragma unroll
    for (int u = 0; u < KPT; u++) {
        const int k = tid + u * THREADS;
        if (!taught || k >= a.k || s.ids[k] < 0) continue;
        // an id that comes more than once is its first entry's to write, with all weights
        const int id = s.ids[k];
        float p = 0.0f;
        bool first = true;
        for (int j = 0; j < a.k; j++) {
            if (s.ids[j] != id) continue;
            if (j < k) first = false;
            p += expf(s.p[j] - tmax - logz);
        }
        if (first) E::store(drow, id, base(zk[u]) - gd * p - (named && label == id ? gl : 0.0f));
    }
    if (named && tid == 0) {
        bool in = false;
        if (taught)
            for (int j = 0; j < a.k; j++) in |= s.ids[j] == (int)label;
        if (!in) E::store(drow, label, base(zl) - gl);
    }
}

template <int DT, int MODE, int THREADS, int NC>
void go(const DistillArgs &a, hipStream_t stream)
{
    distill_kernel<DT, MODE, THREADS, NC><<<(unsigned)a.n, THREADS, 0, stream>>>(a);
}

// A row of up to 8 pieces a thread stays in registers (32 of them), with 256 threads for short
// rows; up to 16 where 1024 threads hold it; longer ones are read again.
template <int DT, int MODE>
void pick(const DistillArgs &a, hipStream_t stream)
{
    const int64_t pieces = a.vocab / Elem<DT>::PER16 + 1;
    if (pieces <= 256 * 2) go<DT, MODE, 256, 2>(a, stream);
    else if (pieces <= 256 * 8) go<DT, MODE, 256, 8>(a, stream);
    else if (pieces <= 1024 * 4) go<DT, MODE, 1024, 4>(a, stream);
    else if (pieces <= 1024 * 8) go<DT, MODE, 1024, 8>(a, stream);
    else if (pieces <= 1024 * 16) go<DT, MODE, 1024, 16>(a, stream);
    else go<DT, MODE, 1024, 0>(a, stream);
}

template <int MODE>
hipError_t by_type(const DistillArgs &a, hipStream_t stream)
{
    if (a.n == 0) return hipSuccess;
    if (a.dt == DT_F32) pick<DT_F32, MODE>(a, stream);
    else if (a.dt == DT_BF16) pick<DT_BF16, MODE>(a, stream);
    else pick<DT_F16, MODE>(a, stream);
    return hipGetLastError();
}

}  // namespace

hipError_t distill_forward(const DistillArgs &a, hipStream_t stream)
{
    return a.dlogits ? by_type<1>(a, stream) : by_type<0>(a, stream);
}

hipError_t distill_backward(const DistillArgs &a, hipStream_t stream) { return by_type<2>(a, stream); }

}  // namespace lm
