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
// so that the logits are read once; a row too long for that (over 102400 16-bit or 51200 fp32 logits) is read
// again, three times in all: 4096 rows of 128256 bf16 827 us.  8192 rows of 50257 bf16 with 64 entries each, loss and
// gradient: 362-373 us apart, 369 in place, 4.5 TB/s of the 1.65 GB read and written (a plain copy reaches 4.8); a T
// without a short cut (3) costs no more.  Rows start anywhere: the 16-byte pieces of a row are those of memory, and
// the few elements before the first and behind the last whole piece go one by one.

#include <type_traits>

#include "lm_common.h"
#include "lm_distill.h"

namespace lm {
namespace {

// Rows that together outgrow the last-level cache pass it by (non-temporal accesses).
constexpr int NT = 2;
constexpr int64_t BIG = 128 << 20;

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

__device__ __forceinline__ int64_t index_at(const void *p, int bytes, int64_t i)
{
    return bytes == 8 ? ((const int64_t *)p)[i] : (int64_t)((const int32_t *)p)[i];
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_hw(float x) { return __builtin_amdgcn_logf(x); }

// A row's teacher entries: what each thread would otherwise keep in registers over the passes.
struct RowLds {
    int ids[DISTILL_MAX_K];          // -1: absent
    float t[DISTILL_MAX_K];          // teacher logit, then its log weight
    float p[DISTILL_MAX_K];          // weight
    float z[DISTILL_MAX_K];          // the student's logit
    float w[DISTILL_MAX_K];          // the weights of all entries with this id, at its first entry; elsewhere -1
    float top[16];
    f32x2 sum[16];
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

// The exponents (z - top) c of a row with maximum `top`, as z c - top c in one rounding: what rounding top c loses
// (`lost`) is the same for every value of the row and goes out with the sums.  For it to stay within what an
// exponential holds, c is at most 2^31 / |top|, and 2^29 / |top| for T of 4 and more: beyond that (a small T, or
// logits at the type's end) floats that differ at all differ by 2^5 and more, and weigh nothing beside the largest
// with either c.  In between the limits keep c at T and at 1 that many times apart, so that a power of an
// exponential has lost that power of what the exponential has.
// (Taking the difference first instead: 410 us in place of 371 for 8192 x 50257 bf16.)
struct Exponent {
    float c, topc;
    __device__ __forceinline__ Exponent(float top, float c0, float T)
    {
        const float most = 0x1.fp30f / fminf(fmaxf(T, 1.0f), 4.0f);
        // (2^64 less: no reciprocal below the normal floats)
        c = fminf(c0, most * 0x1p-64f * __builtin_amdgcn_rcpf(fabsf(top) * 0x1p-64f));
        topc = top * c;
    }
    __device__ __forceinline__ float of(float z) const { return __builtin_fmaf(z, c, -topc); }
    __device__ __forceinline__ float lost(float top) const { return of(top) * LN2; }
};

// exp(z - max) of N values from exp((z - max) / T): the T-th power, where T is 1, 2 or 4 (a
// multiplication or two in place of an exponential, which costs four; `pow` 0: formed by itself).
template <int N>
__device__ __forceinline__ void at_one(int pow, const float *e, const float *z, const Exponent &x1, float *o)
{
    if (pow == 0) {
#pragma unroll
        for (int j = 0; j < N; j++) o[j] = exp2_hw(x1.of(z[j]));
    } else {
#pragma unroll
        for (int j = 0; j < N; j++) o[j] = pow == 1 ? e[j] : e[j] * e[j];
        if (pow == 4)
#pragma unroll
            for (int j = 0; j < N; j++) o[j] *= o[j];
    }
}

// Values 4 h ... of a piece.
template <int DT>
__device__ __forceinline__ void unpack4(u32x4 w, int h, float *v)
{
    if constexpr (DT == DT_F32) Elem<DT>::unpack(w, v);
    else {
        const f32x2 a = unpack2<DT>(w[2 * h]), b = unpack2<DT>(w[2 * h + 1]);
        v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1];
    }
}

// The memory from p on, `bytes` of it, for buffer accesses (beyond it: zeros read, nothing written).
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_from(const void *p, uint32_t bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, bytes, 0x00027000);
}

// MODE 0: loss (and stats); 1: loss and gradient; 2: gradient from stats.  NC: pieces a thread
// keeps in registers (0: none, the row is read again).
template <int DT, int MODE, int THREADS, int NC, int WAVES_PER_SIMD, int AUX>
__global__ __launch_bounds__(THREADS, WAVES_PER_SIMD) void distill_kernel(DistillArgs a)
{
    __shared__ RowLds s;
    using E = Elem<DT>;
    constexpr int W = THREADS / 64, P = E::PER16;
    const int tid = threadIdx.x, lane = tid & 63;
    const int64_t n = blockIdx.x;
    const int vocab = (int)a.vocab;
    const RowShape sh = row_shape<DT>(a.logits, n * a.stride, vocab);
    const u32x4 *body = (const u32x4 *)(sh.row + sh.head * E::SIZE);
    const float invT = 1.0f / a.temperature, cT = invT * LOG2E;
    const int pow = a.temperature == 1.0f ? 1 : a.temperature == 2.0f ? 2 : a.temperature == 4.0f ? 4 : 0;

    // the row, on its way while the teacher's entries are looked at
    u32x4 reg[NC ? NC : 1];
    if constexpr (NC > 0) {
        const auto from = buffer_from(body, sh.pieces * 16);
#pragma unroll
        for (int c = 0; c < NC; c++)
            reg[c] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(from, tid * 16, c * THREADS * 16, AUX));
    }
    // each single element of head and tail is one thread's (there are fewer than 2 P of them)
    const int edge = tid < sh.head ? tid : tid < sh.head + sh.tail ? vocab - sh.tail + (tid - sh.head) : -1;
    const float zedge = edge >= 0 ? E::load(sh.row, edge) : -__builtin_inff();

    // whether the row has entries: every wave looks for itself
    bool any = false;
    for (int k = lane; k < a.k; k += 64) {
        const int64_t id = index_at(a.ids, a.id_bytes, n * a.k + k);
        any |= id >= 0 && id < vocab;
    }
    const int64_t label = a.labels ? index_at(a.labels, a.label_bytes, n) : -1;
    const bool named = label >= 0 && label < vocab && a.alpha != 1.0f;
    const bool taught = __any(any) && a.alpha != 0.0f;
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
            if (edge >= 0) E::store(drow, edge, 0.0f);
        }
        return;
    }

    // the first wave forms the teacher's distribution, and keeps the logits at its entries, read before a
    // gradient may overwrite them; the next barrier shows both to the others
    const float zl = named ? E::load(sh.row, label) : 0.0f;
    if (taught && tid < 64) {
        float m = -__builtin_inff();
        for (int k = lane; k < a.k; k += 64) {
            const int64_t id = index_at(a.ids, a.id_bytes, n * a.k + k);
            const bool there = id >= 0 && id < vocab;
            const float t = there ? load_any(a.teacher_dt, a.teacher, n * a.k + k) : -__builtin_inff();
            s.ids[k] = there ? (int)id : -1;
            s.t[k] = t;
            s.z[k] = there ? E::load(sh.row, id) : 0.0f;
            m = Max()(m, t);
        }
        m = wave_reduce(m, Max());
        const float ref = m == -__builtin_inff() ? 0.0f : m;
        float z = 0.0f;
        for (int k = lane; k < a.k; k += 64) z += exp2_hw((s.t[k] - ref) * cT);
        z = wave_reduce(z, Add());
        const float logz = z > 0.0f || z != z ? log2_hw(z) * LN2 : __builtin_inff();     // every entry at -inf: all weights 0
        for (int k = lane; k < a.k; k += 64) {
            s.t[k] = (s.t[k] - ref) * invT - logz;
            s.p[k] = exp2_hw(s.t[k] * LOG2E);
        }
    }

    // a value stays packed between its uses: unpacked once and kept, the row would take twice the
    // registers and the CU half the rows
    auto each = [&](auto f) {            // f(4 values)
        float v[4];
        if constexpr (NC > 0) {
#pragma unroll
            for (int c = 0; c < NC; c++) {
                asm volatile("" : "+v"(reg[c]));
                if (tid + c * THREADS < sh.pieces) {
#pragma unroll
                    for (int h = 0; h < P / 4; h++) {
                        unpack4<DT>(reg[c], h, v);
                        f(v);
                    }
                }
            }
        } else {
            for (int i = tid; i < sh.pieces; i += THREADS) {
                const u32x4 w = body[i];
#pragma unroll
                for (int h = 0; h < P / 4; h++) {
                    unpack4<DT>(w, h, v);
                    f(v);
                }
            }
        }
    };

    float top, lse_t, lse_1;             // the row's maximum and the two log-sums below it
    float inv_t, inv_1;                  // 1 / the sums
    if constexpr (MODE == 2) {
        top = a.stats[n * 4];
        lse_t = a.stats[n * 4 + 1];
        lse_1 = a.stats[n * 4 + 2];
        inv_t = exp2_hw(-lse_t * LOG2E);
        inv_1 = exp2_hw(-lse_1 * LOG2E);
        __syncthreads();                 // the teacher's entries
    } else {
        float m = zedge;
        each([&](float *v) {
#pragma unroll
            for (int j = 0; j < 4; j += 2) m = __builtin_elementwise_maximum(__builtin_elementwise_maximum(v[j], v[j + 1]), m);
        });
        top = group_reduce<W>(m, Max(), s.top);
    }
    const Exponent xT(top, cT, a.temperature), x1(top, LOG2E, 1.0f);
    // an id that comes more than once is its first entry's to write, with all weights
    bool label_there = false;
    if (MODE != 0 && taught)
        for (int k = tid; k < a.k; k += THREADS) {
            const int id = s.ids[k];
            float w = id < 0 ? -1.0f : 0.0f;
            if (id >= 0)
                for (int j = 0; j < a.k; j++)
                    if (s.ids[j] == id) w = j < k ? -1.0f : w < 0.0f ? w : w + s.p[j];
            s.w[k] = w;
            label_there |= id == (int)label;
        }
    if constexpr (MODE != 2) {
        float st = 0.0f, s1 = 0.0f, kd = 0.0f;
        if (edge >= 0) {
            st = exp2_hw(xT.of(zedge));
            if (named) at_one<1>(pow, &st, &zedge, x1, &s1);
        }
        each([&](float *v) {
            float e[4], o[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                e[j] = exp2_hw(xT.of(v[j]));
                st += e[j];
            }
            if (named) {
                at_one<4>(pow, e, v, x1, o);
#pragma unroll
                for (int j = 0; j < 4; j++) s1 += o[j];
            }
        });
        // sum p (log p - (z - top) / T); the log-sum of the student joins when it is known
        if (taught && tid < 64) {
            for (int k = lane; k < a.k; k += 64)
                if (s.p[k] != 0.0f) kd += s.p[k] * (s.t[k] - (s.z[k] - top) * invT);
            kd = wave_reduce(kd, Add());
        }
        st = wave_reduce(st, Add());
        if (named) s1 = wave_reduce(s1, Add());
        if (lane == 0) s.sum[tid >> 6] = f32x2{st, s1};
        __syncthreads();
        st = s1 = 0.0f;
        for (int w = 0; w < W; w++) {
            const f32x2 t = s.sum[w];
            st += t[0];
            s1 += t[1];
        }
        lse_t = log2_hw(st) * LN2;
        lse_1 = named ? log2_hw(s1) * LN2 : 0.0f;
        inv_t = 1.0f / st;
        inv_1 = 1.0f / s1;
        if (tid == 0) {
            float loss = 0.0f, psum = 0.0f;
            if (taught) {
                // (weights that the exponential rounded to 0 leave the sum at 1, all of them at 0)
                for (int k = 0; k < a.k && psum == 0.0f; k++) psum += s.p[k];
                loss = wd * a.temperature * a.temperature * (psum == 0.0f ? 0.0f : kd + (lse_t - xT.lost(top)));
            }
            if (named) loss += wl * (lse_1 - x1.lost(top) - (zl - top));
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
    const float qd = taught ? gd * inv_t : 0.0f, ql = named ? gl * inv_1 : 0.0f;
    auto gradients = [&]<int N>(const float *z, float *d) {
        float o[N];
#pragma unroll
        for (int j = 0; j < N; j++) d[j] = exp2_hw(xT.of(z[j]));
        if (named) {
            at_one<N>(pow, d, z, x1, o);
#pragma unroll
            for (int j = 0; j < N; j++) d[j] = qd * d[j] + ql * o[j];
        } else {
#pragma unroll
            for (int j = 0; j < N; j++) d[j] *= qd;
        }
    };
    auto base = [&](float z) {
        float d;
        gradients.template operator()<1>(&z, &d);
        return d;
    };
    auto piece = [&](u32x4 w) {
        float v[4], d[P];
#pragma unroll
        for (int h = 0; h < P / 4; h++) {
            unpack4<DT>(w, h, v);
            gradients.template operator()<4>(v, d + 4 * h);
        }
        return E::pack(d);
    };
    if (NC > 0 && alike) {
        const auto to = buffer_from(dbody, sh.pieces * 16);
#pragma unroll
        for (int c = 0; c < NC; c++) {
            asm volatile("" : "+v"(reg[c]));
            __builtin_amdgcn_raw_buffer_store_b128(piece(reg[c]), to, tid * 16, c * THREADS * 16, AUX);
        }
    } else {
        // (the logits are where they were: rows that start otherwise in their 16 bytes are not written in place)
        for (int i = tid; i < sh.pieces; i += THREADS) {
            const u32x4 w = piece(body[i]);
            if (alike) dbody[i] = w;
            else {
                float d[P];
                E::unpack(w, d);
#pragma unroll
                for (int j = 0; j < P; j++) E::store(drow, sh.head + i * P + j, d[j]);
            }
        }
    }
    if (edge >= 0) E::store(drow, edge, base(zedge));
    const bool listed = __syncthreads_or(label_there);     // (and the row is written: what follows replaces some of it)
    if (taught)
        for (int k = tid; k < a.k; k += THREADS)
            if (!(s.w[k] < 0.0f)) {
                const int id = s.ids[k];
                E::store(drow, id, base(s.z[k]) - gd * s.w[k] - (named && label == id ? gl : 0.0f));
            }
    if (named && !listed && tid == 0) E::store(drow, label, base(zl) - gl);
}

template <int DT, int MODE, int THREADS, int NC, int WAVES_PER_SIMD, int AUX>
void go(const DistillArgs &a, hipStream_t stream)
{
    distill_kernel<DT, MODE, THREADS, NC, WAVES_PER_SIMD, AUX><<<(unsigned)a.n, THREADS, 0, stream>>>(a);
}

// How many threads hold a row, and how many of its pieces each.  With rows for every CU, few threads with
// many registers: three rows of 512 threads and 13 pieces run on a CU, whose loads, sums and stores overlap
// (8192 rows of 50257: 368 us; two of 14 pieces 425).  With fewer than two rows a CU, 1024 threads, which
// bring one row in sooner (7 rows of 32000 fp32: loss 6.3 us, its gradient 6.9 us).
template <int DT, int MODE>
void pick(const DistillArgs &a, hipStream_t stream)
{
    const int64_t pieces = a.vocab / Elem<DT>::PER16 + 1;
    const bool few = a.n < 512, big = a.n * pieces * 16 > BIG;
    if (pieces <= 256 * 2) go<DT, MODE, 256, 2, 6, 0>(a, stream);
    else if (pieces <= 256 * 8 && !(few && pieces > 1024)) big ? go<DT, MODE, 256, 8, 6, NT>(a, stream) : go<DT, MODE, 256, 8, 6, 0>(a, stream);
    else if (few && pieces <= 1024 * 4) go<DT, MODE, 1024, 4, 4, 0>(a, stream);
    else if (few && pieces <= 1024 * 13) go<DT, MODE, 1024, 13, 4, 0>(a, stream);
    else if (pieces <= 512 * 13) big ? go<DT, MODE, 512, 13, 6, NT>(a, stream) : go<DT, MODE, 512, 13, 6, 0>(a, stream);
    else if (pieces <= 512 * 25) big ? go<DT, MODE, 512, 25, 4, NT>(a, stream) : go<DT, MODE, 512, 25, 4, 0>(a, stream);
    else go<DT, MODE, 1024, 0, 4, 0>(a, stream);
}

// A launch ends at 2^32 threads: more rows than that take several (a second dimension of the grid cost the kernel
// registers, 392 us in place of 368).
constexpr int64_t ROWS = 1 << 21;

// The rows from `first` on, `n` of them.
DistillArgs rows_of(DistillArgs a, int64_t first, int64_t n)
{
    auto on = [](auto *&p, int64_t bytes) {
        if (p) p = (std::remove_reference_t<decltype(p)>)((char *)p + bytes);
    };
    const int64_t z = a.dt == DT_F32 ? 4 : 2, t = a.teacher_dt == DT_F32 ? 4 : 2;
    a.n = n;
    on(a.logits, first * a.stride * z);
    on(a.teacher, first * a.k * t);
    on(a.ids, first * a.k * a.id_bytes);
    on(a.labels, first * a.label_bytes);
    on(a.loss, first * 4);
    on(a.stats, first * 16);
    on(a.drow, first * 4);
    on(a.dlogits, first * a.dstride * z);
    return a;
}

template <int MODE>
hipError_t by_type(const DistillArgs &all, hipStream_t stream)
{
    hipError_t e = hipSuccess;
    for (int64_t first = 0; first < all.n && e == hipSuccess; first += ROWS) {
        const DistillArgs a = rows_of(all, first, all.n - first < ROWS ? all.n - first : ROWS);
        if (a.dt == DT_F32) pick<DT_F32, MODE>(a, stream);
        else if (a.dt == DT_BF16) pick<DT_BF16, MODE>(a, stream);
        else pick<DT_F16, MODE>(a, stream);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace

hipError_t distill_forward(const DistillArgs &a, hipStream_t stream)
{
    return a.dlogits ? by_type<1>(a, stream) : by_type<0>(a, stream);
}

hipError_t distill_backward(const DistillArgs &a, hipStream_t stream) { return by_type<2>(a, stream); }

}  // namespace lm
