// lm_norm_kernel.h -- the norms before and after a block, fused with its gate and the residual sum.
//
//   n1 = norm(block; w1, c1)   (or block itself)          r = a x + gate * n1
//   h  = norm(r; w2, c2)                                    norm(y) = yh w + c
//   yh = y rsqrt(mean(y^2) + eps)                           (layer norms: y - mean(y) for y)
//
// Backward, with t = dy w for a norm of output gradient dy:
//   dy_in = rs (t - yh mean(t yh) [- mean(t)]),   dw = sum dy yh,   dc = sum dy
//   dR = dr + norm'(dh),  dx = a dR,  dgate = sum dR n1,  dblock = norm'(gate dR)
//
// Bound by memory: forward reads x and block and writes r and h; backward reads x, block, dr and
// dh and writes dx and dblock (r is formed again from x and block, which costs no more reading
// than r itself and is not rounded).  A row lives in registers, at most 16 columns a thread, so
// every array is touched once; rows of up to 1024 columns are one wave's, longer ones a
// workgroup's.  Column sums stay in registers over all rows of a workgroup, then go to fp32
// partial rows that a second kernel adds in order (no float atomics).
#pragma once
#include "lm_common.h"
#include "lm_norm.h"

namespace lm {
namespace {

constexpr int COLS = 16;           // columns a thread holds

// A piece of a weight: of the rows' type or fp32.
template <int DT, int N, bool RAGGED>
__device__ __forceinline__ void load_w(int dt, const void *p, int64_t i, float *v)
{
    if (DT == DT_F32 || dt == DT_F32) load_n<DT_F32, N, RAGGED>(p, i, v);
    else load_n<DT, N, RAGGED>(p, i, v);
}

// A thread's columns: NCH pieces of VEC.  RAGGED: rows start at any element and their length need
// not be a multiple of VEC; the last piece of a row then ends with the row and overlaps the one
// before it by `skip` columns, which are worked out twice (the same bits) and counted once.
template <int VEC, bool RAGGED>
struct Columns {
    static constexpr int NCH = COLS / VEC;
    int col[NCH], skip[NCH];
    bool live[NCH];

    __device__ __forceinline__ Columns(int dim, int threads, int lane)
    {
#pragma unroll
        for (int c = 0; c < NCH; c++) {
            const int at = (c * threads + lane) * VEC;
            live[c] = at < dim;
            col[c] = RAGGED ? min(at, dim - VEC) : at;
            skip[c] = at - col[c];
        }
    }
    __device__ __forceinline__ bool counts(int c, int k) const { return live[c] && (!RAGGED || k >= skip[c]); }
};

// Piece c of a row: 16 bytes, or of an overlapping piece the columns that are its own.
template <int DT, int VEC, bool RAGGED>
__device__ __forceinline__ void store_piece(void *p, int64_t row, const Columns<VEC, RAGGED> &cs, int c, const float *v)
{
    if (!RAGGED || cs.skip[c] == 0) store_n<DT, VEC, RAGGED>(p, row + cs.col[c], v);
    else
#pragma unroll
        for (int k = 0; k < VEC; k++)
            if (k >= cs.skip[c]) Elem<DT>::store(p, row + cs.col[c] + k, v[k]);
}

// Sums of two values over a row's threads.  ROW_WAVES 1: the row is a wave's.
template <bool WAVE_ROW>
__device__ __forceinline__ f32x2 row_sum2(f32x2 v, f32x2 *buf)
{
    v[0] = wave_reduce(v[0], Add());
    v[1] = wave_reduce(v[1], Add());
    if constexpr (!WAVE_ROW) {
        if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
        __syncthreads();
        v = buf[0];
        for (int w = 1; w < (int)blockDim.x / 64; w++) v += buf[w];
    }
    return v;
}

template <bool WAVE_ROW>
__device__ __forceinline__ float row_sum(float v, f32x2 *buf)
{
    v = wave_reduce(v, Add());
    if constexpr (!WAVE_ROW) {
        if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6][0] = v;
        __syncthreads();
        v = buf[0][0];
        for (int w = 1; w < (int)blockDim.x / 64; w++) v += buf[w][0];
    }
    return v;
}

// Mean (layer norms) and 1/deviation of a row in registers: the deviation from the mean itself,
// not from a difference of large sums.
template <int VEC, bool WAVE_ROW, bool LAYER, bool RAGGED>
__device__ __forceinline__ f32x2 moments(const float *v, const Columns<VEC, RAGGED> &cs, float inv_dim, float eps, f32x2 (*buf)[16])
{
    float mean = 0.0f;
    if constexpr (LAYER) {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < COLS; k++) s += cs.counts(k / VEC, k % VEC) ? v[k] : 0.0f;
        mean = row_sum<WAVE_ROW>(s, buf[0]) * inv_dim;
    }
    float q = 0.0f;
#pragma unroll
    for (int k = 0; k < COLS; k++) {
        const float d = v[k] - mean;
        q += cs.counts(k / VEC, k % VEC) ? d * d : 0.0f;
    }
    q = row_sum<WAVE_ROW>(q, buf[1]) * inv_dim;
    return f32x2{mean, 1.0f / sqrtf(q + eps)};
}

template <int DT, int MAXT, bool POST, bool LAYER, bool RAGGED>
__global__ __launch_bounds__(MAXT == 64 ? 256 : MAXT) void norm_fwd_kernel(NormArgs a)
{
    constexpr bool WAVE_ROW = MAXT == 64;
    constexpr int VEC = Elem<DT>::PER16, NCH = COLS / VEC;
    __shared__ f32x2 buf[4][16];
    const int threads = WAVE_ROW ? 64 : blockDim.x;
    const int lane = WAVE_ROW ? threadIdx.x & 63 : threadIdx.x;
    const int dim = (int)a.dim;
    const float inv_dim = 1.0f / (float)dim;
    const int64_t step = (int64_t)gridDim.x * (WAVE_ROW ? 4 : 1);
    const int64_t rows_per_group = a.gate ? a.n / a.groups : 1;
    const Columns<VEC, RAGGED> cs(dim, threads, lane);
    const auto &col = cs.col;
    const auto &live = cs.live;
    for (int64_t row = WAVE_ROW ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x; row < a.n; row += step) {
        float x[COLS], y[COLS];
#pragma unroll
        for (int c = 0; c < NCH; c++) {
#pragma unroll
            for (int k = 0; k < VEC; k++) x[c * VEC + k] = y[c * VEC + k] = 0.0f;
            if (live[c]) {
                load_n<DT, VEC, RAGGED>(a.x, row * a.x_stride + col[c], x + c * VEC);
                load_n<DT, VEC, RAGGED>(a.block, row * a.block_stride + col[c], y + c * VEC);
            }
        }
        f32x2 m1 = {0.0f, 0.0f};
        if constexpr (POST) {
            m1 = moments<VEC, WAVE_ROW, LAYER, RAGGED>(y, cs, inv_dim, a.eps, buf);
#pragma unroll
            for (int c = 0; c < NCH; c++)
                if (live[c]) {
                    float w[VEC], b[VEC] = {};
                    load_w<DT, VEC, RAGGED>(a.weight_dt, a.post_weight, col[c], w);
                    if (a.post_bias) load_w<DT, VEC, RAGGED>(a.weight_dt, a.post_bias, col[c], b);
#pragma unroll
                    for (int k = 0; k < VEC; k++) y[c * VEC + k] = (y[c * VEC + k] - m1[0]) * m1[1] * w[k] + b[k];
                }
        }
        const int64_t gate_row = a.gate && a.groups > 1 ? row / rows_per_group * a.dim : 0;
#pragma unroll
        for (int c = 0; c < NCH; c++) {
            float g[VEC];
            if (a.gate && live[c]) load_w<DT, VEC, RAGGED>(a.weight_dt, a.gate, gate_row + col[c], g);
#pragma unroll
            for (int k = 0; k < VEC; k++) {
                const int i = c * VEC + k;
                x[i] = a.residual_scale * x[i] + (a.gate ? (live[c] ? g[k] * y[i] : 0.0f) : y[i]);
            }
            if (live[c]) store_piece<DT, VEC, RAGGED>(a.r, row * a.dim, cs, c, x + c * VEC);
        }
        const f32x2 m2 = moments<VEC, WAVE_ROW, LAYER, RAGGED>(x, cs, inv_dim, a.eps, buf + 2);
#pragma unroll
        for (int c = 0; c < NCH; c++)
            if (live[c]) {
                float w[VEC], b[VEC] = {}, h[VEC];
                load_w<DT, VEC, RAGGED>(a.weight_dt, a.pre_weight, col[c], w);
                if (a.pre_bias) load_w<DT, VEC, RAGGED>(a.weight_dt, a.pre_bias, col[c], b);
#pragma unroll
                for (int k = 0; k < VEC; k++) h[k] = (x[c * VEC + k] - m2[0]) * m2[1] * w[k] + b[k];
                store_piece<DT, VEC, RAGGED>(a.h, row * a.dim, cs, c, h);
            }
        if (lane == 0) *(f32x4 *)(a.stats + row * 4) = f32x4{m1[0], m1[1], m2[0], m2[1]};
        if constexpr (!WAVE_ROW) __syncthreads();          // the reductions' buffers are free again
    }
}

template <int DT, int MAXT, bool POST, bool LAYER, bool RAGGED>
__global__ __launch_bounds__(MAXT == 64 ? 256 : MAXT) void norm_bwd_kernel(NormArgs a, NormSplit sp)
{
    constexpr bool WAVE_ROW = MAXT == 64;
    constexpr int VEC = Elem<DT>::PER16, NCH = COLS / VEC, WORKERS = WAVE_ROW ? 4 : 1;
    __shared__ f32x2 buf[2][16];
    __shared__ float join[WAVE_ROW ? 3 * 1024 : 1];
    const int threads = WAVE_ROW ? 64 : blockDim.x;
    const int lane = WAVE_ROW ? threadIdx.x & 63 : threadIdx.x;
    const int wave = WAVE_ROW ? threadIdx.x >> 6 : 0;
    const int dim = (int)a.dim;
    const float inv_dim = 1.0f / (float)dim;
    const int64_t rpg = a.n / a.groups;
    const Columns<VEC, RAGGED> cs(dim, threads, lane);
    const auto &col = cs.col;
    const auto &live = cs.live;
    float dpw[COLS] = {}, dpb[COLS] = {}, dqw[COLS] = {}, dqb[COLS] = {}, dg[COLS] = {};
    float *const part = a.workspace;                       // [5][wgs][dim]
    const int64_t kind = (int64_t)sp.wgs * a.dim;

    // the worker's rows: groups g, g + gstep, ...; in each, rows first, first + rstep, ... below last
    int64_t g = blockIdx.x, gstep = a.groups, first = 0, last = rpg, rstep = 1;
    if (sp.per_group) {
        g = blockIdx.x / sp.per_group;
        const int64_t each = (rpg + sp.per_group - 1) / sp.per_group;
        first = (blockIdx.x % sp.per_group) * each;
        last = min(rpg, first + each);
        first += wave;
        rstep = WORKERS;
    } else {
        g = (int64_t)blockIdx.x * WORKERS + wave;
        gstep = (int64_t)sp.wgs * WORKERS;
    }
    for (; g < a.groups; g += gstep) {
        for (int64_t i = first; i < last; i += rstep) {
            const int64_t row = g * rpg + i;
            const f32x4 st = *(const f32x4 *)(a.stats + row * 4);
            float x[COLS], y[COLS], d[COLS], r[COLS];
#pragma unroll
            for (int c = 0; c < NCH; c++) {
#pragma unroll
                for (int k = 0; k < VEC; k++) x[c * VEC + k] = y[c * VEC + k] = d[c * VEC + k] = r[c * VEC + k] = 0.0f;
                if (live[c]) {
                    load_n<DT, VEC, RAGGED>(a.x, row * a.x_stride + col[c], x + c * VEC);
                    load_n<DT, VEC, RAGGED>(a.block, row * a.block_stride + col[c], y + c * VEC);
                    load_n<DT, VEC, RAGGED>(a.dh, row * a.dh_stride + col[c], d + c * VEC);
                    if (a.dr) load_n<DT, VEC, RAGGED>(a.dr, row * a.dr_stride + col[c], r + c * VEC);
                }
            }
            // y: block normalised; x: r normalised; d: dh times the weight
            f32x2 s = {0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < NCH; c++)
                if (live[c]) {
                    float w1[VEC], b1[VEC] = {}, gt[VEC], w2[VEC];
                    if constexpr (POST) {
                        load_w<DT, VEC, RAGGED>(a.weight_dt, a.post_weight, col[c], w1);
                        if (a.post_bias) load_w<DT, VEC, RAGGED>(a.weight_dt, a.post_bias, col[c], b1);
                    }
                    if (a.gate) load_w<DT, VEC, RAGGED>(a.weight_dt, a.gate, g * a.dim + col[c], gt);
                    load_w<DT, VEC, RAGGED>(a.weight_dt, a.pre_weight, col[c], w2);
#pragma unroll
                    for (int k = 0; k < VEC; k++) {
                        const int j = c * VEC + k;
                        float n1 = y[j];
                        if constexpr (POST) {
                            y[j] = (y[j] - st[0]) * st[1];
                            n1 = y[j] * w1[k] + b1[k];
                        }
                        const float R = a.residual_scale * x[j] + (a.gate ? gt[k] * n1 : n1);
                        x[j] = (R - st[2]) * st[3];
                        dpw[j] += d[j] * x[j];
                        if constexpr (LAYER) dpb[j] += d[j];
                        d[j] *= w2[k];
                        if (cs.counts(c, k)) {
                            s[0] += d[j] * x[j];
                            if constexpr (LAYER) s[1] += d[j];
                        }
                    }
                }
            s = row_sum2<WAVE_ROW>(s, buf[0]) * inv_dim;
            f32x2 s1 = {0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < NCH; c++)
                if (live[c]) {
                    float w1[VEC], b1[VEC] = {}, gt[VEC], dx[VEC];
                    if constexpr (POST) {
                        load_w<DT, VEC, RAGGED>(a.weight_dt, a.post_weight, col[c], w1);
                        if (a.post_bias) load_w<DT, VEC, RAGGED>(a.weight_dt, a.post_bias, col[c], b1);
                    }
                    if (a.gate) load_w<DT, VEC, RAGGED>(a.weight_dt, a.gate, g * a.dim + col[c], gt);
#pragma unroll
                    for (int k = 0; k < VEC; k++) {
                        const int j = c * VEC + k;
                        float R = d[j] - x[j] * s[0];
                        if constexpr (LAYER) R -= s[1];
                        R = r[j] + R * st[3];
                        dx[k] = a.residual_scale * R;
                        if (a.gate) {
                            dg[j] += R * (POST ? y[j] * w1[k] + b1[k] : y[j]);
                            R *= gt[k];
                        }
                        d[j] = R;                          // the gradient of n1
                        if constexpr (POST) {
                            dqw[j] += R * y[j];
                            if constexpr (LAYER) dqb[j] += R;
                            d[j] = R * w1[k];
                            if (cs.counts(c, k)) {
                                s1[0] += d[j] * y[j];
                                if constexpr (LAYER) s1[1] += d[j];
                            }
                        }
                    }
                    store_piece<DT, VEC, RAGGED>(a.dx, row * a.dim, cs, c, dx);
                }
            if constexpr (POST) s1 = row_sum2<WAVE_ROW>(s1, buf[1]) * inv_dim;
            else if constexpr (!WAVE_ROW) __syncthreads();  // buf[0] is written again by the next row
#pragma unroll
            for (int c = 0; c < NCH; c++)
                if (live[c]) {
                    if constexpr (POST) {
#pragma unroll
                        for (int k = 0; k < VEC; k++) {
                            const int j = c * VEC + k;
                            float t = d[j] - y[j] * s1[0];
                            if constexpr (LAYER) t -= s1[1];
                            d[j] = t * st[1];
                        }
                    }
                    store_piece<DT, VEC, RAGGED>(a.dblock, row * a.dim, cs, c, d + c * VEC);
                }
            if constexpr (POST && !WAVE_ROW) __syncthreads();   // and so is buf[1]
        }
        if (a.gate && !sp.per_group) {
#pragma unroll
            for (int c = 0; c < NCH; c++)
#pragma unroll
                for (int k = 0; k < VEC; k++) {
                    if (cs.counts(c, k)) store_any(a.weight_dt, a.dgate, g * a.dim + col[c] + k, dg[c * VEC + k]);
                    dg[c * VEC + k] = 0.0f;
                }
        }
    }

    auto put = [&](float *acc, int which) {
        if constexpr (WAVE_ROW) {
            // the other three waves' sums through LDS, added in their order
            __syncthreads();
            if (wave > 0)
#pragma unroll
                for (int j = 0; j < COLS; j++) join[(wave - 1) * 1024 + j * 64 + lane] = acc[j];
            __syncthreads();
            if (wave > 0) return;
#pragma unroll
            for (int j = 0; j < COLS; j++)
                for (int w = 0; w < 3; w++) acc[j] += join[w * 1024 + j * 64 + lane];
        }
#pragma unroll
        for (int c = 0; c < NCH; c++)
            if (live[c]) {
                float *to = part + which * kind + blockIdx.x * a.dim + col[c];
#pragma unroll
                for (int k = 0; k < VEC; k++)
                    if (cs.counts(c, k)) to[k] = acc[c * VEC + k];
            }
    };
    put(dpw, 0);
    if (a.dpre_bias) put(dpb, 1);
    if constexpr (POST) {
        put(dqw, 2);
        if (a.dpost_bias) put(dqb, 3);
    }
    if (a.gate && sp.per_group) put(dg, 4);
}

template <int DT, int MAXT, bool POST, bool LAYER, bool RAGGED>
void go(const NormArgs &a, const NormSplit &sp, bool backward, hipStream_t stream)
{
    const int threads = MAXT == 64 ? 256 : (int)((a.dim + COLS * 64 - 1) / (COLS * 64) * 64);
    if (!backward) {
        const int64_t rows = MAXT == 64 ? (a.n + 3) / 4 : a.n;
        norm_fwd_kernel<DT, MAXT, POST, LAYER, RAGGED><<<(unsigned)(rows < 1 << 20 ? rows : 1 << 20), threads, 0, stream>>>(a);
    } else {
        norm_bwd_kernel<DT, MAXT, POST, LAYER, RAGGED><<<sp.wgs, threads, 0, stream>>>(a, sp);
    }
}

template <int DT, int MAXT, bool RAGGED>
void by_kind(const NormArgs &a, const NormSplit &sp, bool backward, hipStream_t stream)
{
    if (a.post_weight) {
        if (a.layer) go<DT, MAXT, true, true, RAGGED>(a, sp, backward, stream);
        else go<DT, MAXT, true, false, RAGGED>(a, sp, backward, stream);
    } else {
        if (a.layer) go<DT, MAXT, false, true, RAGGED>(a, sp, backward, stream);
        else go<DT, MAXT, false, false, RAGGED>(a, sp, backward, stream);
    }
}

template <int DT, bool RAGGED>
void by_width(const NormArgs &a, const NormSplit &sp, bool backward, hipStream_t stream)
{
    if (a.dim <= 1024) by_kind<DT, 64, RAGGED>(a, sp, backward, stream);
    else if (a.dim <= 4096) by_kind<DT, 256, RAGGED>(a, sp, backward, stream);
    else by_kind<DT, 512, RAGGED>(a, sp, backward, stream);
}

}  // namespace

template <int DT>
hipError_t norm_run(const NormArgs &a, const NormSplit &sp, bool ragged, bool backward, hipStream_t stream)
{
    ragged ? by_width<DT, true>(a, sp, backward, stream) : by_width<DT, false>(a, sp, backward, stream);
    return hipGetLastError();
}

}  // namespace lm
