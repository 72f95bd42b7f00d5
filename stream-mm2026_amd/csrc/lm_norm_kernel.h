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
// than r itself and is not rounded).  A row lives in registers, 8 columns a thread, so every array is
// touched once; the next row's arrays are on their way meanwhile, and the weights stay in registers
// too: loaded row by row they would be waited for behind the next row's (loads return in order).
// Rows of up to 512 columns are one wave's, of up to 1024 two waves', longer ones a workgroup's.
// Column sums stay in registers over all rows of a workgroup, then go to fp32 partial rows that a
// second kernel adds in order (no float atomics).  16384 rows of 4096 bf16: forward 92-97 us (5.7 TB/s),
// backward 172-180 us (4.6 TB/s; a large copy reaches 4.8); 8192 of 768: 12 and 18 us.
#pragma once
#include "lm_common.h"
#include "lm_norm.h"

namespace lm {
namespace {

constexpr int COLS = 8;            // columns a thread holds

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
    char *const at = (char *)p + row * Elem<DT>::SIZE + (uint32_t)(cs.col[c] * Elem<DT>::SIZE);
    if (!RAGGED || cs.skip[c] == 0) store_n<DT, VEC, RAGGED>(at, 0, v);
    else
#pragma unroll
        for (int k = 0; k < VEC; k++)
            if (k >= cs.skip[c]) Elem<DT>::store(at, k, v[k]);
}

// A row's pieces as they come from memory, so that the next row's can be on their way while this one
// is worked on.
template <int DT, int VEC, bool RAGGED>
struct RawRow {
    static constexpr int NCH = COLS / VEC;
    u32x4 w[NCH];

    __device__ __forceinline__ void load(const void *p, int64_t row, const Columns<VEC, RAGGED> &cs)
    {
        using W = typename Pick<RAGGED, u32x4_any, u32x4>::T;
#pragma unroll
        for (int c = 0; c < NCH; c++) {
            w[c] = u32x4{0, 0, 0, 0};
            if (cs.live[c]) w[c] = *(const W *)((const char *)p + row * Elem<DT>::SIZE + (uint32_t)(cs.col[c] * Elem<DT>::SIZE));
        }
    }
    __device__ __forceinline__ void unpack(float *v) const
    {
#pragma unroll
        for (int c = 0; c < NCH; c++) Elem<DT>::unpack(w[c], v + c * VEC);
    }
};

// The thread's columns of a weight, kept as they come from memory: of the rows' type or fp32.
template <int DT, bool WF32, int VEC, bool RAGGED>
struct RawWeight {
    static constexpr int WDT = WF32 ? DT_F32 : DT, NCH = COLS / VEC, PER = VEC * Elem<WDT>::SIZE / 16;
    u32x4 w[NCH * PER];

    __device__ __forceinline__ void load(const void *p, int64_t at, const Columns<VEC, RAGGED> &cs)
    {
        using W = typename Pick<RAGGED, u32x4_any, u32x4>::T;
#pragma unroll
        for (int c = 0; c < NCH; c++)
#pragma unroll
            for (int k = 0; k < PER; k++) {
                w[c * PER + k] = u32x4{0, 0, 0, 0};
                if (p && cs.live[c]) w[c * PER + k] = ((const W *)((const char *)p + (at + cs.col[c]) * Elem<WDT>::SIZE))[k];
            }
    }
    // (loads first waited for inside the row loop would be waited for there on every turn)
    __device__ __forceinline__ void landed()
    {
#pragma unroll
        for (int i = 0; i < NCH * PER; i++) asm volatile("" : "+v"(w[i]));
    }
    __device__ __forceinline__ void unpack(int c, float *v) const
    {
#pragma unroll
        for (int k = 0; k < PER; k++) Elem<WDT>::unpack(w[c * PER + k], v + k * Elem<WDT>::PER16);
    }
};

// How a workgroup's waves share rows: WPR 1 or 2 waves a row (and so several rows at a time), or
// all of them (0).
template <int WPR>
struct Shares {
    int rows, mine, threads, lane, wave0, waves;       // rows at a time, which of them, the row's threads and waves
    __device__ __forceinline__ Shares()
    {
        threads = WPR ? WPR * 64 : blockDim.x;
        rows = WPR ? (int)blockDim.x / threads : 1;
        mine = WPR ? __builtin_amdgcn_readfirstlane((int)threadIdx.x / threads) : 0;
        lane = threadIdx.x - mine * threads;
        waves = threads / 64;
        wave0 = mine * waves;
    }
    // The sum of two values over the row's threads.  `buf` (one value a wave) is free again two
    // barriers on.
    __device__ __forceinline__ f32x2 sum2(f32x2 v, f32x2 *buf) const
    {
        v[0] = wave_reduce(v[0], Add());
        v[1] = wave_reduce(v[1], Add());
        if constexpr (WPR != 1) {
            if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
            __syncthreads();
            v = buf[wave0];
            for (int w = 1; w < waves; w++) v += buf[wave0 + w];
        }
        return v;
    }
    __device__ __forceinline__ float sum(float v, f32x2 *buf) const
    {
        v = wave_reduce(v, Add());
        if constexpr (WPR != 1) {
            if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6][0] = v;
            __syncthreads();
            v = buf[wave0][0];
            for (int w = 1; w < waves; w++) v += buf[wave0 + w][0];
        }
        return v;
    }
};

// Mean (layer norms) and 1/deviation of a row in registers: the deviation from the mean itself,
// not from a difference of large sums.
template <int VEC, int WPR, bool LAYER, bool RAGGED>
__device__ __forceinline__ f32x2 moments(const float *v, const Columns<VEC, RAGGED> &cs, const Shares<WPR> &sh, float inv_dim, float eps,
                                         f32x2 (*buf)[16])
{
    float mean = 0.0f;
    if constexpr (LAYER) {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < COLS; k++) s += cs.counts(k / VEC, k % VEC) ? v[k] : 0.0f;
        mean = sh.sum(s, buf[0]) * inv_dim;
    }
    float q = 0.0f;
#pragma unroll
    for (int k = 0; k < COLS; k++) {
        const float d = v[k] - mean;
        q += cs.counts(k / VEC, k % VEC) ? d * d : 0.0f;
    }
    q = sh.sum(q, buf[1]) * inv_dim;
    return f32x2{mean, 1.0f / sqrtf(q + eps)};
}

template <int DT, bool WF32, int WPR, int MAXT, bool POST, bool LAYER, bool RAGGED>
__global__ __launch_bounds__(MAXT) void norm_fwd_kernel(NormArgs a)
{
    constexpr int VEC = Elem<DT>::PER16, NCH = COLS / VEC;
    __shared__ f32x2 buf[4][16];
    const Shares<WPR> sh;
    const int dim = (int)a.dim;
    const float inv_dim = 1.0f / (float)dim;
    const int64_t step = (int64_t)gridDim.x * sh.rows, rows_per_group = a.gate ? a.n / a.groups : 1;
    const Columns<VEC, RAGGED> cs(dim, sh.threads, sh.lane);
    RawWeight<DT, WF32, VEC, RAGGED> w1, b1, w2, b2, gt;
    if constexpr (POST) {
        w1.load(a.post_weight, 0, cs);
        w1.landed();
        if constexpr (LAYER) b1.load(a.post_bias, 0, cs), b1.landed();
    }
    w2.load(a.pre_weight, 0, cs);
    w2.landed();
    if constexpr (LAYER) b2.load(a.pre_bias, 0, cs), b2.landed();
    gt.load(a.groups > 1 ? nullptr : a.gate, 0, cs);
    gt.landed();
    int64_t row = (int64_t)blockIdx.x * sh.rows + sh.mine;
    RawRow<DT, VEC, RAGGED> xw, yw;
    if (row < a.n) {
        xw.load(a.x, row * a.x_stride, cs);
        yw.load(a.block, row * a.block_stride, cs);
    }
    // every row of the workgroup takes as many turns: they share barriers
    for (int64_t first = (int64_t)blockIdx.x * sh.rows; first < a.n; first += step, row += step) {
        const bool there = row < a.n;
        float x[COLS], y[COLS];
        xw.unpack(x);
        yw.unpack(y);
        if (a.groups > 1 && there) gt.load(a.gate, row / rows_per_group * a.dim, cs);
        if (row + step < a.n) {
            xw.load(a.x, (row + step) * a.x_stride, cs);
            yw.load(a.block, (row + step) * a.block_stride, cs);
        }
        f32x2 m1 = {0.0f, 0.0f};
        if constexpr (POST) {
            m1 = moments<VEC, WPR, LAYER, RAGGED>(y, cs, sh, inv_dim, a.eps, buf);
#pragma unroll
            for (int c = 0; c < NCH; c++) {
                float w[VEC], b[VEC] = {};
                w1.unpack(c, w);
                if constexpr (LAYER) b1.unpack(c, b);
#pragma unroll
                for (int k = 0; k < VEC; k++) y[c * VEC + k] = (y[c * VEC + k] - m1[0]) * m1[1] * w[k] + b[k];
            }
        }
#pragma unroll
        for (int c = 0; c < NCH; c++) {
            float g[VEC];
            gt.unpack(c, g);
#pragma unroll
            for (int k = 0; k < VEC; k++) {
                const int i = c * VEC + k;
                x[i] = a.residual_scale * x[i] + (a.gate ? g[k] * y[i] : y[i]);
            }
            if (there && cs.live[c]) store_piece<DT, VEC, RAGGED>(a.r, row * a.dim, cs, c, x + c * VEC);
        }
        const f32x2 m2 = moments<VEC, WPR, LAYER, RAGGED>(x, cs, sh, inv_dim, a.eps, buf + 2);
#pragma unroll
        for (int c = 0; c < NCH; c++) {
            float w[VEC], b[VEC] = {}, h[VEC];
            w2.unpack(c, w);
            if constexpr (LAYER) b2.unpack(c, b);
#pragma unroll
            for (int k = 0; k < VEC; k++) h[k] = (x[c * VEC + k] - m2[0]) * m2[1] * w[k] + b[k];
            if (there && cs.live[c]) store_piece<DT, VEC, RAGGED>(a.h, row * a.dim, cs, c, h);
        }
        if (there && sh.lane == 0) *(f32x4 *)(a.stats + row * 4) = f32x4{m1[0], m1[1], m2[0], m2[1]};
        if constexpr (WPR != 1) __syncthreads();           // the reductions' buffers are free again
    }
}

template <int DT, bool WF32, int WPR, int MAXT, bool POST, bool LAYER, bool RAGGED>
__global__ __launch_bounds__(MAXT) void norm_bwd_kernel(NormArgs a, NormSplit sp)
{
    constexpr int VEC = Elem<DT>::PER16, NCH = COLS / VEC, ROWS = WPR ? 4 / WPR : 1;
    __shared__ f32x2 buf[2][16];
    __shared__ float join[WPR ? (ROWS - 1) * WPR * 64 * COLS + 1 : 1];
    const Shares<WPR> sh;
    const int dim = (int)a.dim;
    const float inv_dim = 1.0f / (float)dim;
    const int64_t rpg = a.n / a.groups;
    const Columns<VEC, RAGGED> cs(dim, sh.threads, sh.lane);
    float dpw[COLS] = {}, dpb[COLS] = {}, dqw[COLS] = {}, dqb[COLS] = {}, dg[COLS] = {};
    float *const part = a.workspace;                       // [5][wgs][dim]
    const int64_t kind = (int64_t)sp.wgs * a.dim;
    RawWeight<DT, WF32, VEC, RAGGED> w1, b1, w2, gt;
    if constexpr (POST) {
        w1.load(a.post_weight, 0, cs);
        w1.landed();
        if constexpr (LAYER) b1.load(a.post_bias, 0, cs), b1.landed();
    }
    w2.load(a.pre_weight, 0, cs);
    w2.landed();

    // The workgroup's groups of gates g0, g0 + gstep, ... and of each the rows from `first` to `last`;
    // with few groups its rows at a time are rows of one group, with many they are of a group each.
    int64_t g0 = blockIdx.x, gstep = a.groups, first = 0, last = rpg;
    const bool split = sp.per_group != 0;
    if (split) {
        g0 = blockIdx.x / sp.per_group;
        const int64_t each = (rpg + sp.per_group - 1) / sp.per_group;
        first = (blockIdx.x % sp.per_group) * each;
        last = min(rpg, first + each);
    } else {
        g0 = (int64_t)blockIdx.x * ROWS;
        gstep = (int64_t)sp.wgs * ROWS;
    }
    const int64_t mine_g = split ? 0 : sh.mine, mine_i = split ? sh.mine : 0, istep = split ? ROWS : 1;
    RawRow<DT, VEC, RAGGED> xw, yw, dw, rw;
    f32x4 next_st = {0.0f, 0.0f, 0.0f, 0.0f};
    auto fetch = [&](int64_t row) {
        next_st = *(const f32x4 *)(a.stats + row * 4);
        xw.load(a.x, row * a.x_stride, cs);
        yw.load(a.block, row * a.block_stride, cs);
        dw.load(a.dh, row * a.dh_stride, cs);
        if (a.dr) rw.load(a.dr, row * a.dr_stride, cs);
    };
#pragma unroll
    for (int c = 0; c < NCH; c++) xw.w[c] = yw.w[c] = dw.w[c] = rw.w[c] = u32x4{0, 0, 0, 0};
    if (g0 + mine_g < a.groups && first + mine_i < last) fetch((g0 + mine_g) * rpg + first + mine_i);
    for (int64_t gb = g0; gb < a.groups; gb += gstep) {
        const int64_t g = gb + mine_g;
        gt.load(g < a.groups ? a.gate : nullptr, g * a.dim, cs);
        gt.landed();
        for (int64_t ib = first; ib < last; ib += istep) {
            const int64_t i = ib + mine_i, row = g * rpg + i;
            const bool there = g < a.groups && i < last;
            const f32x4 st = next_st;
            float x[COLS], y[COLS], d[COLS], r[COLS];
            xw.unpack(x);
            yw.unpack(y);
            dw.unpack(d);
            rw.unpack(r);
            if (i + istep < last) {
                if (g < a.groups) fetch(row + istep);
            } else if (ib + istep >= last && g + gstep < a.groups && first + mine_i < last) fetch((g + gstep) * rpg + first + mine_i);
            // y: block normalised; x: r normalised; d: dh times the weight
            f32x2 s = {0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < NCH; c++) {
                float u1[VEC], c1[VEC] = {}, gg[VEC], u2[VEC];
                if constexpr (POST) {
                    w1.unpack(c, u1);
                    if constexpr (LAYER) b1.unpack(c, c1);
                }
                gt.unpack(c, gg);
                w2.unpack(c, u2);
#pragma unroll
                for (int k = 0; k < VEC; k++) {
                    const int j = c * VEC + k;
                    const bool counts = there && cs.counts(c, k);
                    float n1 = y[j];
                    if constexpr (POST) {
                        y[j] = (y[j] - st[0]) * st[1];
                        n1 = y[j] * u1[k] + c1[k];
                    }
                    const float R = a.residual_scale * x[j] + (a.gate ? gg[k] * n1 : n1);
                    x[j] = (R - st[2]) * st[3];
                    if (counts) {
                        dpw[j] += d[j] * x[j];
                        if constexpr (LAYER) dpb[j] += d[j];
                    }
                    d[j] *= u2[k];
                    if (counts) {
                        s[0] += d[j] * x[j];
                        if constexpr (LAYER) s[1] += d[j];
                    }
                }
            }
            s = sh.sum2(s, buf[0]) * inv_dim;
            // (unpacked again below rather than kept unpacked meanwhile)
            if constexpr (POST) w1.landed();
            if constexpr (POST && LAYER) b1.landed();
            gt.landed();
            f32x2 s1 = {0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < NCH; c++) {
                float u1[VEC], c1[VEC] = {}, gg[VEC], dx[VEC];
                if constexpr (POST) {
                    w1.unpack(c, u1);
                    if constexpr (LAYER) b1.unpack(c, c1);
                }
                gt.unpack(c, gg);
#pragma unroll
                for (int k = 0; k < VEC; k++) {
                    const int j = c * VEC + k;
                    const bool counts = there && cs.counts(c, k);
                    float R = d[j] - x[j] * s[0];
                    if constexpr (LAYER) R -= s[1];
                    R = r[j] + R * st[3];
                    dx[k] = a.residual_scale * R;
                    if (a.gate) {
                        if (counts) dg[j] += R * (POST ? y[j] * u1[k] + c1[k] : y[j]);
                        R *= gg[k];
                    }
                    d[j] = R;                              // the gradient of n1
                    if constexpr (POST) {
                        if (counts) {
                            dqw[j] += R * y[j];
                            if constexpr (LAYER) dqb[j] += R;
                        }
                        d[j] = R * u1[k];
                        if (counts) {
                            s1[0] += d[j] * y[j];
                            if constexpr (LAYER) s1[1] += d[j];
                        }
                    }
                }
                if (there && cs.live[c]) store_piece<DT, VEC, RAGGED>(a.dx, row * a.dim, cs, c, dx);
            }
            if constexpr (POST) s1 = sh.sum2(s1, buf[1]) * inv_dim;
            else if constexpr (WPR != 1) __syncthreads();  // buf[0] is written again by the next row
#pragma unroll
            for (int c = 0; c < NCH; c++) {
                if constexpr (POST) {
#pragma unroll
                    for (int k = 0; k < VEC; k++) {
                        const int j = c * VEC + k;
                        float t = d[j] - y[j] * s1[0];
                        if constexpr (LAYER) t -= s1[1];
                        d[j] = t * st[1];
                    }
                }
                if (there && cs.live[c]) store_piece<DT, VEC, RAGGED>(a.dblock, row * a.dim, cs, c, d + c * VEC);
            }
            if constexpr (POST && WPR != 1) __syncthreads();   // and so is buf[1]
        }
        if (a.gate && !split && g < a.groups) {
#pragma unroll
            for (int c = 0; c < NCH; c++)
#pragma unroll
                for (int k = 0; k < VEC; k++) {
                    if (cs.counts(c, k)) Elem<WF32 ? DT_F32 : DT>::store(a.dgate, g * a.dim + cs.col[c] + k, dg[c * VEC + k]);
                    dg[c * VEC + k] = 0.0f;
                }
        }
    }

    auto put = [&](float *acc, int which) {
        if constexpr (ROWS > 1) {
            // the sums of the workgroup's other rows through LDS, added in their order
            __syncthreads();
            if (sh.mine > 0)
#pragma unroll
                for (int j = 0; j < COLS; j++) join[((sh.mine - 1) * COLS + j) * sh.threads + sh.lane] = acc[j];
            __syncthreads();
            if (sh.mine > 0) return;
#pragma unroll
            for (int j = 0; j < COLS; j++)
                for (int w = 0; w < ROWS - 1; w++) acc[j] += join[(w * COLS + j) * sh.threads + sh.lane];
        }
#pragma unroll
        for (int c = 0; c < NCH; c++) {
            float *to = part + which * kind + blockIdx.x * a.dim + cs.col[c];
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
    if (a.gate && split) put(dg, 4);
}

template <int DT, bool WF32, int WPR, int MAXT, bool POST, bool LAYER, bool RAGGED>
void go(const NormArgs &a, const NormSplit &sp, bool backward, hipStream_t stream)
{
    const int threads = WPR ? 256 : (int)((a.dim + COLS * 64 - 1) / (COLS * 64) * 64);
    if (!backward) {
        const int64_t rows = WPR ? (a.n + 4 / WPR - 1) / (4 / WPR) : a.n;
        norm_fwd_kernel<DT, WF32, WPR, MAXT, POST, LAYER, RAGGED><<<(unsigned)(rows < sp.fwd_wgs ? rows : sp.fwd_wgs), threads, 0, stream>>>(a);
    } else {
        norm_bwd_kernel<DT, WF32, WPR, MAXT, POST, LAYER, RAGGED><<<sp.wgs, threads, 0, stream>>>(a, sp);
    }
}

template <int DT, bool WF32, int WPR, int MAXT, bool RAGGED>
void by_kind(const NormArgs &a, const NormSplit &sp, bool backward, hipStream_t stream)
{
    if (a.post_weight) {
        if (a.layer) go<DT, WF32, WPR, MAXT, true, true, RAGGED>(a, sp, backward, stream);
        else go<DT, WF32, WPR, MAXT, true, false, RAGGED>(a, sp, backward, stream);
    } else {
        if (a.layer) go<DT, WF32, WPR, MAXT, false, true, RAGGED>(a, sp, backward, stream);
        else go<DT, WF32, WPR, MAXT, false, false, RAGGED>(a, sp, backward, stream);
    }
}

template <int DT, bool WF32, bool RAGGED>
void by_width(const NormArgs &a, const NormSplit &sp, bool backward, hipStream_t stream)
{
    if (sp.waves == 1) by_kind<DT, WF32, 1, 256, RAGGED>(a, sp, backward, stream);
    else if (sp.waves == 2) by_kind<DT, WF32, 2, 256, RAGGED>(a, sp, backward, stream);
    else if (sp.waves <= 8) by_kind<DT, WF32, 0, 512, RAGGED>(a, sp, backward, stream);
    else by_kind<DT, WF32, 0, 1024, RAGGED>(a, sp, backward, stream);
}

}  // namespace

template <int DT, bool WF32>
hipError_t norm_run(const NormArgs &a, const NormSplit &sp, bool ragged, bool backward, hipStream_t stream)
{
    ragged ? by_width<DT, WF32, true>(a, sp, backward, stream) : by_width<DT, WF32, false>(a, sp, backward, stream);
    return hipGetLastError();
}

}  // namespace lm
