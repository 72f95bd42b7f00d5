// lm_attn_kernel.h -- causal attention over a window of the last keys and a few first ones (sinks).
//
//   S = scale q k^T over the visible keys,  P = softmax(S) (all 0 where a row sees nothing),  o = P v
//   dv = P^T do,  dS = P * (do v^T - rowsum(do * o)),  dq = scale dS k,  dk = scale dS^T q
//
// Rows.  The `group` heads that share a key head are rows of one matrix: row r is position
// r / group of head r % group.  Their keys are read once for all of them, their dk and dv are
// summed in the accumulators, and a single position with a group of heads fills a tile.
//
// Products.  v_mfma_f32_32x32x16: A and B hold 8 consecutive k of one row (column) per lane,
// lanes 32-63 the next 8; the result has column lane & 31 and rows 8 (r / 4) + 4 (lane >> 5) + r % 4.
// Every score product is formed so that its result, rounded to 16 bits, is the B operand of the next
// product without moving between lanes: k slot (half, j) of that product then stands for row
// 4 half + j (j < 4) or 8 + 4 half + j - 4, and its A operand is read in the same order by the
// transposing LDS reads (ds_read_b64_tr_b16), which take 4 rows x 16 columns and hand each lane 4
// rows of one column.  Softmax statistics then belong to lanes (a column is a row of the attention):
// maximum and sum need one exchange between the wave's halves.
//
// LDS tiles are row major, 16-byte pieces XOR-ed with their row so that both the row reads (16
// lanes, 16 rows, one piece) and the transposing reads (4 rows x 2 pieces) fall on different banks.
#pragma once
#include "lm_attn.h"
#include "lm_common.h"

namespace lm {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr int TILE = 64;                       // keys (backward for the keys: rows) of an LDS tile

template <int DT>
__device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c)
{
    if constexpr (DT == DT_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ f32x16 zero16()
{
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; i++) z[i] = 0.0f;
    return z;
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32, 64); }

// A tile of rows of HD 16-bit elements in LDS.
template <int HD>
struct Tile {
    static constexpr int PIECES = HD / 8, ROW = HD * 2;
    static __device__ __forceinline__ int turn(int row)
    {
        return HD == 128 ? ((row & 7) << 1) | ((row >> 3) & 1) : (row & 6) | ((row >> 3) & 1);
    }
    static __device__ __forceinline__ int at(int row, int piece) { return row * ROW + ((piece ^ turn(row)) << 4); }

    // A operand, its k along the elements: row `row` + lane & 31, elements 16 c + 8 half ...
    static __device__ __forceinline__ u32x4 rows(const char *t, int row, int c, int lane)
    {
        return *(const u32x4 *)(t + at(row + (lane & 31), 2 * c + (lane >> 5)));
    }
    // A operand, its k along the rows: element 32 d + lane & 31 of the 16 rows from `row`, in the
    // order of a result's registers
    static __device__ __forceinline__ u32x4 columns(const char *t, int row, int d, int lane)
    {
        typedef __attribute__((address_space(3))) s16x4 *lds4;
        const int i = lane & 15, r = row + 4 * (lane >> 5) + (i >> 2), piece = 4 * d + ((lane >> 3) & 2) + ((i >> 1) & 1);
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(t + at(r, piece) + (i & 1) * 8));
        const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(t + at(r + 8, piece) + (i & 1) * 8));
        const u32x2 u = __builtin_bit_cast(u32x2, x), w = __builtin_bit_cast(u32x2, y);
        return u32x4{u[0], u[1], w[0], w[1]};
    }
};

// 8 results (registers r0 .. r0 + 7) rounded to the B operand of 16 k.
template <int DT>
__device__ __forceinline__ u32x4 operand(const f32x16 &s, int r0)
{
    return u32x4{pack2<DT>(s[r0], s[r0 + 1]), pack2<DT>(s[r0 + 2], s[r0 + 3]), pack2<DT>(s[r0 + 4], s[r0 + 5]),
                 pack2<DT>(s[r0 + 6], s[r0 + 7])};
}

// The row of a result's register r within its 32.
__device__ __forceinline__ int result_row(int r, int lane) { return 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3); }

// What a row at position p sees, and what a block of rows sees of a block of keys.
struct Sight {
    int window, sinks;
    __device__ __forceinline__ bool one(int p, int j) const { return j <= p && (p - j < window || j < sinks); }
    __device__ __forceinline__ bool none(int pa, int pb, int ka, int kb) const
    {
        return ka > pb || (pa - kb >= window && ka >= sinks);
    }
    __device__ __forceinline__ bool all(int pa, int pb, int ka, int kb) const
    {
        return kb <= pa && (pb - ka < window || kb < sinks);
    }
};

// The key tiles that rows at positions pa .. pb see: those of the sinks that lie before the window's,
// then the window's.
struct KeyTiles {
    int sink_tiles, first, count;
    __device__ __forceinline__ KeyTiles(const AttnArgs &a, int pa, int pb)
    {
        first = max(0, pa - a.window + 1) / TILE;
        sink_tiles = min(first, (a.sinks + TILE - 1) / TILE);
        count = sink_tiles + pb / TILE - first + 1;
    }
    __device__ __forceinline__ int key(int i) const { return (i < sink_tiles ? i : first + i - sink_tiles) * TILE; }
};

// THREADS threads bring a tile of rows from memory to LDS by way of registers: load(), then store()
// once the tile's last readers are done.  Rows outside [0, rows) and elements from dim on are zero,
// and so are the rows that `hidden` names: what lies there (a masked key may hold anything) must not
// meet a weight of zero.
template <int HD, int THREADS>
struct Stage {
    static constexpr int N = TILE * HD / 8 / THREADS;
    u32x4 v[N];

    template <typename Address, typename Valid>
    __device__ __forceinline__ void load(Address address, Valid valid, int dim)
    {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int e = i * THREADS + threadIdx.x, row = e / (HD / 8), d = e % (HD / 8) * 8;
            v[i] = u32x4{0, 0, 0, 0};
            if (d < dim && valid(row)) v[i] = *(const u32x4 *)(address(row) + d);
        }
    }
    __device__ __forceinline__ void store(char *tile) const
    {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int e = i * THREADS + threadIdx.x, row = e / (HD / 8), piece = e % (HD / 8);
            *(u32x4 *)(tile + Tile<HD>::at(row, piece)) = v[i];
        }
    }
};

// The bits of the keys [key, key + 64) that the mask shows.
__device__ __forceinline__ uint64_t shown(const AttnArgs &a, int b, int key)
{
    if (!a.key_mask) return ~0ull;
    const int j = key + (threadIdx.x & 63);
    return __ballot(j < a.keys && a.key_mask[b * a.mask_stride + j] != 0);
}

__device__ __forceinline__ const uint16_t *at(const AttnTensor &t, int b, int h) { return (const uint16_t *)t.p + b * t.b + h * t.h; }

// ---------------------------------------------------------------- forward
// WAVES x 32 rows; the keys in tiles of 64, or the share of them that blockIdx.z takes.
template <int DT, int HD, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void attn_fwd_kernel(AttnArgs a)
{
    constexpr int C = HD / 16, ND = HD / 32;
    __shared__ __attribute__((aligned(16))) char lds[2][TILE * HD * 2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int b = blockIdx.y / a.key_heads, hk = blockIdx.y % a.key_heads;
    const int total = a.rows * a.group, r0 = blockIdx.x * WAVES * 32, row = r0 + wave * 32 + (lane & 31);
    const Sight sight = {a.window, a.sinks};
    const int before = a.keys - a.rows;
    const int rr = min(row, total - 1), t = rr / a.group, head = hk * a.group + rr % a.group, pos = before + t;
    const bool real = row < total;

    u32x4 q[C];
    {
        const uint16_t *p = at(a.q, b, head) + t * a.q.t;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int d = 16 * c + 8 * (lane >> 5);
            q[c] = u32x4{0, 0, 0, 0};
            if (d < a.dim) q[c] = *(const u32x4 *)(p + d);
        }
    }
    const int wa = min(r0 + wave * 32, total - 1), wb = min(r0 + wave * 32 + 31, total - 1);
    const int pa = __builtin_amdgcn_readfirstlane(before + wa / a.group), pb = __builtin_amdgcn_readfirstlane(before + wb / a.group);
    const KeyTiles tiles(a, before + r0 / a.group, before + min(r0 + WAVES * 32 - 1, total - 1) / a.group);
    const int per = (tiles.count + a.splits - 1) / a.splits, it0 = blockIdx.z * per, it1 = min(tiles.count, it0 + per);

    f32x16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) o[d] = zero16();
    float m = -__builtin_inff(), l = 0.0f;         // in units of log2; l of this lane's keys alone
    const float c2 = a.scale * LOG2E;
    const uint16_t *kp = at(a.k, b, hk), *vp = at(a.v, b, hk);
    Stage<HD, WAVES * 64> ks, vs;
    uint64_t next_shown = 0;
    auto fetch = [&](int it) {
        const int key = tiles.key(it);
        next_shown = shown(a, b, key);
        auto valid = [&](int r) { return key + r < a.keys && (next_shown >> r & 1); };
        ks.load([&](int r) { return kp + (int64_t)(key + r) * a.k.t; }, valid, a.dim);
        vs.load([&](int r) { return vp + (int64_t)(key + r) * a.v.t; }, valid, a.dim);
    };
    if (it0 < it1) fetch(it0);
    for (int it = it0; it < it1; it++) {
        const int key = tiles.key(it);
        const uint64_t see = next_shown;
        __syncthreads();
        ks.store(lds[0]);
        vs.store(lds[1]);
        __syncthreads();
        if (it + 1 < it1) fetch(it + 1);
        if (see == 0 || sight.none(pa, pb, key, key + TILE - 1)) continue;

        f32x16 s[2] = {zero16(), zero16()};
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int n = 0; n < 2; n++) s[n] = mma<DT>(Tile<HD>::rows(lds[0], 32 * n, c, lane), q[c], s[n]);
        if (see != ~0ull || !sight.all(pa, pb, key, key + TILE - 1)) {
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int j = 32 * n + result_row(r, lane);
                    if (!(sight.one(pos, key + j) && (see >> j & 1))) s[n][r] = -__builtin_inff();
                }
        }
        float top = s[0][0];
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int r = 0; r < 16; r++) top = fmaxf(top, s[n][r]);
        top = fmaxf(top, other_half(top)) * c2;
        if (__ballot(top > m)) {
            const float now = fmaxf(m, top);
            const float keep = m == now ? 1.0f : exp2_hw(m - now);     // (both -inf: nothing yet)
            m = now;
            l *= keep;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int r = 0; r < 16; r++) o[d][r] *= keep;
        }
        const float ref = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                s[n][r] = exp2_hw(__builtin_fmaf(s[n][r], c2, -ref));
                l += s[n][r];
            }
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const u32x4 p = operand<DT>(s[n], 8 * k);
#pragma unroll
                for (int d = 0; d < ND; d++) o[d] = mma<DT>(Tile<HD>::columns(lds[1], 32 * n + 16 * k, d, lane), p, o[d]);
            }
    }
    l += other_half(l);
    if (!real) return;
    if (a.splits > 1) {
        // unnormalised sums, their maximum and weight, for the join
        const int64_t at_row = ((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * total + row;
        float *po = a.partial + at_row * a.dim, *ml = a.partial + (int64_t)a.splits * gridDim.y * total * a.dim + at_row * 2;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int e = 32 * d + result_row(r, lane);
                if (e < a.dim) *(f32x4 *)(po + e) = f32x4{o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]};
            }
        if (lane < 32) {
            ml[0] = m;
            ml[1] = l;
        }
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t *po = (uint16_t *)at(a.o, b, head) + t * a.o.t;
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int e = 32 * d + result_row(r, lane);
            if (e < a.dim)
                *(u32x2 *)(po + e) = u32x2{pack2<DT>(o[d][r] * inv, o[d][r + 1] * inv), pack2<DT>(o[d][r + 2] * inv, o[d][r + 3] * inv)};
        }
    if (lane < 32) a.lse[((int64_t)b * a.heads + head) * a.rows + t] = l == 0.0f ? -__builtin_inff() : (m + log2f(l)) * LN2;
}

// Joins the parts of the keys: one wave a row, a lane for 2 elements.
template <int DT>
__global__ __launch_bounds__(64) void attn_join_kernel(AttnArgs a)
{
    const int total = a.rows * a.group, row = blockIdx.x, lane = threadIdx.x;
    const int b = blockIdx.y / a.key_heads, hk = blockIdx.y % a.key_heads;
    const int64_t rows = (int64_t)gridDim.y * total, at_row = (int64_t)blockIdx.y * total + row;
    const float *ml = a.partial + a.splits * rows * a.dim;
    float m = -__builtin_inff();
    for (int z = 0; z < a.splits; z++) m = fmaxf(m, ml[(z * rows + at_row) * 2]);
    const float ref = m == -__builtin_inff() ? 0.0f : m;
    float l = 0.0f, o0 = 0.0f, o1 = 0.0f;
    const int e = 2 * lane;
    for (int z = 0; z < a.splits; z++) {
        const float w = exp2_hw(ml[(z * rows + at_row) * 2] - ref);
        l += w * ml[(z * rows + at_row) * 2 + 1];
        if (e < a.dim) {
            const f32x2 v = *(const f32x2 *)(a.partial + (z * rows + at_row) * a.dim + e);
            o0 += w * v[0];
            o1 += w * v[1];
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int t = row / a.group, head = hk * a.group + row % a.group;
    uint16_t *po = (uint16_t *)at(a.o, b, head) + t * a.o.t;
    if (e < a.dim) *(uint32_t *)(po + e) = pack2<DT>(o0 * inv, o1 * inv);
    if (lane == 0) a.lse[((int64_t)b * a.heads + head) * a.rows + t] = l == 0.0f ? -__builtin_inff() : (m + log2f(l)) * LN2;
}

// ---------------------------------------------------------------- backward
// delta = rowsum(dout * out): 8 lanes a row.
template <int DT>
__global__ __launch_bounds__(256) void attn_delta_kernel(AttnArgs a)
{
    const int64_t row = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3), rows = (int64_t)a.batch * a.heads * a.rows;
    if (row >= rows) return;
    const int t = (int)(row % a.rows), h = (int)(row / a.rows % a.heads), b = (int)(row / a.rows / a.heads);
    const uint16_t *o = at(a.o, b, h) + t * a.o.t, *g = at(a.dout, b, h) + t * a.dout.t;
    float s = 0.0f;
    for (int d = (threadIdx.x & 7) * 8; d < a.dim; d += 64) {
        float x[8], y[8];
        load_n<DT, 8>(o, d, x);
        load_n<DT, 8>(g, d, y);
#pragma unroll
        for (int k = 0; k < 8; k++) s += x[k] * y[k];
    }
#pragma unroll
    for (int d = 4; d; d >>= 1) s += __shfl_xor(s, d, 64);
    if ((threadIdx.x & 7) == 0) a.delta[row] = s;
}

// A weight of all but 2^-16 leaves its row's other keys less than the rounding of `out` puts into
// delta: the softmax is constant there and dS is 0 (exactly so where a row sees one key).
__device__ __forceinline__ float score_gradient(float p, float dp, float delta) { return p > 1.0f - 0x1p-16f ? 0.0f : p * (dp - delta); }

// dq of WAVES x 32 rows: the forward pass's walk over the keys.
template <int DT, int HD, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void attn_dq_kernel(AttnArgs a)
{
    constexpr int C = HD / 16, ND = HD / 32;
    __shared__ __attribute__((aligned(16))) char lds[2][TILE * HD * 2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int b = blockIdx.y / a.key_heads, hk = blockIdx.y % a.key_heads;
    const int total = a.rows * a.group, r0 = blockIdx.x * WAVES * 32, row = r0 + wave * 32 + (lane & 31);
    const Sight sight = {a.window, a.sinks};
    const int before = a.keys - a.rows;
    const int rr = min(row, total - 1), t = rr / a.group, head = hk * a.group + rr % a.group, pos = before + t;
    const bool real = row < total;

    u32x4 q[C], g[C];
    {
        const uint16_t *p = at(a.q, b, head) + t * a.q.t, *pg = at(a.dout, b, head) + t * a.dout.t;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int d = 16 * c + 8 * (lane >> 5);
            q[c] = g[c] = u32x4{0, 0, 0, 0};
            if (d < a.dim) {
                q[c] = *(const u32x4 *)(p + d);
                g[c] = *(const u32x4 *)(pg + d);
            }
        }
    }
    const int64_t stat = ((int64_t)b * a.heads + head) * a.rows + t;
    float lse = a.lse[stat] * LOG2E;
    if (lse == -__builtin_inff()) lse = __builtin_inff();          // an empty row: every weight 0
    const float delta = a.delta[stat];
    const int wa = min(r0 + wave * 32, total - 1), wb = min(r0 + wave * 32 + 31, total - 1);
    const int pa = __builtin_amdgcn_readfirstlane(before + wa / a.group), pb = __builtin_amdgcn_readfirstlane(before + wb / a.group);
    const KeyTiles tiles(a, before + r0 / a.group, before + min(r0 + WAVES * 32 - 1, total - 1) / a.group);

    f32x16 dq[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) dq[d] = zero16();
    const float c2 = a.scale * LOG2E;
    const uint16_t *kp = at(a.k, b, hk), *vp = at(a.v, b, hk);
    Stage<HD, WAVES * 64> ks, vs;
    uint64_t next_shown = 0;
    auto fetch = [&](int it) {
        const int key = tiles.key(it);
        next_shown = shown(a, b, key);
        auto valid = [&](int r) { return key + r < a.keys && (next_shown >> r & 1); };
        ks.load([&](int r) { return kp + (int64_t)(key + r) * a.k.t; }, valid, a.dim);
        vs.load([&](int r) { return vp + (int64_t)(key + r) * a.v.t; }, valid, a.dim);
    };
    fetch(0);
    for (int it = 0; it < tiles.count; it++) {
        const int key = tiles.key(it);
        const uint64_t see = next_shown;
        __syncthreads();
        ks.store(lds[0]);
        vs.store(lds[1]);
        __syncthreads();
        if (it + 1 < tiles.count) fetch(it + 1);
        if (see == 0 || sight.none(pa, pb, key, key + TILE - 1)) continue;
        const bool whole = see == ~0ull && sight.all(pa, pb, key, key + TILE - 1);
#pragma unroll
        for (int n = 0; n < 2; n++) {
            f32x16 s = zero16(), dp = zero16();
#pragma unroll
            for (int c = 0; c < C; c++) {
                s = mma<DT>(Tile<HD>::rows(lds[0], 32 * n, c, lane), q[c], s);
                dp = mma<DT>(Tile<HD>::rows(lds[1], 32 * n, c, lane), g[c], dp);
            }
            if (whole) {
#pragma unroll
                for (int r = 0; r < 16; r++) s[r] = exp2_hw(__builtin_fmaf(s[r], c2, -lse)) * (dp[r] - delta);
            } else {
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int j = 32 * n + result_row(r, lane);
                    const float p = exp2_hw(__builtin_fmaf(s[r], c2, -lse));
                    s[r] = sight.one(pos, key + j) && (see >> j & 1) ? score_gradient(p, dp[r], delta) : 0.0f;
                }
            }
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const u32x4 p = operand<DT>(s, 8 * k);
#pragma unroll
                for (int d = 0; d < ND; d++) dq[d] = mma<DT>(Tile<HD>::columns(lds[0], 32 * n + 16 * k, d, lane), p, dq[d]);
            }
        }
    }
    if (!real) return;
    uint16_t *po = (uint16_t *)at(a.dq, b, head) + t * a.dq.t;
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int e = 32 * d + result_row(r, lane);
            if (e < a.dim)
                *(u32x2 *)(po + e) = u32x2{pack2<DT>(dq[d][r] * a.scale, dq[d][r + 1] * a.scale),
                                           pack2<DT>(dq[d][r + 2] * a.scale, dq[d][r + 3] * a.scale)};
        }
}

// dk and dv of WAVES x 32 keys: over the rows that see any of them, 64 at a time.
template <int DT, int HD, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void attn_dkv_kernel(AttnArgs a)
{
    constexpr int C = HD / 16, ND = HD / 32;
    __shared__ __attribute__((aligned(16))) char lds[2][TILE * HD * 2];
    __shared__ __attribute__((aligned(16))) float lse_s[TILE], delta_s[TILE];
    __shared__ __attribute__((aligned(16))) int pos_s[TILE];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int b = blockIdx.y / a.key_heads, hk = blockIdx.y % a.key_heads;
    const int k0 = blockIdx.x * WAVES * 32, ka = k0 + wave * 32, key = ka + (lane & 31);
    const Sight sight = {a.window, a.sinks};
    const int before = a.keys - a.rows, total = a.rows * a.group;
    const bool real = key < a.keys;
    const bool seen = real && (!a.key_mask || a.key_mask[b * a.mask_stride + key] != 0);
    const bool all_seen = __ballot(seen) == ~0ull;

    u32x4 kf[C], vf[C];
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int d = 16 * c + 8 * (lane >> 5);
        kf[c] = vf[c] = u32x4{0, 0, 0, 0};
        if (d < a.dim && seen) {
            kf[c] = *(const u32x4 *)(at(a.k, b, hk) + (int64_t)key * a.k.t + d);
            vf[c] = *(const u32x4 *)(at(a.v, b, hk) + (int64_t)key * a.v.t + d);
        }
    }
    f32x16 dk[ND], dv[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) dk[d] = dv[d] = zero16();
    const float c2 = a.scale * LOG2E;
    // the positions that see a key of this workgroup
    const int k1 = min(a.keys, k0 + WAVES * 32) - 1;
    const int t0 = max(0, k0 - before);
    const int t1 = k0 < a.sinks ? a.rows - 1 : (int)min((int64_t)a.rows - 1, (int64_t)k1 + a.window - 1 - before);
    const int first = t0 * a.group, last = (t1 + 1) * a.group;
    Stage<HD, WAVES * 64> qs, gs;
    float lse_r = 0.0f, delta_r = 0.0f;
    int pos_r = 0;
    auto fetch = [&](int row0) {
        auto valid = [&](int r) { return row0 + r < last; };
        auto head = [&](int r) { return hk * a.group + (row0 + r) % a.group; };
        qs.load([&](int r) { return at(a.q, b, head(r)) + (row0 + r) / a.group * a.q.t; }, valid, a.dim);
        gs.load([&](int r) { return at(a.dout, b, head(r)) + (row0 + r) / a.group * a.dout.t; }, valid, a.dim);
        if (threadIdx.x < TILE) {
            const int r = min(row0 + (int)threadIdx.x, total - 1);
            const int64_t stat = ((int64_t)b * a.heads + hk * a.group + r % a.group) * a.rows + r / a.group;
            lse_r = a.lse[stat] * LOG2E;
            // no weight where a row sees nothing, nor behind the last row
            delta_r = a.delta[stat];
            if (lse_r == -__builtin_inff() || row0 + (int)threadIdx.x >= last) {
                lse_r = __builtin_inff();
                delta_r = 0.0f;
            }
            pos_r = before + r / a.group;
        }
    };
    if (first < last) fetch(first);
    for (int row0 = first; row0 < last; row0 += TILE) {
        __syncthreads();
        qs.store(lds[0]);
        gs.store(lds[1]);
        if (threadIdx.x < TILE) {
            lse_s[threadIdx.x] = lse_r;
            delta_s[threadIdx.x] = delta_r;
            pos_s[threadIdx.x] = pos_r;
        }
        __syncthreads();
        if (row0 + TILE < last) fetch(row0 + TILE);
#pragma unroll
        for (int n = 0; n < 2; n++) {
            if (row0 + 32 * n >= last) continue;
            const int pa = before + (row0 + 32 * n) / a.group, pb = before + (min(row0 + 32 * n + 31, last - 1)) / a.group;
            if (sight.none(pa, pb, ka, ka + 31)) continue;
            const bool whole = all_seen && sight.all(pa, pb, ka, ka + 31);
            f32x16 s = zero16(), dp = zero16();
#pragma unroll
            for (int c = 0; c < C; c++) {
                s = mma<DT>(Tile<HD>::rows(lds[0], 32 * n, c, lane), kf[c], s);
                dp = mma<DT>(Tile<HD>::rows(lds[1], 32 * n, c, lane), vf[c], dp);
            }
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int i = 32 * n + result_row(r, lane);
                const f32x4 ls = *(const f32x4 *)(lse_s + i), de = *(const f32x4 *)(delta_s + i);
                const u32x4 po = *(const u32x4 *)(pos_s + i);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    float p = exp2_hw(__builtin_fmaf(s[r + k], c2, -ls[k]));
                    if (whole) dp[r + k] = p * (dp[r + k] - de[k]);
                    else {
                        if (!(seen && sight.one((int)po[k], key))) p = 0.0f;
                        dp[r + k] = score_gradient(p, dp[r + k], de[k]);
                    }
                    s[r + k] = p;
                }
            }
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const u32x4 p = operand<DT>(s, 8 * k), ds = operand<DT>(dp, 8 * k);
#pragma unroll
                for (int d = 0; d < ND; d++) {
                    dv[d] = mma<DT>(Tile<HD>::columns(lds[1], 32 * n + 16 * k, d, lane), p, dv[d]);
                    dk[d] = mma<DT>(Tile<HD>::columns(lds[0], 32 * n + 16 * k, d, lane), ds, dk[d]);
                }
            }
        }
    }
    if (!real) return;
    uint16_t *pk = (uint16_t *)at(a.dk, b, hk) + (int64_t)key * a.dk.t, *pv = (uint16_t *)at(a.dv, b, hk) + (int64_t)key * a.dv.t;
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int e = 32 * d + result_row(r, lane);
            if (e >= a.dim) continue;
            *(u32x2 *)(pk + e) = u32x2{pack2<DT>(dk[d][r] * a.scale, dk[d][r + 1] * a.scale),
                                       pack2<DT>(dk[d][r + 2] * a.scale, dk[d][r + 3] * a.scale)};
            *(u32x2 *)(pv + e) = u32x2{pack2<DT>(dv[d][r], dv[d][r + 1]), pack2<DT>(dv[d][r + 2], dv[d][r + 3])};
        }
}

template <int DT, int HD>
void run_forward(const AttnArgs &a, hipStream_t stream)
{
    const int total = a.rows * a.group;
    if (total <= 32)
        attn_fwd_kernel<DT, HD, 1><<<dim3(1, a.batch * a.key_heads, a.splits), 64, 0, stream>>>(a);
    else
        attn_fwd_kernel<DT, HD, 4><<<dim3((total + 127) / 128, a.batch * a.key_heads, a.splits), 256, 0, stream>>>(a);
    if (a.splits > 1) attn_join_kernel<DT><<<dim3(total, a.batch * a.key_heads), 64, 0, stream>>>(a);
}

template <int DT, int HD>
void run_backward(const AttnArgs &a, hipStream_t stream)
{
    const int total = a.rows * a.group;
    const int64_t rows = (int64_t)a.batch * a.heads * a.rows;
    if (rows) attn_delta_kernel<DT><<<(unsigned)((rows + 31) / 32), 256, 0, stream>>>(a);
    attn_dkv_kernel<DT, HD, 4><<<dim3((a.keys + 127) / 128, a.batch * a.key_heads), 256, 0, stream>>>(a);
    if (rows) attn_dq_kernel<DT, HD, 4><<<dim3((total + 127) / 128, a.batch * a.key_heads), 256, 0, stream>>>(a);
}

}  // namespace

template <int DT>
hipError_t attn_forward(const AttnArgs &a, hipStream_t stream)
{
    if (a.dim <= 64) run_forward<DT, 64>(a, stream);
    else run_forward<DT, 128>(a, stream);
    return hipGetLastError();
}

template <int DT>
hipError_t attn_backward(const AttnArgs &a, hipStream_t stream)
{
    if (a.dim <= 64) run_backward<DT, 64>(a, stream);
    else run_backward<DT, 128>(a, stream);
    return hipGetLastError();
}

}  // namespace lm
