// lm_expert_kernel.h -- matrix products grouped by expert: expert e owns the rows offsets[e] .. offsets[e + 1].
//
//   forward   y[r, o]    = sum_i x[r, i] W[e, o, i]
//   dx        dx[r, i]   = sum_o dy[r, o] W[e, o, i]
//   dweight   dW[e, o, i] = sum over e's rows of dy[r, o] x[r, i]
//
// All three are C[m, n] = sum_k A[m, k] B[n, k] over tiles of m and n, and differ in which operand is dense along k.
// How many tiles an expert has is known on the device only: the grid holds the most that the sizes allow, a wave finds
// its tile by a scan over the experts' row counts, and what is left over ends at once.
#pragma once
#include "lm_common.h"
#include "lm_expert.h"

namespace lm {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) char lds_char;
typedef const __attribute__((address_space(1))) uint32_t global_word;
typedef __attribute__((address_space(3))) uint32_t lds_word;

enum Form { FORWARD = 0, DX = 1, DWEIGHT = 2 };
constexpr int BK = 64;                    // k of one LDS tile

template <int DT>
__device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c)
{
    if constexpr (DT == DT_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// What reads behind the end of k find: LDS tiles are filled by loads alone, so a piece that does not exist comes from here.
__device__ __attribute__((aligned(16))) const uint32_t ZEROS[4] = {0, 0, 0, 0};

struct Tile {
    int expert, first, last;              // the expert's rows [first, last)
    int m, n;                             // the tile's place among its rows and columns of tiles
};

// The row counts that a plan gives, kept within its slots whatever it holds.
__device__ __forceinline__ int bound(const int32_t *offsets, int e, int slots) { return min(max(offsets[e], 0), slots); }

// Tile `index` of those that the experts' rows make, bm rows each and n_tiles side by side; false behind the last one.
// The expert behind the last stands for the rows of none, whose results are zero.
__device__ __forceinline__ bool find_tile(const int32_t *offsets, int experts, int slots, int bm, int n_tiles, uint32_t index, Tile &t)
{
    const int lane = threadIdx.x & 63;
    uint32_t before = 0;
    for (int e0 = 0; e0 <= experts; e0 += 64) {
        const int e = e0 + lane;
        int first = 0, last = 0;
        if (e <= experts) {
            first = bound(offsets, e, slots);
            last = e < experts ? bound(offsets, e + 1, slots) : slots;
        }
        const uint32_t tiles = last > first ? (uint32_t)((last - first + bm - 1) / bm) * n_tiles : 0;
        uint32_t upto = tiles;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t o = __shfl_up(upto, d, 64);
            if (lane >= d) upto += o;
        }
        const uint64_t mine = __ballot(before + upto > index);
        if (mine) {
            const int at = __builtin_ctzll(mine);
            const uint32_t rest = index - before - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(tiles, at));
            t.expert = e0 + at;
            t.first = __builtin_amdgcn_readlane(first, at);
            t.last = __builtin_amdgcn_readlane(last, at);
            t.m = rest / n_tiles;
            t.n = rest % n_tiles;
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// The row of x that row r of the sorted buffer stands for.
__device__ __forceinline__ int64_t source_row(const ProductArgs &a, int r)
{
    if (a.k == 0) return r;
    const uint32_t token = (uint32_t)a.rows[r] / (uint32_t)a.k;
    return token < (uint64_t)a.tokens ? token : 0;
}

// One operand's LDS tile of ROWS x BK.  ALONG: its memory is dense along k (a row of the tile is a row of memory, BK of its
// elements); otherwise dense across (a row of the tile is one k, ROWS elements).  16-byte pieces are XOR-ed with their row, so
// that the lanes of a read fall on different banks; loads write LDS in lane order, so the lanes' addresses are permuted instead.
template <int ROWS, bool ALONG, int THREADS>
struct Operand {
    static constexpr int BYTES = ROWS * BK * 2;
    static constexpr int PIECES = ALONG ? BK / 8 : ROWS / 8;            // of 16 bytes in a row of the tile
    static constexpr int LOADS = BYTES / 16 / THREADS;
    static constexpr int STEP = THREADS / PIECES;                       // rows between a thread's loads

    static __device__ __forceinline__ int turn(int row) { return ALONG ? (row >> 1) & 7 : (row & 3) << 2; }
    static __device__ __forceinline__ int row_of(int i) { return threadIdx.x / PIECES + i * STEP; }
    static __device__ __forceinline__ int piece_of(int i) { return (threadIdx.x % PIECES) ^ turn(row_of(i)); }

    static __device__ __forceinline__ void load(lds_char *tile, int i, const char *from)
    {
        lds_char *to = tile + (i * THREADS + (threadIdx.x & ~63)) * 16;
        __builtin_amdgcn_global_load_lds((global_word *)from, (lds_word *)to, 16, 0, 0);
    }

    // 32 rows from `row0`, k 16 step .. : lane l holds row l & 31 and 8 of the k, l >> 5 saying which
    static __device__ __forceinline__ u32x4 read(const lds_char *tile, int row0, int step)
    {
        const int lane = threadIdx.x & 63;
        if constexpr (ALONG) {
            const int row = lane & 31;
            const int at = row * (BK * 2) + (((lane >> 5) ^ turn(row)) << 4);
            return *(const __attribute__((address_space(3))) u32x4 *)(tile + (at ^ (step << 5)) + row0 * (BK * 2));
        } else {
            typedef __attribute__((address_space(3))) s16x4 *lds4;
            const int k = 8 * (lane >> 5) + ((lane >> 2) & 3);
            const int piece = (row0 >> 3) + ((lane >> 3) & 2) + ((lane >> 1) & 1);
            const lds_char *p = tile + ((piece ^ turn(k)) << 4) + (lane & 1) * 8 + (k + 16 * step) * (ROWS * 2);
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + 4 * ROWS * 2));
            const u32x2 u = __builtin_bit_cast(u32x2, lo), w = __builtin_bit_cast(u32x2, hi);
            return u32x4{u[0], u[1], w[0], w[1]};
        }
    }
};

// A workgroup's tile of BM x BN of the result, WM x WN waves.
template <int DT, int FORM, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM *WN * 64, WM *WN == 8 ? 2 : 2) void product_kernel(ProductArgs a, int m_tiles, int n_tiles)
{
    constexpr int THREADS = WM * WN * 64, MI = BM / WM / 32, NI = BN / WN / 32;
    using OpA = Operand<BM, FORM != DWEIGHT, THREADS>;
    using OpB = Operand<BN, FORM == FORWARD, THREADS>;
    __shared__ __attribute__((aligned(256))) char lds[2 * (OpA::BYTES + OpB::BYTES)];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    Tile t;
    const int slots = (int)a.slots;
    if constexpr (FORM == DWEIGHT) {
        const uint32_t per = (uint32_t)m_tiles * n_tiles;
        t.expert = blockIdx.x / per;
        const uint32_t rest = blockIdx.x % per;
        t.m = rest / n_tiles;
        t.n = rest % n_tiles;
        t.first = bound(a.offsets, t.expert, slots);
        t.last = max(t.first, bound(a.offsets, t.expert + 1, slots));
    } else {
        if (!find_tile(a.offsets, a.experts, slots, BM, n_tiles, blockIdx.x, t)) return;
    }
    const int m0 = t.m * BM, n0 = t.n * BN;
    const int M = FORM == DWEIGHT ? a.out : t.last - t.first, N = FORM == FORWARD ? a.out : a.in;
    const bool none = t.expert == a.experts;
    const int K = none ? 0 : FORM == FORWARD ? a.in : FORM == DX ? a.out : t.last - t.first;
    const char *const zeros = (const char *)ZEROS;
    const char *const weight = (const char *)a.weight + (none ? 0 : (int64_t)t.expert * a.weight_expert_stride) * 2;

    // where each thread's pieces come from: rows of memory along k are clamped to the last, those across k to the first column
    const char *pa[OpA::LOADS], *pb[OpB::LOADS];
    int sa[OpA::LOADS], sb[OpB::LOADS];           // DWEIGHT: nothing; the k index that a piece stands for
#pragma unroll
    for (int i = 0; i < OpA::LOADS; i++) {
        if constexpr (FORM == DWEIGHT) {
            const int col = m0 + OpA::piece_of(i) * 8;
            sa[i] = OpA::row_of(i);
            pa[i] = (const char *)a.dy + ((t.first + sa[i]) * a.dy_stride + (col < M ? col : 0)) * 2;
        } else {
            const int r = t.first + min(m0 + OpA::row_of(i), M - 1);
            sa[i] = OpA::piece_of(i) * 8;
            if constexpr (FORM == FORWARD) pa[i] = (const char *)a.x + ((none ? 0 : source_row(a, r)) * a.x_stride + sa[i]) * 2;
            else pa[i] = (const char *)a.dy + (r * a.dy_stride + sa[i]) * 2;
        }
    }
#pragma unroll
    for (int i = 0; i < OpB::LOADS; i++) {
        if constexpr (FORM == FORWARD) {
            sb[i] = OpB::piece_of(i) * 8;
            pb[i] = weight + (min(n0 + OpB::row_of(i), N - 1) * a.weight_row_stride + sb[i]) * 2;
        } else {
            const int col = n0 + OpB::piece_of(i) * 8;
            sb[i] = OpB::row_of(i);
            const int at = col < N ? col : 0;
            if constexpr (FORM == DX) pb[i] = weight + (sb[i] * a.weight_row_stride + at) * 2;
            else pb[i] = (const char *)a.x + at * 2;
        }
    }
    // DWEIGHT: the rows of x that the next tile's rows stand for
    int64_t next[OpB::LOADS];
    auto look_ahead = [&](int k0) {
        if constexpr (FORM == DWEIGHT) {
#pragma unroll
            for (int i = 0; i < OpB::LOADS; i++) next[i] = k0 + sb[i] < K ? source_row(a, t.first + k0 + sb[i]) : 0;
        }
    };
    auto fill = [&](int k0, int buffer) {
        lds_char *la = (lds_char *)lds + buffer * (OpA::BYTES + OpB::BYTES), *lb = la + OpA::BYTES;
        const int64_t ka = FORM == DWEIGHT ? k0 * a.dy_stride * 2 : (int64_t)k0 * 2;
        const int64_t kb = FORM == FORWARD ? (int64_t)k0 * 2 : k0 * a.weight_row_stride * 2;
#pragma unroll
        for (int i = 0; i < OpA::LOADS; i++) OpA::load(la, i, k0 + sa[i] < K ? pa[i] + ka : zeros);
#pragma unroll
        for (int i = 0; i < OpB::LOADS; i++) {
            const char *p = FORM == DWEIGHT ? pb[i] + next[i] * a.x_stride * 2 : pb[i] + kb;
            OpB::load(lb, i, k0 + sb[i] < K ? p : zeros);
        }
    };

    f32x16 acc[NI][MI];
#pragma unroll
    for (int i = 0; i < NI; i++)
#pragma unroll
        for (int j = 0; j < MI; j++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[i][j][r] = 0.0f;
    const int wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);
    if (K > 0) {
        look_ahead(0);
        fill(0, 0);
        look_ahead(BK);
    }
    for (int k0 = 0, buffer = 0; k0 < K; k0 += BK, buffer ^= 1) {
        __syncthreads();
        if (k0 + BK < K) {
            fill(k0 + BK, buffer ^ 1);
            look_ahead(k0 + 2 * BK);
        }
        const lds_char *la = (const lds_char *)lds + buffer * (OpA::BYTES + OpB::BYTES), *lb = la + OpA::BYTES;
#pragma unroll
        for (int s = 0; s < BK / 16; s++) {
            u32x4 fa[MI], fb[NI];
#pragma unroll
            for (int i = 0; i < NI; i++) fb[i] = OpB::read(lb, wn + 32 * i, s);
#pragma unroll
            for (int j = 0; j < MI; j++) fa[j] = OpA::read(la, wm + 32 * j, s);
#pragma unroll
            for (int i = 0; i < NI; i++)
#pragma unroll
                for (int j = 0; j < MI; j++) acc[i][j] = mma<DT>(fb[i], fa[j], acc[i][j]);
        }
    }

    // a lane holds row m = lane & 31 of a 32 x 32 block, columns 8 (r / 4) + 4 (lane >> 5) + r % 4
#pragma unroll
    for (int j = 0; j < MI; j++) {
        const int m = m0 + wm + 32 * j + (lane & 31);
        if (m >= M) continue;
#pragma unroll
        for (int i = 0; i < NI; i++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const int n = n0 + wn + 32 * i + 8 * g + 4 * (lane >> 5);
                if (n >= N) continue;
                const float v[4] = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
                if constexpr (FORM == FORWARD) store_n<DT, 4>(a.y, (int64_t)(t.first + m) * a.out + n, v);
                else if constexpr (FORM == DX) {
                    if (a.scratch) store_n<DT_F32, 4>(a.scratch, (int64_t)(t.first + m) * a.in + n, v);
                    else store_n<DT, 4>(a.dx, (int64_t)(t.first + m) * a.in + n, v);
                } else {
                    const int64_t at = ((int64_t)t.expert * a.out + m) * a.in + n;
                    if (a.dweight_f32) store_n<DT_F32, 4>(a.dweight, at, v);
                    else store_n<DT, 4>(a.dweight, at, v);
                }
            }
    }
}

template <int DT, int FORM, int BM, int BN, int WM, int WN>
hipError_t launch(const ProductArgs &a, hipStream_t stream)
{
    const int n = FORM == FORWARD ? a.out : a.in;
    const int64_t n_tiles = (n + BN - 1) / BN;
    const int64_t m_tiles = FORM == DWEIGHT ? (a.out + BM - 1) / BM : 0;
    // each expert, and the rows of none, may end with a tile that is not full
    const int64_t parts = a.slots < a.experts + 1 ? a.slots : a.experts + 1;
    const int64_t wgs = FORM == DWEIGHT ? a.experts * m_tiles * n_tiles : (a.slots / BM + parts) * n_tiles;
    if (wgs == 0) return hipSuccess;
    product_kernel<DT, FORM, BM, BN, WM, WN><<<(unsigned)wgs, WM * WN * 64, 0, stream>>>(a, (int)m_tiles, (int)n_tiles);
    return hipGetLastError();
}

template <int DT, int FORM>
hipError_t pick(const ProductArgs &a, hipStream_t stream)
{
    return launch<DT, FORM, 128, 128, 2, 2>(a, stream);
}

}  // namespace

template <int DT>
hipError_t product_forward(const ProductArgs &a, hipStream_t stream)
{
    return pick<DT, FORWARD>(a, stream);
}

template <int DT>
hipError_t product_backward(const ProductArgs &a, hipStream_t stream)
{
    if (a.dx) {
        hipError_t e = pick<DT, DX>(a, stream);
        if (e != hipSuccess) return e;
        if (a.k) {
            // the sum of a token's rows, from fp32: rounded once
            CombineArgs c = {};
            c.n = a.tokens;
            c.k = a.k;
            c.experts = a.experts;
            c.dim = a.in;
            c.y = a.scratch;
            c.y_dt = DT_F32;
            c.y_stride = a.in;
            c.places = a.places;
            c.offsets = a.offsets;
            c.out = a.dx;
            c.out_dt = DT;
            c.out_stride = a.in;
            e = combine_forward(c, stream);
            if (e != hipSuccess) return e;
        }
    }
    return a.dweight ? pick<DT, DWEIGHT>(a, stream) : hipSuccess;
}

}  // namespace lm
