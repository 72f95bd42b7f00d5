// lm_expert_kernel.h -- matrix products grouped by expert: expert e owns the rows offsets[e] .. offsets[e + 1].
//
//   forward   y[r, o]    = sum_i x[r, i] W[e, o, i]
//   dx        dx[r, i]   = sum_o dy[r, o] W[e, o, i]
//   dweight   dW[e, o, i] = sum over e's rows of dy[r, o] x[r, i]
//
// All three are C[m, n] = sum_k A[m, k] B[n, k] over tiles of m and n, and differ in which operand is dense along k.
// How many tiles an expert has is known on the device only: workgroups are as many as the chip holds and take tiles in turn,
// each found by a scan over the experts' row counts.
//
// A tile of 256 x 256 x 64 is 2048 cycles of products for the two waves of a SIMD.  Its operands' reads from LDS (192 KB) and the
// loads' writes to it (64 KB) take nearly as long, so both run beside the products: loads go to LDS without registers in
// between, operands are read a step ahead, and the next tile's loads are issued before this one's stores.  16384 rows of
// 4096 x 11008 (bf16): forward 1380 us, 1.07 PFLOP/s; dx 1570, 0.94; dweight 1370, 1.08 (a library's dense products of the same
// sizes 1173, 1102, 1566); matrix units are busy for 61 to 66 % of the cycles, at the 1.7 GHz that the power allows.
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

// 4 rows of one column from a tile with rows across.  The pointer is restrict so that the compiler does not make the read
// wait for the loads into the other tile that are on their way (the barrier waits for those).
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
__device__ __forceinline__ s16x4 read_turned(lds_s16x4 *__restrict__ p) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16(p); }

struct Tile {
    int expert, first, last;              // the expert's rows [first, last)
    int m, n;                             // the tile's place among its rows and columns of tiles
};

// The row counts that a plan gives, kept within its slots whatever it holds.
__device__ __forceinline__ int bound(const int32_t *offsets, int e, int slots) { return min(max(offsets[e], 0), slots); }

__device__ __forceinline__ uint32_t wave_scan(uint32_t v)
{
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(v, d, 64);
        if (lane >= d) v += o;
    }
    return v;
}

// A workgroup's tiles in turn.  Workgroups go round robin over the 8 XCDs, each with an L2 of its own: each XCD takes an
// eighth of the tiles in a row, its workgroups every so many of them.  Within an expert 8 rows of tiles go at a time, column
// by column, so that the tiles in flight on an XCD share rows and columns; a row of tiles that is not full comes last.
struct Tiles {
    uint32_t index, end, step;            // the next tile, of all of them
    int experts, slots, m_tiles, n_tiles;
    // where a lane's expert of the first 64 begins and ends, and the tiles up to its last
    int first, last;
    uint32_t tiles, upto;

    __device__ __forceinline__ void share(uint32_t total)
    {
        const uint32_t xcd = blockIdx.x & 7, each = total >> 3, more = total & 7, begin = xcd * each + min(xcd, more);
        index = begin + (blockIdx.x >> 3);
        end = begin + each + (xcd < more);
        step = gridDim.x >> 3;
    }
    // The tiles of the experts' rows.  The expert behind the last stands for the rows of none, whose results are zero.
    __device__ __forceinline__ void look_at(const int32_t *offsets, int bm, int e)
    {
        first = last = 0;
        if (e <= experts) {
            first = bound(offsets, e, slots);
            last = e < experts ? bound(offsets, e + 1, slots) : slots;
        }
        tiles = last > first ? (uint32_t)((last - first + bm - 1) / bm) * n_tiles : 0;
        upto = wave_scan(tiles);
    }
    __device__ __forceinline__ void of_rows(const int32_t *offsets, int bm)
    {
        const int lane = threadIdx.x & 63;
        uint32_t total = 0;
        for (int e0 = experts & ~63; e0 >= 0; e0 -= 64) {
            look_at(offsets, bm, e0 + lane);
            total += __builtin_amdgcn_readlane(upto, 63);
        }
        share(total);
    }
    __device__ __forceinline__ void place(uint32_t rest, int rows_of_tiles, Tile &t) const
    {
        constexpr int GROUP = 8;
        const uint32_t per = GROUP * n_tiles, group = rest / per, in = rest - group * per;
        const uint32_t rows = min((uint32_t)(rows_of_tiles - group * GROUP), (uint32_t)GROUP);
        t.n = in / rows;
        t.m = group * GROUP + (in - t.n * rows);
    }
    // The next tile; false behind the last.
    __device__ __forceinline__ bool next_of_rows(const int32_t *offsets, int bm, Tile &t)
    {
        if (index >= end) return false;
        uint32_t at = index;
        index += step;
        Tiles x = *this;                  // (of later experts: looked at anew)
        for (int e0 = 0; e0 <= experts; e0 += 64) {
            if (e0) x.look_at(offsets, bm, e0 + (threadIdx.x & 63));
            const uint64_t mine = __ballot(x.upto > at);
            if (mine) {
                const int lane = __builtin_ctzll(mine);
                t.expert = e0 + lane;
                t.first = __builtin_amdgcn_readlane(x.first, lane);
                t.last = __builtin_amdgcn_readlane(x.last, lane);
                place(at - (__builtin_amdgcn_readlane(x.upto, lane) - __builtin_amdgcn_readlane(x.tiles, lane)), (t.last - t.first + bm - 1) / bm, t);
                return true;
            }
            at -= __builtin_amdgcn_readlane(x.upto, 63);
        }
        return false;
    }
    __device__ __forceinline__ bool next_of_weights(const int32_t *offsets, Tile &t)
    {
        if (index >= end) return false;
        const uint32_t per = (uint32_t)m_tiles * n_tiles;
        t.expert = index / per;
        place(index - t.expert * per, m_tiles, t);
        t.first = bound(offsets, t.expert, slots);
        t.last = max(t.first, bound(offsets, t.expert + 1, slots));
        index += step;
        return true;
    }
};

// The token that a slot belongs to: slot / k by the reciprocal (2^32 - 1) / k, which is too small by one at most for slots
// below 2^30.  Whatever a plan's rows hold, a row of x.
__device__ __forceinline__ uint32_t token_of(const ProductArgs &a, int slot)
{
    const uint32_t s = slot;
    uint32_t token = __umulhi(s, a.k_inverse);
    if (s - token * a.k >= (uint32_t)a.k) token++;
    return token < (uint32_t)a.tokens ? token : 0;
}
// The row of x that row r of the sorted buffer stands for.
template <bool GATHER>
__device__ __forceinline__ int64_t source_row(const ProductArgs &a, int r)
{
    if constexpr (GATHER) return token_of(a, a.rows[r]);
    else return r;
}

// One operand's LDS tile of ROWS x BK.  ALONG: its memory is dense along k (a row of the tile is a row of memory, BK of its
// elements); otherwise dense across (a row of the tile is one k, ROWS elements).  16-byte pieces are XOR-ed with their row, so
// that the lanes of a read fall on different banks; loads write LDS in lane order, so the lanes' addresses are permuted instead.
// The conflicts that are counted go with the results' way out, which costs about twice its accesses: they are 2 % of the LDS
// cycles with 64 steps of k a tile (forward of 4096 x 11008), 9 % with 12 (forward of 768 x 2048), 18 % with four (dweight
// of 60 skewed experts).
template <int ROWS, bool ALONG, int THREADS, int BK>
struct Operand {
    static_assert(BK == 64, "turn");
    static constexpr int BYTES = ROWS * BK * 2;
    static constexpr int PIECES = ALONG ? BK / 8 : ROWS / 8;            // of 16 bytes in a row of the tile
    static constexpr int LOADS = BYTES / 16 / THREADS;
    static constexpr int STEP = THREADS / PIECES;                       // rows between a thread's loads
    static_assert(STEP % (ALONG ? 16 : 4) == 0, "a thread's pieces are turned alike");

    static __device__ __forceinline__ int turn(int row) { return ALONG ? row >> 1 & 7 : (row & 3) << 2; }
    static __device__ __forceinline__ int row_of(int i) { return threadIdx.x / PIECES + i * STEP; }
    static __device__ __forceinline__ int piece_of(int i) { return (threadIdx.x % PIECES) ^ turn(row_of(i)); }

    static __device__ __forceinline__ void load(lds_char *tile, int wave, int i, const char *from)
    {
        lds_char *to = tile + (i * THREADS + wave * 64) * 16;
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
            const int k = 8 * (lane >> 5) + ((lane >> 2) & 3);
            const int piece = (row0 >> 3) + ((lane >> 3) & 2) + ((lane >> 1) & 1);
            const lds_char *p = tile + ((piece ^ turn(k)) << 4) + (lane & 1) * 8 + (k + 16 * step) * (ROWS * 2);
            const s16x4 lo = read_turned((lds_s16x4 *)p);
            const s16x4 hi = read_turned((lds_s16x4 *)(p + 4 * ROWS * 2));
            const u32x2 u = __builtin_bit_cast(u32x2, lo), w = __builtin_bit_cast(u32x2, hi);
            return u32x4{u[0], u[1], w[0], w[1]};
        }
    }
};

// The order that the scheduler gives a step: behind each product two reads of the next step's operands, so that the last
// of them arrive before they are needed, then the LOADS of a later tile.
template <int READS, int PRODUCTS, int LOADS = 0>
__device__ __forceinline__ void interleave()
{
    if constexpr (PRODUCTS > 0) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        constexpr int n = PRODUCTS == 1 ? READS : READS < 2 ? READS : 2;
        constexpr int loads = READS - n > 0 ? 0 : (LOADS + PRODUCTS - 1) / PRODUCTS;
        if constexpr (n > 0) __builtin_amdgcn_sched_group_barrier(0x100, n, 0);
        if constexpr (loads > 0) __builtin_amdgcn_sched_group_barrier(0x010, loads, 0);
        interleave<READS - n, PRODUCTS - 1, LOADS - loads>();
    }
}

// Until at most LEFT of the wave's loads (and stores) are on their way.
template <int LEFT>
__device__ __forceinline__ void wait_loads()
{
    constexpr int n = LEFT < 63 ? LEFT : 63;
    __builtin_amdgcn_s_waitcnt(0x0f70 | (n & 15) | (n >> 4) << 14);
}

// GATHER: row r is token rows[r] / k of x; DX: the result goes to scratch, in fp32.
template <int DT, int FORM, bool GATHER, int BM, int BN, int WM, int WN, int BK, int STAGES>
__global__ __launch_bounds__(WM *WN * 64, 2) void product_kernel(ProductArgs a, int m_tiles, int n_tiles)
{
    constexpr int THREADS = WM * WN * 64, MI = BM / WM / 32, NI = BN / WN / 32;
    using OpA = Operand<BM, FORM != DWEIGHT, THREADS, BK>;
    using OpB = Operand<BN, FORM == FORWARD, THREADS, BK>;
    __shared__ __attribute__((aligned(256))) char lds[STAGES * (OpA::BYTES + OpB::BYTES) + WM * WN * 4096];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const char *const zeros = (const char *)ZEROS;
    const int N = FORM == FORWARD ? a.out : a.in;

    Tiles tiles;
    tiles.experts = a.experts;
    tiles.slots = (int)a.slots;
    tiles.m_tiles = m_tiles;
    tiles.n_tiles = n_tiles;
    if constexpr (FORM == DWEIGHT) tiles.share((uint32_t)m_tiles * n_tiles * a.experts);
    else tiles.of_rows(a.offsets, BM);
    auto find = [&](Tile &t) {
        if constexpr (FORM == DWEIGHT) return tiles.next_of_weights(a.offsets, t);
        else return tiles.next_of_rows(a.offsets, BM, t);
    };
    auto height = [&](const Tile &t) { return FORM == DWEIGHT ? a.out : t.last - t.first; };
    auto depth = [&](const Tile &t) {
        if constexpr (FORM == DWEIGHT) return t.last - t.first;
        else return t.expert == a.experts ? 0 : FORM == FORWARD ? a.in : a.out;
    };

    // Where each thread's pieces come from, k first, and the k that a piece stands for.  Rows of memory along k are clamped to
    // the last, those across k to the first column (and lie STEP rows apart: one pointer for all of a thread's pieces).
    const char *pa[FORM == DWEIGHT ? 1 : OpA::LOADS], *pb[FORM == FORWARD ? OpB::LOADS : 1];
    int sa[OpA::LOADS], sb[OpB::LOADS];
#pragma unroll
    for (int i = 0; i < OpA::LOADS; i++) sa[i] = FORM == DWEIGHT ? OpA::row_of(i) : OpA::piece_of(i) * 8;
#pragma unroll
    for (int i = 0; i < OpB::LOADS; i++) sb[i] = FORM == FORWARD ? OpB::piece_of(i) * 8 : OpB::row_of(i);
    // With GATHER, the slots of the rows that are needed next, on their way: FORWARD those of a tile of A, DWEIGHT those of the k
    // that is fetched next.  (A slot becomes a token only where it is needed: here it would have to arrive first, behind
    // all loads that were issued before it.)
    constexpr bool AHEAD = GATHER && FORM != DX;
    int ahead[FORM == DWEIGHT ? OpB::LOADS : OpA::LOADS];
    auto row_of_a = [&](const Tile &t, int i) { return t.first + min(t.m * BM + OpA::row_of(i), t.last - t.first - 1); };
    auto look_ahead = [&](const Tile &t, int K, int k0) {
        if constexpr (AHEAD && FORM == DWEIGHT) {
            if (K == 0) return;
#pragma unroll
            for (int i = 0; i < OpB::LOADS; i++) ahead[i] = a.rows[t.first + min(k0 + sb[i], K - 1)];
        } else if constexpr (AHEAD) {
#pragma unroll
            for (int i = 0; i < OpA::LOADS; i++) ahead[i] = a.rows[row_of_a(t, i)];
        }
    };
    auto aim = [&](const Tile &t) {
        const int m0 = t.m * BM, n0 = t.n * BN;
        const char *const weight = (const char *)a.weight + (t.expert == a.experts ? 0 : (int64_t)t.expert * a.weight_expert_stride) * 2;
        if constexpr (FORM == DWEIGHT) {
            const int col = m0 + OpA::piece_of(0) * 8;
            pa[0] = (const char *)a.dy + ((t.first + sa[0]) * a.dy_stride + (col < a.out ? col : 0)) * 2;
        } else
#pragma unroll
            for (int i = 0; i < OpA::LOADS; i++)
                if constexpr (AHEAD) pa[i] = (const char *)a.x + (token_of(a, ahead[i]) * a.x_stride + sa[i]) * 2;
                else if constexpr (FORM == FORWARD) pa[i] = (const char *)a.x + (row_of_a(t, i) * a.x_stride + sa[i]) * 2;
                else pa[i] = (const char *)a.dy + (row_of_a(t, i) * a.dy_stride + sa[i]) * 2;
        if constexpr (FORM == FORWARD) {
#pragma unroll
            for (int i = 0; i < OpB::LOADS; i++) pb[i] = weight + (min(n0 + OpB::row_of(i), N - 1) * a.weight_row_stride + sb[i]) * 2;
        } else {
            const int col = n0 + OpB::piece_of(0) * 8, at = col < N ? col : 0;
            if constexpr (FORM == DX) pb[0] = weight + (sb[0] * a.weight_row_stride + at) * 2;
            else pb[0] = (const char *)a.x + ((AHEAD ? 0 : (t.first + sb[0]) * a.x_stride) + at) * 2;
        }
    };
    // (what lies behind the end of k is ZEROS, so that no step of the loop branches)
    auto fetch = [&](int K, int k0, int buffer) {
        lds_char *la = (lds_char *)lds + buffer * (OpA::BYTES + OpB::BYTES), *lb = la + OpA::BYTES;
#pragma unroll
        for (int i = 0; i < OpA::LOADS; i++) {
            const char *p = pa[FORM == DWEIGHT ? 0 : i];
            p += FORM == DWEIGHT ? (k0 + i * OpA::STEP) * a.dy_stride * 2 : (int64_t)k0 * 2;
            OpA::load(la, wave, i, k0 + sa[i] < K ? p : zeros);
        }
#pragma unroll
        for (int i = 0; i < OpB::LOADS; i++) {
            const char *p = pb[FORM == FORWARD ? i : 0];
            if constexpr (FORM == DWEIGHT) p += (AHEAD ? token_of(a, ahead[i]) : k0 + i * OpB::STEP) * a.x_stride * 2;
            else p += FORM == FORWARD ? (int64_t)k0 * 2 : (k0 + i * OpB::STEP) * a.weight_row_stride * 2;
            OpB::load(lb, wave, i, k0 + sb[i] < K ? p : zeros);
        }
    };

    f32x16 acc[NI][MI];
    const int wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);
    u32x4 fa[2][MI], fb[2][NI];
    auto read = [&](int buffer, int step, int set) {
        const lds_char *la = (const lds_char *)lds + buffer * (OpA::BYTES + OpB::BYTES), *lb = la + OpA::BYTES;
#pragma unroll
        for (int i = 0; i < NI; i++) fb[set][i] = OpB::read(lb, wn + 32 * i, step);
#pragma unroll
        for (int j = 0; j < MI; j++) fa[set][j] = OpA::read(la, wm + 32 * j, step);
    };
    auto multiply = [&](int set) {
#pragma unroll
        for (int i = 0; i < NI; i++)
#pragma unroll
            for (int j = 0; j < MI; j++) acc[i][j] = mma<DT>(fb[set][i], fa[set][j], acc[i][j]);
    };
    constexpr int STEPS = BK / 16;
    static_assert(STEPS % 2 == 0, "the sets of operands alternate");
    // All loads into the buffer that is read next have arrived, and everybody has read the one that is filled next.  `behind`:
    // the wave's stores of the tile before, which were issued behind those loads and need not have arrived.
    constexpr int STAGE = OpA::LOADS + OpB::LOADS;
    auto arrive = [&, &ahead = ahead]<int LEFT>(int behind) {
        constexpr int WIDE = MI * NI * 4, NARROW = MI * 4;
        if (behind == WIDE) wait_loads<LEFT + WIDE>();
        else if (behind == NARROW) wait_loads<LEFT + NARROW>();
        else wait_loads<LEFT>();
        __syncthreads();
        if constexpr (FORM == DWEIGHT && GATHER)
#pragma unroll
            for (int i = 0; i < OpB::LOADS; i++) asm volatile("" : "+v"(ahead[i]));        // (not looked at any earlier)
    };
    constexpr int READS = MI * (FORM == DWEIGHT ? 2 : 1) + NI * (FORM == FORWARD ? 1 : 2);
    auto steps = [&](int buffer) {
#pragma unroll
        for (int s = 0; s + 1 < STEPS; s++) {
            read(buffer, s + 1, (s + 1) & 1);
            multiply(s & 1);
            interleave<READS, MI * NI>();
        }
    };

    // The first buffers of a tile, filled; ahead is what look_ahead gave for it.
    auto begin = [&](const Tile &t) {
        const int K = depth(t);
        aim(t);
        if (K == 0) return;
#pragma unroll
        for (int i = 0; i < STAGES; i++) {
            fetch(K, i * BK, i);
            if constexpr (FORM == DWEIGHT) look_ahead(t, K, (i + 1) * BK);
        }
    };

    // The operands of each step are read during the products of the one before.  The barrier lies ahead of a buffer's last
    // products: by then its operands are all in registers, so it takes a later k, and the first operands of the next
    // buffer are read during the last products of this one.
    Tile t, then;
    if (!find(t)) return;
    look_ahead(t, depth(t), 0);
    begin(t);
    int behind = 0;
    for (bool more = true; more; t = then) {
#pragma unroll
        for (int i = 0; i < NI; i++)
#pragma unroll
            for (int j = 0; j < MI; j++)
#pragma unroll
                for (int r = 0; r < 16; r++) acc[i][j][r] = 0.0f;
        const int K = depth(t), m0 = t.m * BM, n0 = t.n * BN, M = height(t);
        const bool idle = m0 + wm >= M;            // a wave whose rows all lie behind the last one only fetches
        if (FORM == DWEIGHT && GATHER) behind = 0;            // (the loads of rows lie between those of the buffers)
        int buffer = 0;
        if (K > 0) arrive.template operator()<(STAGES - 1) * STAGE>(behind);
        if (idle) {
            for (int k0 = BK; k0 < K; k0 += BK) {
                arrive.template operator()<(STAGES - 2) * STAGE>(0);
                fetch(K, k0 + (STAGES - 1) * BK, buffer);
                if constexpr (FORM == DWEIGHT) look_ahead(t, K, k0 + STAGES * BK);
                buffer = buffer + 1 == STAGES ? 0 : buffer + 1;
            }
            more = find(then);
            if (more) look_ahead(then, depth(then), 0);
        } else if (K > 0) {
            read(0, 0, 0);
            for (int k0 = BK; k0 < K; k0 += BK) {
                steps(buffer);
                arrive.template operator()<(STAGES - 2) * STAGE>(behind);
                behind = 0;
                const int next = buffer + 1 == STAGES ? 0 : buffer + 1;
                read(next, 0, 0);
                fetch(K, k0 + (STAGES - 1) * BK, buffer);
                if constexpr (FORM == DWEIGHT) look_ahead(t, K, k0 + STAGES * BK);
                multiply((STEPS - 1) & 1);
                interleave<READS, MI * NI, STAGE>();
                buffer = next;
            }
            more = find(then);
            if (more) look_ahead(then, depth(then), 0);
            steps(buffer);
            multiply((STEPS - 1) & 1);
        } else {
            more = find(then);
            if (more) look_ahead(then, depth(then), 0);
        }
        // everybody has read the last buffer, and what was fetched behind the end of k is no longer on its way
        wait_loads<0>();
        __syncthreads();
        if (more) begin(then);
        __builtin_amdgcn_sched_barrier(0);         // (`behind` counts the stores as issued after these loads)

        // A lane holds row m = lane & 31 of a 32 x 32 block, columns 8 g + 4 (lane >> 5) + r.  The halves of a wave swap so that
        // each lane of a 16-bit result has 8 columns; 32 rows x 128 bytes then go through LDS, of which each wave has 4 KB, and
        // eight lanes store 128 bytes of a row (a line; stored as they lie, a quarter of a line each, they cost L2 four
        // times the requests).
        const int half = lane >> 5, store_row = lane >> 3, store_piece = lane & 7;
        const bool wide = FORM == DX ? GATHER : FORM == DWEIGHT ? a.dweight_f32 != 0 : false;
        const int64_t row0 = FORM == DWEIGHT ? (int64_t)t.expert * a.out : t.first;
        lds_char *const mine = (lds_char *)lds + STAGES * (OpA::BYTES + OpB::BYTES) + wave * 4096;
        auto store = [&](const u32x4 *v, int j, int n, char *to, int size) {
            // v[p]: 16 bytes, piece 2 p + half of this lane's row
#pragma unroll
            for (int p = 0; p < 4; p++)
                *(__attribute__((address_space(3))) u32x4 *)(mine + (lane & 31) * 128 + (((2 * p + half) ^ (lane >> 1 & 7)) << 4)) = v[p];
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int row = 8 * q + store_row, m = m0 + wm + 32 * j + row, at = n + store_piece * (16 / size);
                const u32x4 w = *(const __attribute__((address_space(3))) u32x4 *)(mine + row * 128 + ((store_piece ^ (row >> 1 & 7)) << 4));
                u32x4 *const place = (u32x4 *)(to + ((row0 + m) * N + at) * size);
                if (m < M && at < N) {
                    // (past the caches: left there they push out the operands.  60 skewed experts, 692 MB in fp32: 380 us against
                    // 485, with a clip_grads of them behind it 816 against 875; 25 MB in bf16, which a cache could keep for that
                    // clip_grads: 78 against 77)
                    if constexpr (FORM == DWEIGHT) __builtin_nontemporal_store(w, place);
                    else *place = w;
                }
            }
        };
        if (!idle) {
            if (wide) {
                char *const to = (char *)(FORM == DX ? (void *)a.scratch : a.dweight);
#pragma unroll
                for (int j = 0; j < MI; j++)
#pragma unroll
                    for (int i = 0; i < NI; i++) {
                        u32x4 v[4];
#pragma unroll
                        for (int g = 0; g < 4; g++)
#pragma unroll
                            for (int r = 0; r < 4; r++) v[g][r] = __float_as_uint(acc[i][j][4 * g + r]);
                        store(v, j, n0 + wn + 32 * i, to, 4);
                    }
            } else {
                static_assert(NI == 2, "128 bytes of a row");
                char *const to = (char *)(FORM == FORWARD ? a.y : FORM == DX ? a.dx : a.dweight);
#pragma unroll
                for (int j = 0; j < MI; j++) {
                    u32x4 v[4];
#pragma unroll
                    for (int i = 0; i < NI; i++)
#pragma unroll
                        for (int g = 0; g < 4; g += 2)
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                const auto w = __builtin_amdgcn_permlane32_swap(pack2<DT>(acc[i][j][4 * g + 2 * h], acc[i][j][4 * g + 2 * h + 1]),
                                                                                pack2<DT>(acc[i][j][4 * g + 4 + 2 * h], acc[i][j][4 * g + 5 + 2 * h]), false, false);
                                v[2 * i + g / 2][h] = w[0];
                                v[2 * i + g / 2][2 + h] = w[1];
                            }
                    store(v, j, n0 + wn, to, 2);
                }
            }
        }
        // (stores that no lane makes are not issued: of a tile that is not full they are waited for)
        behind = m0 + BM <= M && n0 + BN <= N ? wide ? MI * NI * 4 : MI * 4 : 0;
        __builtin_amdgcn_sched_barrier(0);
    }
}

template <int DT, int FORM, bool GATHER, int BM, int BN, int WM, int WN, int BK, int STAGES>
hipError_t launch(const ProductArgs &a, hipStream_t stream)
{
    const int n = FORM == FORWARD ? a.out : a.in;
    const int64_t n_tiles = (n + BN - 1) / BN;
    const int64_t m_tiles = FORM == DWEIGHT ? (a.out + BM - 1) / BM : 0;
    // each expert, and the rows of none, may end with a tile that is not full
    const int64_t parts = a.slots < a.experts + 1 ? a.slots : a.experts + 1;
    int64_t tiles = FORM == DWEIGHT ? a.experts * m_tiles * n_tiles : (a.slots / BM + parts) * n_tiles;
    if (tiles == 0) return hipSuccess;
    // as many workgroups as the 256 CUs hold, an eighth of them on each XCD
    constexpr int RESIDENT = 256 * (160 * 1024 / (STAGES * (BM + BN) * BK * 2 + WM * WN * 4096));
    tiles = (tiles + 7) / 8 * 8;
    product_kernel<DT, FORM, GATHER, BM, BN, WM, WN, BK, STAGES><<<(unsigned)(tiles < RESIDENT ? tiles : RESIDENT), WM * WN * 64, 0, stream>>>(a, (int)m_tiles, (int)n_tiles);
    return hipGetLastError();
}

// Forward for few rows an expert (decoding): the weights are read once and bound it.  A workgroup has 16 rows and 32 columns;
// its four waves share k, 64 at a time, read their operands of 16x16x32 products straight from memory (a line of each weight
// row at a time, FLY of them in flight) and add their sums in LDS in the order of the waves.  1 token, 2 of 8 experts of
// 4096 x 11008: 38 to 40 us, 4.5 TB/s, with other weights read in between; 29.8 where the last-level cache still holds them in part
// (tiles of 128: 65).  Narrow experts are bound by the dependent reads ahead of the weights (row counts, slot, row), which one
// trip of loads follows: 37 tokens, 2 of 16 experts of 768 x 2048, 12.5 us for about 40 MB.  Up to 8 rows an expert on average: at 8 153 us against 163 with
// tiles of 128 for 4096 x 11008, at 16 205 against 163.
constexpr int FEW_M = 16, FEW_N = 32;

template <int DT>
__device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c)
{
    if constexpr (DT == DT_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <int DT, bool GATHER>
__global__ __launch_bounds__(256) void product_few_kernel(ProductArgs a, int n_tiles)
{
    constexpr int FLY = 4;
    __shared__ f32x4 sums[3][2][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Tiles tiles;
    tiles.experts = a.experts;
    tiles.slots = (int)a.slots;
    tiles.m_tiles = 0;
    tiles.n_tiles = n_tiles;
    tiles.of_rows(a.offsets, FEW_M);
    for (Tile t; tiles.next_of_rows(a.offsets, FEW_M, t); __syncthreads()) {
        const int m = t.m * FEW_M + (lane & 15), n0 = t.n * FEW_N, piece = (lane >> 4) * 8;
        const bool here = t.first + m < t.last;
        f32x4 acc[2] = {};
        if (t.expert < a.experts) {
            const char *const x = (const char *)a.x + (here ? source_row<GATHER>(a, t.first + m) * a.x_stride + piece : 0) * 2;
            const char *w[2];
#pragma unroll
            for (int i = 0; i < 2; i++)
                w[i] = (const char *)a.weight + ((int64_t)t.expert * a.weight_expert_stride + min(n0 + 16 * i + (lane & 15), a.out - 1) * a.weight_row_stride + piece) * 2;
            for (int k0 = wave * 64; k0 < a.in; k0 += 256 * FLY) {
                u32x4 fx[FLY][2], fw[FLY][2][2];
#pragma unroll
                for (int u = 0; u < FLY; u++)
#pragma unroll
                    for (int s = 0; s < 2; s++) {
                        const int k = k0 + 256 * u + 32 * s;
                        const bool in = k + piece < a.in;
#pragma unroll
                        for (int i = 0; i < 2; i++) fw[u][s][i] = in ? *(const u32x4 *)(w[i] + k * 2) : u32x4{};
                        fx[u][s] = in && here ? *(const u32x4 *)(x + k * 2) : u32x4{};
                    }
#pragma unroll
                for (int u = 0; u < FLY; u++)
#pragma unroll
                    for (int s = 0; s < 2; s++)
#pragma unroll
                        for (int i = 0; i < 2; i++) acc[i] = mma16<DT>(fw[u][s][i], fx[u][s], acc[i]);
            }
        }
        if (wave)
#pragma unroll
            for (int i = 0; i < 2; i++) sums[wave - 1][i][lane] = acc[i];
        __syncthreads();
        if (wave || !here) continue;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const f32x4 v = ((acc[i] + sums[0][i][lane]) + sums[1][i][lane]) + sums[2][i][lane];
            const int n = n0 + 16 * i + 4 * (lane >> 4);
            const float f[4] = {v[0], v[1], v[2], v[3]};
            if (n < a.out) store_n<DT, 4>(a.y, (int64_t)(t.first + m) * a.out + n, f);
        }
    }
}

template <int DT, bool GATHER>
hipError_t launch_few(const ProductArgs &a, hipStream_t stream)
{
    const int64_t n_tiles = (a.out + FEW_N - 1) / FEW_N, parts = a.slots < a.experts + 1 ? a.slots : a.experts + 1;
    constexpr int64_t MOST = 1 << 16;          // (each takes several tiles then)
    const int64_t wgs = ((a.slots / FEW_M + parts) * n_tiles + 7) / 8 * 8;
    product_few_kernel<DT, GATHER><<<(unsigned)(wgs < MOST ? wgs : MOST), 256, 0, stream>>>(a, (int)n_tiles);
    return hipGetLastError();
}

// Tiles of 256 x 256 where they are enough to fill most of the chip and, of rows, mostly full: 512 rows an expert, or 256 where
// k is long enough to make up for a tile's beginning and end.  Tiles of 128 x 128 (two workgroups a CU) otherwise.
// Measured, us, 256 against 128 (dx with its tokens' sums):
//   8 experts of 4096 x 11008   forward              dx                   dweight
//     128 rows an expert        217, 225             275, 215             197, 242
//     256                       247, 295             318, 386             276, 343
//     1024                      764, 888             928, 977             722, 952
//   8 experts of 768 x 2048
//     256                       21, 16               52, 31               15, 15
//     1024                      42, 38               55, 41               31, 37
//     2048                      67, 67               67, 77               53, 66
//   60 experts of 1408 x 2048, skewed
//     233                       156, 145             169, 147             172, 181
//     273, evenly               170, 156             180, 154             150, not timed
//     930                       394, 440             412, 424             583, 576
// (The rule does not follow every line: 8 experts of 768 x 2048 at 1024 rows go forward in tiles of 256, 42 us against 38.)
template <int DT, int FORM, bool GATHER>
hipError_t pick(const ProductArgs &a, hipStream_t stream)
{
    const int64_t in_tiles = (a.in + 255) / 256, out_tiles = (a.out + 255) / 256, rows_of_tiles = a.slots / 256 + a.experts / 2;
    if constexpr (FORM == FORWARD)
        if (a.slots <= 8 * (int64_t)a.experts) return launch_few<DT, GATHER>(a, stream);
    const int64_t full = (FORM == FORWARD ? a.in : a.out) >= 4096 ? 256 : 512;
    const bool large = FORM == DWEIGHT ? a.experts * in_tiles * out_tiles >= 128
                                       : a.slots >= full * a.experts && rows_of_tiles * (FORM == FORWARD ? out_tiles : in_tiles) >= 192;
    if (large) return launch<DT, FORM, GATHER, 256, 256, 2, 4, 64, 2>(a, stream);
    return launch<DT, FORM, GATHER, 128, 128, 2, 2, 64, 2>(a, stream);
}

}  // namespace

template <int DT>
hipError_t product_forward(const ProductArgs &a, hipStream_t stream)
{
    return a.k ? pick<DT, FORWARD, true>(a, stream) : pick<DT, FORWARD, false>(a, stream);
}

template <int DT>
hipError_t product_backward(const ProductArgs &a, hipStream_t stream)
{
    if (a.dx) {
        hipError_t e = a.k ? pick<DT, DX, true>(a, stream) : pick<DT, DX, false>(a, stream);
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
    if (!a.dweight) return hipSuccess;
    return a.k ? pick<DT, DWEIGHT, true>(a, stream) : pick<DT, DWEIGHT, false>(a, stream);
}

}  // namespace lm
