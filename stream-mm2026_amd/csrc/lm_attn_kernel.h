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
// LDS tiles are row major, 16-byte pieces XOR-ed with their row: sixteen lanes of a row read (16 rows,
// one piece each) and sixteen of a transposing read (4 rows x 2 pieces) then fall on different ones
// of the 64 banks (with 32 bytes between rows instead the row reads took twice the cycles).  Tiles
// come in pairs, one read while the other is filled: one barrier a tile.
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
constexpr int FEW = 8;                          // parts of the keys that one wave joins
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
// The other half-wave's value of the same column, for a maximum or a sum of both.
template <typename F>
__device__ __forceinline__ float both_halves(float x, F op)
{
    const uint32_t w = __builtin_bit_cast(uint32_t, x);
    const auto h = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return op(__uint_as_float(h[0]), __uint_as_float(h[1]));
}

// A tile of rows of HD 16-bit elements in LDS, aligned to its rows.  `t` is the tile's offset in LDS.
typedef __attribute__((address_space(3))) char lds_char;
template <int HD>
struct Tile {
    static constexpr int ROW = HD * 2;

    static __device__ __forceinline__ int turn(int row)
    {
        return (HD == 128 ? ((row & 7) << 1) | ((row >> 3) & 1) : (row & 6) | ((row >> 3) & 1)) << 4;
    }
    static __device__ __forceinline__ int at(int row, int piece) { return row * ROW + ((piece << 4) ^ turn(row)); }

    // A lane's place in the tile for each kind of read; what differs between reads are constants.
    static __device__ __forceinline__ int row_place(int lane) { return at(lane & 31, lane >> 5); }
    static __device__ __forceinline__ int column_place(int lane)
    {
        return at(4 * (lane >> 5) + ((lane >> 2) & 3), ((lane >> 3) & 2) + ((lane >> 1) & 1)) + (lane & 1) * 8;
    }
    // A operand, its k along the elements: row `row` + lane & 31, elements 16 c + 8 half ...
    static __device__ __forceinline__ u32x4 rows(const lds_char *t, int place, int row, int c)
    {
        return *(const __attribute__((address_space(3))) u32x4 *)(t + (place ^ (c << 5)) + row * ROW);
    }
    // A operand, its k along the rows: element 32 d + lane & 31 of the 16 rows from `row`, in the
    // order of a result's registers
    static __device__ __forceinline__ u32x4 columns(const lds_char *t, int place, int row, int d)
    {
        typedef __attribute__((address_space(3))) s16x4 *lds4;
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(t + (place ^ (d << 6)) + row * ROW));
        const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(t + (place ^ (d << 6 | 16)) + (row + 8) * ROW));
        const u32x2 u = __builtin_bit_cast(u32x2, x), w = __builtin_bit_cast(u32x2, y);
        return u32x4{u[0], u[1], w[0], w[1]};
    }
};

// 8 results (registers r0 .. r0 + 7) rounded to the B operand of 16 k: the matrix instructions take 16 bits.  Weights
// and score gradients as two parts each in every tile would make the outputs those of products in fp32 (errors 1.00
// to 1.02 times theirs; so 1.22 to 1.40) and took 161 us in place of 141 (8 x 12 x 1024 of 64, with gradients), 1805 in
// place of 1332 (8192 positions of 32 heads of 128, window 2048) and 157 in place of 122 (fp16, ragged).
template <int DT>
__device__ __forceinline__ u32x4 operand(const f32x16 &s, int r0)
{
    return u32x4{pack2<DT>(s[r0], s[r0 + 1]), pack2<DT>(s[r0 + 2], s[r0 + 3]), pack2<DT>(s[r0 + 4], s[r0 + 5]),
                 pack2<DT>(s[r0 + 6], s[r0 + 7])};
}

// The weights of fp16 are multiplied by 2^14 before they are rounded, which the sums give back: they are at most 1,
// and over n keys about 1 / n, of which fp16 holds ever fewer bits below 2^-14 (dv of 200,000 keys: off by 0.20 %,
// 0.02 % so).
template <int DT>
constexpr float RAISE = DT == DT_F16 ? 14.0f : 0.0f;

// What that rounding left, as an operand of its own.  Rows that see few keys have the largest score
// gradients, and the tiles in which they see them are not all visible: only there dS is multiplied as
// two parts (dq of 8 x 12 x 1024 of 64: 1.49 times the error of a product in fp32 before, 1.35 with it for
// 2 us of 37, and 1.27 with delta as below).
template <int DT>
__device__ __forceinline__ u32x4 remainder(const f32x16 &s, int r0, u32x4 rounded)
{
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const f32x2 x = unpack2<DT>(rounded[i]);
        o[i] = pack2<DT>(s[r0 + 2 * i] - x[0], s[r0 + 2 * i + 1] - x[1]);
    }
    return o;
}

// fp16 holds fewer bits below 2^-14, and a score gradient is about |dout| / keys: rounded as it is, dq of 4500
// keys with dout of 1e-3 was off by 0.5 % (0.07 % is its own rounding).  Each column is therefore multiplied by a
// power of two that keeps its largest score gradient so far within 2^13 .. 2^15, and the sums with it; the power
// goes out of them at the end.  Like a running maximum it is looked at every tile and seldom changes.  bfloat16
// has the exponents of fp32 and needs none of this.
template <int DT>
struct Lift {
    static constexpr bool ON = DT == DT_F16;
    float up = ON ? 0x1p60f : 1.0f;                // down to dout's and the weights' smallest; no float overflows

    template <int ND>
    __device__ __forceinline__ void fit(f32x16 &ds, f32x16 (&sums)[ND])
    {
        if constexpr (ON) {
            float top = 0.0f;
#pragma unroll
            for (int r = 0; r < 16; r++) {
                ds[r] *= up;
                top = fmaxf(top, fabsf(ds[r]));
            }
            top = both_halves(top, [](float x, float y) { return fmaxf(x, y); });
            if (__ballot(top > 0x1p15f)) {
                // (an infinite one stays what it is)
                const bool over = top > 0x1p15f && top < __builtin_inff();
                const float by = over ? __builtin_ldexpf(1.0f, 14 - __builtin_amdgcn_frexp_expf(top)) : 1.0f;
                up *= by;
#pragma unroll
                for (int r = 0; r < 16; r++) ds[r] *= by;
#pragma unroll
                for (int d = 0; d < ND; d++)
#pragma unroll
                    for (int r = 0; r < 16; r++) sums[d][r] *= by;
            }
        }
    }
    __device__ __forceinline__ float down() const { return 1.0f / up; }      // (exact: a power of two)
};

// Waits for loaded registers here.  Loads that are first used inside a loop are otherwise waited for
// there, on every turn, and with them the loop's own loads for its next turn.
template <int N>
__device__ __forceinline__ void landed(u32x4 (&v)[N])
{
#pragma unroll
    for (int i = 0; i < N; i++) asm volatile("" : "+v"(v[i]));
}

// The row of a result's register r within its 32.
__device__ __forceinline__ int result_row(int r, int lane) { return 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3); }

// What a row at position p sees, and what a block of rows sees of a block of keys.
struct Sight {
    int window, sinks;
    __device__ __forceinline__ bool one(int p, int j) const { return (j <= p) & ((p - j < window) | (j < sinks)); }
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

// A buffer descriptor over the memory from p on: 32-bit byte offsets, and an offset of 2^31 and more
// reads zeros without touching memory.
constexpr uint32_t NOWHERE = 0x80000000u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_from(const void *p)
{
    return __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, NOWHERE, 0x00027000);
}

// Which of a lane's 16 results its row at position p sees: bit r for key + result_row(r), of the 32
// keys from `key` on that `shown` shows.
__device__ __forceinline__ uint32_t visible16(const Sight &sight, int p, int key, uint32_t shown, int lane)
{
    uint32_t bits = 0;
    shown >>= 4 * (lane >> 5);
    key += 4 * (lane >> 5);
#pragma unroll
    for (int r = 0; r < 16; r++) {
        const int j = 8 * (r >> 2) + (r & 3);
        bits |= (uint32_t)(sight.one(p, key + j) & (bool)(shown >> j & 1)) << r;
    }
    return bits;
}

__device__ __forceinline__ void hide(f32x16 &s, uint32_t visible)
{
#pragma unroll
    for (int r = 0; r < 16; r++) s[r] = (visible >> r & 1) ? s[r] : -__builtin_inff();
}

// THREADS threads bring a tile of ROWS rows from memory to LDS by way of registers: load(), then
// store() once the tile's last readers are done.  A piece at NOWHERE is zero: rows that are not
// there, elements from dim on, and masked keys, which may hold anything and must not meet a weight
// of zero.
template <int HD, int THREADS, int ROWS>
struct Stage {
    static constexpr int N = ROWS * HD / 8 / THREADS, STEP = THREADS * 8 / HD;      // rows between a thread's pieces
    u32x4 v[N];

    static __device__ __forceinline__ int row() { return threadIdx.x / (HD / 8); }
    static __device__ __forceinline__ int piece() { return threadIdx.x % (HD / 8); }
    template <typename Offset>
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t from, Offset offset)
    {
#pragma unroll
        for (int i = 0; i < N; i++)
            v[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(from, offset(i), 0, 0));
    }
    __device__ __forceinline__ void store(lds_char *tile) const
    {
#pragma unroll
        for (int i = 0; i < N; i++) {
            // (STEP rows on, the row's turn is the same where STEP is a multiple of 16)
            const int at = STEP % 16 ? Tile<HD>::at(row() + i * STEP, piece()) : Tile<HD>::at(row(), piece()) + i * STEP * Tile<HD>::ROW;
            *(__attribute__((address_space(3))) u32x4 *)(tile + at) = v[i];
        }
    }
};

// A tile of 64 keys: its rows of k and v, and which of them are shown.
template <int HD, int THREADS>
struct KeyStage {
    using S = Stage<HD, THREADS, TILE>;
    S k, v;
    uint32_t mask;                 // the mask's byte of key `lane`; looked at in store(), when it has come

    __device__ __forceinline__ void load(const AttnArgs &a, int b, int hk, int key)
    {
        const int left = a.keys - key;
        if (a.key_mask) {
            const int j = threadIdx.x & 63;
            mask = j < left ? a.key_mask[b * a.mask_stride + key + j] : 0;
        }
        const auto kr = buffer_from((const uint16_t *)a.k.p + b * a.k.b + hk * a.k.h + key * a.k.t);
        const auto vr = buffer_from((const uint16_t *)a.v.p + b * a.v.b + hk * a.v.h + key * a.v.t);
        const int row = S::row(), d = S::piece() * 8;
        const uint32_t kt = (uint32_t)a.k.t * 2, vt = (uint32_t)a.v.t * 2;
        const uint32_t ko = d < a.dim ? row * kt + d * 2 : NOWHERE, vo = d < a.dim ? row * vt + d * 2 : NOWHERE;
        if (left >= TILE) {
            k.load(kr, [&](int i) { return ko + i * S::STEP * kt; });
            v.load(vr, [&](int i) { return vo + i * S::STEP * vt; });
        } else {
            k.load(kr, [&](int i) { return row + i * S::STEP < left ? ko + i * S::STEP * kt : NOWHERE; });
            v.load(vr, [&](int i) { return row + i * S::STEP < left ? vo + i * S::STEP * vt : NOWHERE; });
        }
    }
    // Returns which keys are shown; the hidden ones' rows are zero.
    __device__ __forceinline__ uint64_t store(const AttnArgs &a, lds_char *ktile, lds_char *vtile)
    {
        const uint64_t see = a.key_mask ? __ballot(mask != 0) : ~0ull;
        if (see != ~0ull) {
#pragma unroll
            for (int i = 0; i < S::N; i++)
                if (!(see >> (S::row() + i * S::STEP) & 1)) k.v[i] = v.v[i] = u32x4{0, 0, 0, 0};
        }
        k.store(ktile);
        v.store(vtile);
        return see;
    }
};

__device__ __forceinline__ const uint16_t *at(const AttnTensor &t, int b, int h) { return (const uint16_t *)t.p + b * t.b + h * t.h; }

// ---------------------------------------------------------------- forward
// WAVES x 32 rows; the keys in tiles of 64, or the share of them that blockIdx.z takes.  Bound by the waves'
// issue: per score two products of the head size against one exponential and about six vector instructions,
// so most of a tile's cycles are the softmax's.  A maximum that does not grow skips the rescaling.  Tiles of
// up to 32 rows run as one wave, where latency counts.  Window 2048 with 4 sinks over 8192 positions, 32
// heads of 128 on 8 of keys, bf16: 300-310 us, 0.8 PFLOP/s of visible products; 12 heads of 64, 8 x 1024
// causal: 30 us.
template <int DT, int HD, int WAVES>
__global__ __launch_bounds__(WAVES * 64, WAVES == 1 ? 1 : HD == 64 ? 3 : 2) void attn_fwd_kernel(AttnArgs a)
{
    constexpr int C = HD / 16, ND = HD / 32;
    constexpr int BYTES = TILE * Tile<HD>::ROW;
    __shared__ __attribute__((aligned(256))) char lds_[4 * BYTES];          // k, v; k, v of the next tile
    lds_char *const lds = (lds_char *)lds_;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = blockIdx.x / a.key_heads, hk = blockIdx.x % a.key_heads;
    const int total = a.rows * a.group, r0 = (gridDim.y - 1 - blockIdx.y) * WAVES * 32, row = r0 + wave * 32 + (lane & 31);
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

    landed(q);
    f32x16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) o[d] = zero16();
    float m = -__builtin_inff(), l = 0.0f;         // in units of log2; l of this lane's keys alone, and raised
    const float c2 = a.scale * LOG2E;
    KeyStage<HD, WAVES * 64> next;
    int rp = Tile<HD>::row_place(lane), cp = Tile<HD>::column_place(lane);
    uint64_t see = 0;
    int turn = 0;                                  // the tile being read
    if (it0 < it1) {
        next.load(a, b, hk, tiles.key(it0));
        see = next.store(a, lds, lds + BYTES);
        if (it0 + 1 < it1) next.load(a, b, hk, tiles.key(it0 + 1));
    }
    __syncthreads();
    for (int it = it0; it < it1; it++) {
        const int key = tiles.key(it);
        const lds_char *kt = lds + turn, *vt = kt + BYTES;
        asm volatile("" : "+v"(rp), "+v"(cp));     // the reads' addresses are formed where they are used, not kept
        if (see != 0 && !sight.none(pa, pb, key, key + TILE - 1)) {
            f32x16 s[2] = {zero16(), zero16()};
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int n = 0; n < 2; n++) s[n] = mma<DT>(Tile<HD>::rows(kt, rp, 32 * n, c), q[c], s[n]);
            if (see != ~0ull || !sight.all(pa, pb, key, key + TILE - 1)) {
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    const uint32_t bits = visible16(sight, pos, key + 32 * n, (uint32_t)(see >> (32 * n)), lane);
                    hide(s[n], bits);
                }
            }
            float top = s[0][0];
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int r = 0; r < 16; r++) top = fmaxf(top, s[n][r]);
            top = both_halves(top, [](float x, float y) { return fmaxf(x, y); }) * c2;
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
            const float ref = (m == -__builtin_inff() ? 0.0f : m) - RAISE<DT>;
            float sum = 0.0f;              // (added to l once a tile: beside a large l single weights would be lost)
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    s[n][r] = exp2_hw(__builtin_fmaf(s[n][r], c2, -ref));
                    sum += s[n][r];
                }
            l += sum;
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const u32x4 p = operand<DT>(s[n], 8 * k);
#pragma unroll
                    for (int d = 0; d < ND; d++) o[d] = mma<DT>(Tile<HD>::columns(vt, cp, 32 * n + 16 * k, d), p, o[d]);
                }
        }
        turn ^= 2 * BYTES;
        if (it + 1 < it1) {
            see = next.store(a, lds + turn, lds + turn + BYTES);
            if (it + 2 < it1) next.load(a, b, hk, tiles.key(it + 2));
        }
        __syncthreads();
    }
    l = both_halves(l, Add());
    m -= RAISE<DT>;                                // what the sums stand against
    if (!real) return;
    if (a.splits > 1) {
        // unnormalised sums, their maximum and weight, for the join
        const int64_t at_row = ((int64_t)blockIdx.z * gridDim.x + blockIdx.x) * total + row;
        float *po = a.partial + at_row * a.dim, *ml = a.partial + (int64_t)a.splits * gridDim.x * total * a.dim + at_row * 2;
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

// Joins the parts of the keys, where they are few: a wave a row, a lane 2 elements.
template <int DT>
__global__ __launch_bounds__(256) void attn_join_few_kernel(AttnArgs a)
{
    const int total = a.rows * a.group, lane = threadIdx.x & 63, row = blockIdx.y * 4 + (threadIdx.x >> 6);
    if (row >= total) return;
    const int b = blockIdx.x / a.key_heads, hk = blockIdx.x % a.key_heads;
    const int64_t rows = (int64_t)gridDim.x * total, at_row = (int64_t)blockIdx.x * total + row;
    const float *ml = a.partial + a.splits * rows * a.dim;
    const int e = 2 * lane;
    f32x2 p[FEW], v[FEW];
#pragma unroll
    for (int i = 0; i < FEW; i++) {
        p[i] = i < a.splits ? *(const f32x2 *)(ml + (i * rows + at_row) * 2) : f32x2{-__builtin_inff(), 0.0f};
        v[i] = i < a.splits && e < a.dim ? *(const f32x2 *)(a.partial + (i * rows + at_row) * a.dim + e) : f32x2{0.0f, 0.0f};
    }
    float m = p[0][0];
#pragma unroll
    for (int i = 1; i < FEW; i++) m = fmaxf(m, p[i][0]);
    const float ref = m == -__builtin_inff() ? 0.0f : m;
    float l = 0.0f, o0 = 0.0f, o1 = 0.0f;
#pragma unroll
    for (int i = 0; i < FEW; i++) {
        const float w = exp2_hw(p[i][0] - ref);
        l += w * p[i][1];
        o0 += w * v[i][0];
        o1 += w * v[i][1];
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int t = row / a.group, head = hk * a.group + row % a.group;
    if (e < a.dim) *(uint32_t *)((uint16_t *)at(a.o, b, head) + t * a.o.t + e) = pack2<DT>(o0 * inv, o1 * inv);
    if (lane == 0) a.lse[((int64_t)b * a.heads + head) * a.rows + t] = l == 0.0f ? -__builtin_inff() : (m + log2f(l)) * LN2;
}

// Joins many parts: a workgroup a row, its waves every fourth part, a lane 2 elements.
template <int DT>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a)
{
    __shared__ float weight[MAX_SPLITS], sums[4][128], buf[2][4];
    const int total = a.rows * a.group, row = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int b = blockIdx.x / a.key_heads, hk = blockIdx.x % a.key_heads;
    const int64_t rows = (int64_t)gridDim.x * total, at_row = (int64_t)blockIdx.x * total + row;
    const float *ml = a.partial + a.splits * rows * a.dim;
    const int z = threadIdx.x;                       // MAX_SPLITS = 2 x 256 parts at most
    f32x2 p[2];
#pragma unroll
    for (int i = 0; i < 2; i++)
        p[i] = z + 256 * i < a.splits ? *(const f32x2 *)(ml + ((z + 256 * i) * rows + at_row) * 2) : f32x2{-__builtin_inff(), 0.0f};
    const float m = group_reduce<4>(fmaxf(p[0][0], p[1][0]), [](float x, float y) { return fmaxf(x, y); }, buf[0]);
    const float ref = m == -__builtin_inff() ? 0.0f : m;
    float l = 0.0f;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const float w = exp2_hw(p[i][0] - ref);
        weight[z + 256 * i] = w;
        l += w * p[i][1];
    }
    l = group_reduce<4>(l, Add(), buf[1]);           // (its barrier also shows the weights)
    float o0 = 0.0f, o1 = 0.0f;
    const int e = 2 * lane;
    if (e < a.dim) {
#pragma unroll 8
        for (int i = wave; i < a.splits; i += 4) {
            const f32x2 v = *(const f32x2 *)(a.partial + (i * rows + at_row) * a.dim + e);
            o0 += weight[i] * v[0];
            o1 += weight[i] * v[1];
        }
        sums[wave][e] = o0;
        sums[wave][e + 1] = o1;
    }
    __syncthreads();
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int t = row / a.group, head = hk * a.group + row % a.group;
    if (wave == 0 && e < a.dim) {
        o0 = sums[0][e] + sums[1][e] + sums[2][e] + sums[3][e];
        o1 = sums[0][e + 1] + sums[1][e + 1] + sums[2][e + 1] + sums[3][e + 1];
        *(uint32_t *)((uint16_t *)at(a.o, b, head) + t * a.o.t + e) = pack2<DT>(o0 * inv, o1 * inv);
    }
    if (threadIdx.x == 0) a.lse[((int64_t)b * a.heads + head) * a.rows + t] = l == 0.0f ? -__builtin_inff() : (m + log2f(l)) * LN2;
}

// ---------------------------------------------------------------- backward
// delta = rowsum(dout * out): 16 lanes a row.  A row that sees up to FEW_KEYS keys takes sum P (do v^T) from
// them instead: `out` is rounded, and what that puts into delta falls with the number of keys, while the
// rounding of dS does not (a handful of positions: the error of dq 1.05 times that of products in fp32, 2.3
// before; 8 x 12 x 1024 of 64 10 us, 6 before; a wave a row in turn 38).  It is divided by the sum of the same
// weights, which lse's rounding leaves off 1: a weight of 1 - 2^-17 beside one of 2^-17 keeps its gradient.  A row
// that sees one key has no score gradient at all: its delta says LONE.
constexpr int FEW_KEYS = 16;
constexpr int DELTA_Y = 32768;                     // 16 rows each along the grid's second dimension, the rest along the third
constexpr uint32_t LONE = 0x7fc01e01u;             // a NaN of these bits
__device__ __forceinline__ bool is_lone(float delta) { return __builtin_bit_cast(uint32_t, delta) == LONE; }

template <int DT>
__global__ __launch_bounds__(256, 6) void attn_delta_kernel(AttnArgs a)
{
    __shared__ int list_[16][FEW_KEYS];
    const int lane = threadIdx.x & 63, part = lane & 15;
    // (the first rows of all heads first: they see the fewest keys and take longest)
    const int b = blockIdx.x / a.key_heads, hk = blockIdx.x % a.key_heads;
    const int total = a.rows * a.group, row = (blockIdx.z * DELTA_Y + blockIdx.y) * 16 + (threadIdx.x >> 4), rr = min(row, total - 1);
    if (row - (int)(threadIdx.x >> 4) >= total) return;
    const int t = rr / a.group, h = hk * a.group + rr % a.group, pos = a.keys - a.rows + t;
    const int64_t stat = ((int64_t)b * a.heads + h) * a.rows + t;
    const uint16_t *o = at(a.o, b, h) + t * a.o.t, *g = at(a.dout, b, h) + t * a.dout.t;
    const float lse = a.lse[stat];
    float s = 0.0f;
    if (const int d = part * 8; d < a.dim) {
        float x[8], y[8];
        load_n<DT, 8>(o, d, x);
        load_n<DT, 8>(g, d, y);
#pragma unroll
        for (int k = 0; k < 8; k++) s += x[k] * y[k];
    }
#pragma unroll
    for (int d = 8; d; d >>= 1) s += __shfl_xor(s, d, 64);
    // the row's keys in a list, the nearest first and the sinks last, until there are too many
    const int lo = max(0, pos - a.window + 1), near = pos - lo + 1, walk = near + min(a.sinks, lo);
    int *list = list_[threadIdx.x >> 4];
    bool few = lse != -__builtin_inff() && (a.key_mask || walk <= FEW_KEYS);
    int count = 0;
    for (int w = 0; __any(few && w < walk); w += 64) {
        bool seen[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int at = w + 16 * i + part, key = at < near ? pos - at : at - near;
            seen[i] = few && at < walk && (!a.key_mask || a.key_mask[b * a.mask_stride + key] != 0);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int at = w + 16 * i + part, key = at < near ? pos - at : at - near;
            const uint32_t m = (uint32_t)(__ballot(seen[i]) >> (lane & 48)) & 65535;
            const int place = count + __popc(m & ((1u << part) - 1));
            if (seen[i] && place < FEW_KEYS) list[place] = key;
            count += __popc(m);
        }
        few = few && count <= FEW_KEYS;
    }
    __builtin_amdgcn_wave_barrier();
    if (__any(few)) {
        // a key a lane
        const bool mine = few && part < count;
        const int64_t key = mine ? list[part] : pos;
        const uint16_t *q = at(a.q, b, h) + t * a.q.t, *k = at(a.k, b, hk) + key * a.k.t, *v = at(a.v, b, hk) + key * a.v.t;
        float sc = 0.0f, dp = 0.0f;
#pragma unroll 2
        for (int d = 0; d < a.dim; d += 8) {
            float x[8], y[8];
            load_n<DT, 8>(q, d, x);
            load_n<DT, 8>(k, d, y);
#pragma unroll
            for (int e = 0; e < 8; e++) sc += x[e] * y[e];
            load_n<DT, 8>(g, d, x);
            load_n<DT, 8>(v, d, y);
#pragma unroll
            for (int e = 0; e < 8; e++) dp += x[e] * y[e];
        }
        float p = mine ? exp2_hw(__builtin_fmaf(sc, a.scale * LOG2E, -lse * LOG2E)) : 0.0f;
        float de = mine ? p * dp : 0.0f;
#pragma unroll
        for (int d = 8; d; d >>= 1) {
            p += __shfl_xor(p, d, 64);
            de += __shfl_xor(de, d, 64);
        }
        if (few) s = p == 0.0f ? 0.0f : de / p;
        if (few && count == 1 && fabsf(lse) < __builtin_inff()) s = __builtin_bit_cast(float, LONE);
    }
    if (row < total && part == 0) a.delta[stat] = s;
}

// Scores that are hidden have no gradient, nor have those of LONE rows: bit 16 + r of `bits` is 0 (bit r: whether
// the score is visible; one word, for want of registers).  Such rows meet their key in tiles that are not all
// visible, the only ones to ask.
__device__ __forceinline__ void settle(f32x16 &ds, uint32_t bits)
{
#pragma unroll
    for (int r = 0; r < 16; r++) ds[r] = (bits >> (16 + r) & 1) ? ds[r] : 0.0f;
}

// dq of WAVES x 32 rows: the forward pass's walk over the keys, 32 keys at a time so that scores, their
// gradients and the sums fit the registers of two waves a SIMD.  Three products a score; the walk that is
// shared with dk and dv would save two of their seven and need atomic sums of dq, whose order changes
// results.  The forward's window of 2048: 397-409 us; 8 x 12 x 1024 of 64: 38 us.
template <int DT, int HD, int WAVES>
__global__ __launch_bounds__(WAVES * 64, HD == 64 ? 3 : 2) void attn_dq_kernel(AttnArgs a)
{
    constexpr int C = HD / 16, ND = HD / 32;
    constexpr int BYTES = TILE * Tile<HD>::ROW;
    __shared__ __attribute__((aligned(256))) char lds_[4 * BYTES];          // k, v; k, v of the next tile
    lds_char *const lds = (lds_char *)lds_;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = blockIdx.x / a.key_heads, hk = blockIdx.x % a.key_heads;
    const int total = a.rows * a.group, r0 = (gridDim.y - 1 - blockIdx.y) * WAVES * 32, row = r0 + wave * 32 + (lane & 31);
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
    float delta = a.delta[stat];
    const int wa = min(r0 + wave * 32, total - 1), wb = min(r0 + wave * 32 + 31, total - 1);
    const int pa = __builtin_amdgcn_readfirstlane(before + wa / a.group), pb = __builtin_amdgcn_readfirstlane(before + wb / a.group);
    const KeyTiles tiles(a, before + r0 / a.group, before + min(r0 + WAVES * 32 - 1, total - 1) / a.group);

    landed(q);
    landed(g);
    asm volatile("" : "+v"(lse), "+v"(delta));
    f32x16 dq[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) dq[d] = zero16();
    const float c2 = a.scale * LOG2E;
    Lift<DT> lift;
    KeyStage<HD, WAVES * 64> next;
    int rp = Tile<HD>::row_place(lane), cp = Tile<HD>::column_place(lane);
    uint64_t see = 0;
    int turn = 0;                                  // the tile being read
    next.load(a, b, hk, tiles.key(0));
    see = next.store(a, lds, lds + BYTES);
    if (tiles.count > 1) next.load(a, b, hk, tiles.key(1));
    __syncthreads();
    for (int it = 0; it < tiles.count; it++) {
        const int key = tiles.key(it);
        const lds_char *kt = lds + turn, *vt = kt + BYTES;
        asm volatile("" : "+v"(rp), "+v"(cp));     // the reads' addresses are formed where they are used, not kept
        if (see != 0 && !sight.none(pa, pb, key, key + TILE - 1)) {
            const bool whole = see == ~0ull && sight.all(pa, pb, key, key + TILE - 1);
            for (int n = 0; n < 2; n++) {
                uint32_t bits = 0;                           // which of the lane's 16 results are visible; have a gradient
                if (!whole) {
                    bits = visible16(sight, pos, key + 32 * n, (uint32_t)(see >> (32 * n)), lane);
                    bits |= is_lone(delta) ? 0 : bits << 16;
                }
                __builtin_amdgcn_sched_barrier(0);
                f32x16 s = zero16(), dp = zero16();
#pragma unroll
                for (int c = 0; c < C; c++) {
                    s = mma<DT>(Tile<HD>::rows(kt + n * (32 * Tile<HD>::ROW), rp, 0, c), q[c], s);
                    dp = mma<DT>(Tile<HD>::rows(vt + n * (32 * Tile<HD>::ROW), rp, 0, c), g[c], dp);
                }
                if (!whole) hide(s, bits);
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    s[r] = exp2_hw(__builtin_fmaf(s[r], c2, -lse));
                    dp[r] = s[r] * (dp[r] - delta);
                }
                if (!whole) settle(dp, bits);
                lift.fit(dp, dq);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const u32x4 p = operand<DT>(dp, 8 * k);
#pragma unroll
                    for (int d = 0; d < ND; d++) dq[d] = mma<DT>(Tile<HD>::columns(kt + n * (32 * Tile<HD>::ROW), cp, 16 * k, d), p, dq[d]);
                    if (!whole) {
                        const u32x4 rest = remainder<DT>(dp, 8 * k, p);
#pragma unroll
                        for (int d = 0; d < ND; d++) dq[d] = mma<DT>(Tile<HD>::columns(kt + n * (32 * Tile<HD>::ROW), cp, 16 * k, d), rest, dq[d]);
                    }
                }
            }
        }
        turn ^= 2 * BYTES;
        if (it + 1 < tiles.count) {
            see = next.store(a, lds + turn, lds + turn + BYTES);
            if (it + 2 < tiles.count) next.load(a, b, hk, tiles.key(it + 2));
        }
        __syncthreads();
    }
    if (!real) return;
    const float scale = a.scale * lift.down();
    uint16_t *po = (uint16_t *)at(a.dq, b, head) + t * a.dq.t;
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int e = 32 * d + result_row(r, lane);
            if (e < a.dim)
                *(u32x2 *)(po + e) = u32x2{pack2<DT>(dq[d][r] * scale, dq[d][r + 1] * scale),
                                           pack2<DT>(dq[d][r + 2] * scale, dq[d][r + 3] * scale)};
        }
}

// dk and dv of WAVES x 32 keys: over the rows that see any of them, 32 at a time.  A workgroup takes the
// positions whose window holds a key of its block; those behind that, which see the sinks alone, go to
// workgroups of their own, and where there are few blocks each one's walk is cut into shares (DkvSplit);
// the sums are fp32 partial results then.  Four products a score.  Heads of 128 hold k in registers and v
// in LDS (both in registers spilled; separate kernels for dk and dv formed the scores twice and were slower
// together).  The forward's window of 2048: 586-600 us, with the sinks' far positions in their block's own walk
// 900; 8 x 12 x 1024 of 64: 61 us; ragged fp16 sequences of few blocks 50 us (46 without the powers of two) and 7 to
// add their parts, in one walk each 109.
template <int DT, int HD, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void attn_dkv_kernel(AttnArgs a, DkvSplit cut)
{
    constexpr int C = HD / 16, ND = HD / 32;
    // the keys' v in registers where there is room, otherwise in LDS
    constexpr bool VREGS = HD == 64;
    using S = Stage<HD, WAVES * 64, 32>;
    constexpr int BYTES = 32 * Tile<HD>::ROW;
    __shared__ __attribute__((aligned(256))) char lds_[4 * BYTES + (VREGS ? 0 : WAVES * BYTES)];   // q, dout; q, dout of the next tile; v
    __shared__ __attribute__((aligned(16))) float lse_s[2][32], delta_s[2][32];
    __shared__ __attribute__((aligned(16))) int pos_s[2][32];
    lds_char *const lds = (lds_char *)lds_;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = blockIdx.x / a.key_heads, hk = blockIdx.x % a.key_heads;
    // blockIdx.y: the blocks of keys, then their other parts: of the walk, or the sinks' far positions
    const int y = blockIdx.y, more = y - cut.blocks;
    const int share = cut.shares > 1 ? y / cut.blocks : 0;
    const int far = cut.shares > 1 || more < 0 ? -1 : more % cut.far;
    const int block = far >= 0 ? more / cut.far : y - share * cut.blocks;
    const int k0 = block * WAVES * 32, ka = k0 + wave * 32, key = ka + (lane & 31);
    const Sight sight = {a.window, a.sinks};
    const int before = a.keys - a.rows;
    const bool real = key < a.keys;
    const bool seen = real && (!a.key_mask || a.key_mask[b * a.mask_stride + key] != 0);
    const bool all_seen = __ballot(seen) == ~0ull;

    lds_char *const vtile = lds + (4 + wave) * BYTES;
    int rp = Tile<HD>::row_place(lane), cp = Tile<HD>::column_place(lane);
    u32x4 kf[C], vf[VREGS ? C : 1];
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int d = 16 * c + 8 * (lane >> 5);
        u32x4 v = {0, 0, 0, 0};
        kf[c] = v;
        if (d < a.dim && seen) {
            kf[c] = *(const u32x4 *)(at(a.k, b, hk) + (int64_t)key * a.k.t + d);
            v = *(const u32x4 *)(at(a.v, b, hk) + (int64_t)key * a.v.t + d);
        }
        if constexpr (VREGS) vf[c] = v;
        else *(__attribute__((address_space(3))) u32x4 *)(vtile + Tile<HD>::at(lane & 31, 2 * c + (lane >> 5))) = v;      // read by this wave alone
    }
    auto values = [&](int c) {
        if constexpr (VREGS) return vf[c];
        else return Tile<HD>::rows(vtile, rp, 0, c);
    };
    landed(kf);
    if constexpr (VREGS) landed(vf);
    f32x16 dk[ND], dv[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) dk[d] = dv[d] = zero16();
    const float c2 = a.scale * LOG2E;
    Lift<DT> lift;
    // the positions that see a key of this workgroup: [p0, p1)
    const int k1 = min(a.keys, k0 + WAVES * 32) - 1;
    const int near = min(a.keys, k1 + a.window);
    int p0 = max(k0, before), p1 = near;
    if (far >= 0) {
        p0 = max(near + far * cut.step, before);
        p1 = min(a.keys, near + (far + 1) * cut.step);
    } else if (k0 < a.sinks && cut.far == 0) p1 = a.keys;
    if (cut.shares > 1) {
        const int each = (max(0, p1 - p0) + cut.shares - 1) / cut.shares;
        p0 += share * each;
        p1 = min(p1, p0 + each);
    }
    const int first = (p0 - before) * a.group, last = (p1 - before) * a.group;      // rows
    S qs, gs;
    float lse_r = 0.0f, delta_r = 0.0f;
    int pos_r = 0;
    const float per_group = 1.0f / (float)a.group;
    const uint16_t *const qp = at(a.q, b, hk * a.group), *const gp = at(a.dout, b, hk * a.group);
    // the next tile to bring: its first row is head `over` of position t0 (a tile on is `whole_t` positions
    // and `rest` heads on)
    int t0 = p0 - before, over = 0, row_in = first;
    const int whole_t = 32 / a.group, rest = 32 - whole_t * a.group;
    // where the thread's pieces of a tile and its row's statistics lie, from position t0 on: the same for
    // every tile where the heads that share a key head divide 32
    uint32_t qo[S::N], go[S::N];
    int stat_r = 0, stat_t = 0;
    auto place = [&]() {
#pragma unroll
        for (int i = 0; i < S::N; i++) {
            // small numbers, divided in fp32
            const int r = over + S::row() + i * S::STEP, t = (int)(((float)r + 0.5f) * per_group), g = r - t * a.group;
            const bool there = S::piece() * 8 < a.dim;
            qo[i] = there ? (t * (uint32_t)a.q.t + g * (uint32_t)a.q.h + S::piece() * 8) * 2 : NOWHERE;
            go[i] = there ? (t * (uint32_t)a.dout.t + g * (uint32_t)a.dout.h + S::piece() * 8) * 2 : NOWHERE;
        }
        const int r = over + (threadIdx.x & 31);
        stat_t = (int)(((float)r + 0.5f) * per_group);
        stat_r = (r - stat_t * a.group) * a.rows + stat_t;
    };
    place();
    const int64_t stat0 = ((int64_t)b * a.heads + hk * a.group) * a.rows;
    auto fetch = [&]() {
        const auto qr = buffer_from(qp + t0 * a.q.t), gr = buffer_from(gp + t0 * a.dout.t);
        if (row_in + 32 <= last) {
            qs.load(qr, [&](int i) { return qo[i]; });
            gs.load(gr, [&](int i) { return go[i]; });
        } else {
            auto there = [&](int i) { return row_in + S::row() + i * S::STEP < last; };
            qs.load(qr, [&](int i) { return there(i) ? qo[i] : NOWHERE; });
            gs.load(gr, [&](int i) { return there(i) ? go[i] : NOWHERE; });
        }
        if (threadIdx.x < 32) {                          // (looked at when the tile is stored)
            pos_r = -1;                                  // behind the last row there is no weight
            if (row_in + (int)threadIdx.x < last) {
                lse_r = a.lse[stat0 + t0 + stat_r];
                delta_r = a.delta[stat0 + t0 + stat_r];
                pos_r = before + t0 + stat_t;
            }
        }
        row_in += 32;
        t0 += whole_t;
        if (rest) {
            over += rest;
            if (over >= a.group) {
                over -= a.group;
                t0++;
            }
            place();
        }
    };
    auto store = [&](int side) {
        qs.store(lds + side * 2 * BYTES);
        gs.store(lds + side * 2 * BYTES + BYTES);
        if (threadIdx.x < 32) {
            const bool none = pos_r < 0 || lse_r == -__builtin_inff();   // nor where a row sees nothing
            lse_s[side][threadIdx.x] = none ? __builtin_inff() : __builtin_fmaf(lse_r, LOG2E, -RAISE<DT>);
            delta_s[side][threadIdx.x] = none ? 0.0f : delta_r;
            pos_s[side][threadIdx.x] = pos_r;
        }
    };
    int side = 0;
    // the positions of the tile being read: pa, and no more than pb
    int pa = p0, pb = p0;
    if (first < last) {
        fetch();
        pb = before + t0;
        store(0);
        if (row_in < last) fetch();
    }
    __syncthreads();
    for (int row0 = first; row0 < last; row0 += 32) {
        const lds_char *qt = lds + side * 2 * BYTES, *gt = qt + BYTES;
        asm volatile("" : "+v"(rp), "+v"(cp));     // the reads' addresses are formed where they are used, not kept
        if (!sight.none(pa, pb, ka, ka + 31)) {
            const bool whole = all_seen && sight.all(pa, pb, ka, ka + 31);
            uint32_t bits = 0;                               // which of the lane's 16 results are visible; have a gradient
            if (!whole) {
                for (int r = 0; r < 16; r += 4) {
                    const u32x4 po = *(const u32x4 *)(pos_s[side] + result_row(r, lane));
                    const f32x4 de = *(const f32x4 *)(delta_s[side] + result_row(r, lane));
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const bool one = seen && sight.one((int)po[k], key);
                        bits |= ((uint32_t)one | (uint32_t)(one && !is_lone(de[k])) << 16) << (r + k);
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            f32x16 s = zero16(), dp = zero16();
#pragma unroll
            for (int c = 0; c < C; c++) {
                s = mma<DT>(Tile<HD>::rows(qt, rp, 0, c), kf[c], s);
                dp = mma<DT>(Tile<HD>::rows(gt, rp, 0, c), values(c), dp);
            }
            if (!whole) hide(s, bits);
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const f32x4 ls = *(const f32x4 *)(lse_s[side] + result_row(r, lane)), de = *(const f32x4 *)(delta_s[side] + result_row(r, lane));
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    s[r + k] = exp2_hw(__builtin_fmaf(s[r + k], c2, -ls[k]));
                    dp[r + k] = s[r + k] * (dp[r + k] - de[k]);
                }
            }
            if (!whole) settle(dp, bits);
            lift.fit(dp, dk);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const u32x4 p = operand<DT>(s, 8 * k), ds = operand<DT>(dp, 8 * k);
#pragma unroll
                for (int d = 0; d < ND; d++) {
                    dv[d] = mma<DT>(Tile<HD>::columns(gt, cp, 16 * k, d), p, dv[d]);
                    dk[d] = mma<DT>(Tile<HD>::columns(qt, cp, 16 * k, d), ds, dk[d]);
                }
                if (!whole) {
                    const u32x4 rest = remainder<DT>(dp, 8 * k, ds);
#pragma unroll
                    for (int d = 0; d < ND; d++) dk[d] = mma<DT>(Tile<HD>::columns(qt, cp, 16 * k, d), rest, dk[d]);
                }
            }
        }
        side ^= 1;
        pa = pb;
        if (row0 + 32 < last) {
            pb = before + t0;
            store(side);
            if (row_in < last) fetch();
        }
        __syncthreads();
    }
    if (!real) return;
    if constexpr (Lift<DT>::ON) {
        const float back = __builtin_ldexpf(1.0f, -(int)RAISE<DT>), down = lift.down() * back;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                dk[d][r] *= down;
                dv[d][r] *= back;
            }
    }
    const int part_keys = cut.keys(a);
    if (key < part_keys) {
        float *part = cut.sums(a, blockIdx.x, share + far + 1) + (int64_t)key * a.dim;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int e = 32 * d + result_row(r, lane);
                if (e >= a.dim) continue;
                *(f32x4 *)(part + e) = f32x4{dk[d][r], dk[d][r + 1], dk[d][r + 2], dk[d][r + 3]};
                *(f32x4 *)(part + (int64_t)part_keys * a.dim + e) = f32x4{dv[d][r], dv[d][r + 1], dv[d][r + 2], dv[d][r + 3]};
            }
        return;
    }
    if (far >= 0) return;
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

// Adds the parts of dk and dv: a thread 2 elements of one key.
template <int DT>
__global__ __launch_bounds__(256) void attn_parts_kernel(AttnArgs a, DkvSplit cut)
{
    const int b = blockIdx.x / a.key_heads, hk = blockIdx.x % a.key_heads, keys = cut.keys(a), parts = cut.parts();
    const int i = blockIdx.y * 256 + threadIdx.x, key = i / (a.dim / 2), e = i % (a.dim / 2) * 2;
    if (key >= keys) return;
    const float *part = cut.sums(a, blockIdx.x, 0) + (int64_t)key * a.dim + e;
    const int64_t other = (int64_t)keys * a.dim;
    f32x2 k = {0.0f, 0.0f}, v = {0.0f, 0.0f};
#pragma unroll 4
    for (int f = 0; f < parts; f++, part += 2 * other) {
        k += *(const f32x2 *)part;
        v += *(const f32x2 *)(part + other);
    }
    *(uint32_t *)((uint16_t *)at(a.dk, b, hk) + (int64_t)key * a.dk.t + e) = pack2<DT>(k[0] * a.scale, k[1] * a.scale);
    *(uint32_t *)((uint16_t *)at(a.dv, b, hk) + (int64_t)key * a.dv.t + e) = pack2<DT>(v[0], v[1]);
}

// (A launch's error is read before the next one: that one's success would take its place.)
template <int DT, int HD>
hipError_t run_forward(const AttnArgs &a, hipStream_t stream)
{
    const int total = a.rows * a.group, heads = a.batch * a.key_heads;
    if (total <= 32)
        attn_fwd_kernel<DT, HD, 1><<<dim3(heads, 1, a.splits), 64, 0, stream>>>(a);
    else
        attn_fwd_kernel<DT, HD, 4><<<dim3(heads, (total + 127) / 128, a.splits), 256, 0, stream>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.splits == 1) return e;
    if (a.splits > FEW) attn_join_kernel<DT><<<dim3(heads, total), 256, 0, stream>>>(a);
    else attn_join_few_kernel<DT><<<dim3(heads, (total + 3) / 4), 256, 0, stream>>>(a);
    return hipGetLastError();
}

template <int DT, int HD>
hipError_t run_backward(const AttnArgs &a, hipStream_t stream)
{
    const int total = a.rows * a.group, heads = a.batch * a.key_heads;
    const int64_t rows = (int64_t)a.batch * a.heads * a.rows;
    const DkvSplit cut = dkv_split(a);
    hipError_t e = hipSuccess;
    if (rows) {
        const int tiles = (total + 15) / 16;
        attn_delta_kernel<DT><<<dim3(heads, tiles < DELTA_Y ? tiles : DELTA_Y, (tiles + DELTA_Y - 1) / DELTA_Y), 256, 0, stream>>>(a);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    attn_dkv_kernel<DT, HD, 4><<<dim3(heads, cut.blocks * cut.shares + cut.sink_blocks * cut.far), 256, 0, stream>>>(a, cut);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    if (cut.parts() > 1) {
        attn_parts_kernel<DT><<<dim3(heads, (unsigned)(((int64_t)cut.keys(a) * a.dim / 2 + 255) / 256)), 256, 0, stream>>>(a, cut);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    if (rows) attn_dq_kernel<DT, HD, 4><<<dim3(heads, (total + 127) / 128), 256, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace

template <int DT>
hipError_t attn_forward(const AttnArgs &a, hipStream_t stream)
{
    return a.dim <= 64 ? run_forward<DT, 64>(a, stream) : run_forward<DT, 128>(a, stream);
}

template <int DT>
hipError_t attn_backward(const AttnArgs &a, hipStream_t stream)
{
    return a.dim <= 64 ? run_backward<DT, 64>(a, stream) : run_backward<DT, 128>(a, stream);
}

}  // namespace lm
