// lm_embed.hip -- embedding lookup with scaling, and its dense gradient by sorted tokens.
//
//   out[i, :] = s * W[tok_i, :]            dW[v, :] = s * sum_{i : tok_i = v} g[i, :]
//
// Both are bound by memory: the lookup reads and writes each row once; the gradient reads g once
// and writes the whole table, which for a vocabulary far larger than the batch is most of it.
//
// The gradient adds each token's rows in the order of their positions, in fp32, whatever the
// grid: no float atomics, so a call gives the same bits every time.  Three launches:
//   1. sort: workgroup b owns a range of the vocabulary, reads all tokens (L2 serves the repeats),
//      keeps those of its range in order and counts those below it, which is where its entries
//      start in the sorted list: a stable counting sort without any exchange between workgroups.
//      It also knows the rows that no token names, and writes their zeros.
//   2. sums: a wave takes SEG sorted entries and one slice of columns, and adds runs of equal
//      tokens in registers.  A run inside its entries is final; the parts of a run that crosses
//      the border go to fp32 partial rows.
//   3. join: the wave that holds a crossing run's first entry adds its parts in order.
// The gradient of 8192 tokens over 50257 x 768: 23-30 us for the sort and 131 MB of zeros, 12 and 4 us for
// the rest; of 16384 tokens that favour few over 32000 x 4096 bf16: 34, 61 and 8 us.
#include "lm_common.h"
#include "lm_embed.h"

namespace lm {
namespace {

constexpr int SEG = 16;            // sorted entries per wave of the sums
constexpr int SORT_THREADS = 1024, SORT_WAVES = SORT_THREADS / 64;
constexpr int MAX_RANGE = 512;     // rows of the vocabulary that one workgroup sorts (its LDS counters)
constexpr int LOOKUP_X = 1 << 22;  // workgroups of the lookup along a grid's first dimension, which ends at 2^32 threads
constexpr int LIST = 256;          // entries a wave of the sort keeps in LDS before it reads them again

__device__ __forceinline__ int64_t token_at(const void *tokens, int bytes, int64_t i)
{
    return bytes == 8 ? ((const int64_t *)tokens)[i] : (int64_t)((const int32_t *)tokens)[i];
}

// ---------------------------------------------------------------- lookup
// A workgroup takes whole rows, about 1024 pieces of VEC elements (blockIdx.y cuts longer rows): four
// independent 16-byte loads a thread in flight.  8192 rows of 768 fp32: 11 us; 16384 rows of 4096 bf16
// whose tokens favour few: 48 us, 5.6 TB/s of rows read and written (repeated rows come from cache).
template <int WDT, int ODT, int VEC>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const void *tokens, int token_bytes, int64_t n, int64_t vocab, int dim,
                                                        float scale, const void *weight, int64_t weight_stride, void *out,
                                                        int rows_per_wg, int pieces)
{
    const int64_t row0 = ((int64_t)blockIdx.z * LOOKUP_X + blockIdx.x) * rows_per_wg;
    if (row0 >= n) return;
    const int rows = (int)min((int64_t)rows_per_wg, n - row0);
    const int total = rows * pieces;
    for (int c0 = blockIdx.y * 1024 + threadIdx.x; c0 < total; c0 += gridDim.y * 1024) {
        float v[4][VEC];
        int64_t at[4];
        bool bad[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int c = c0 + u * 256;
            at[u] = -1;
            bad[u] = false;
            if (c < total) {
                const int r = c / pieces, p = c - r * pieces;
                const int64_t tok = token_at(tokens, token_bytes, row0 + r);
                at[u] = (row0 + r) * dim + p * VEC;
                bad[u] = tok < 0 || tok >= vocab;
                if (!bad[u]) load_n<WDT, VEC>(weight, tok * weight_stride + p * VEC, v[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (at[u] >= 0) {
                // a token outside the table has no row: NaN says so, and nothing outside is read
#pragma unroll
                for (int k = 0; k < VEC; k++) v[u][k] = bad[u] ? __builtin_nanf("") : v[u][k] * scale;
                store_n<ODT, VEC>(out, at[u], v[u]);
            }
    }
}

// ---------------------------------------------------------------- sort
struct SortLds {
    int hist[SORT_WAVES][MAX_RANGE];              // counts, then each wave's next place
    uint32_t list[SORT_WAVES][LIST];              // the first entries of each wave: token less the range's first,
    uint32_t pos[SORT_WAVES][LIST];               // and position
    int wave_sum[SORT_WAVES];
    int below[SORT_WAVES];
};

// Lanes of the wave holding the same key (valid lanes only), by one ballot per bit.
__device__ __forceinline__ uint64_t same_key(uint32_t key, bool valid, int bits)
{
    uint64_t m = __ballot(valid);
    for (int b = 0; b < bits; b++) {
        const uint64_t set = __ballot((key >> b) & 1);
        m &= (key >> b) & 1 ? set : ~set;
    }
    return m;
}

template <int DWDT, int VEC>
__global__ __launch_bounds__(SORT_THREADS) void embed_sort_kernel(const void *tokens, int token_bytes, int n, int vocab, int range,
                                                                  int range_bits, int64_t padding, int *sorted_tok, int *sorted_pos,
                                                                  int *count, void *dweight, int64_t dweight_stride, int dim, bool zero)
{
    __shared__ SortLds s;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int lo = blockIdx.x * range, hi = min(vocab, lo + range), width = hi - lo;
    const uint64_t lower = (1ull << lane) - 1;
    for (int i = threadIdx.x; i < SORT_WAVES * MAX_RANGE; i += SORT_THREADS) (&s.hist[0][0])[i] = 0;
    // each wave reads one stretch of the positions, 64 at a time
    const int stretch = (int)((((int64_t)n + SORT_WAVES - 1) / SORT_WAVES + 63) / 64 * 64);
    const int first = (int)min((int64_t)n, (int64_t)wave * stretch), last = (int)min((int64_t)n, (int64_t)first + stretch);
    int kept = 0, below = 0;
    __syncthreads();
    for (int i0 = first; i0 < last; i0 += 256) {
        int64_t tok[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int i = i0 + u * 64 + lane;
            tok[u] = i < last ? token_at(tokens, token_bytes, i) : -1;
            if (tok[u] == padding) tok[u] = -1;
        }
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const bool mine = tok[u] >= lo && tok[u] < hi;
            const uint64_t m = __ballot(mine);
            below += __popcll(__ballot(tok[u] >= 0 && tok[u] < lo));
            if (m) {
                const int at = kept + __popcll(m & lower);
                if (mine) {
                    const int key = (int)(tok[u] - lo);
                    atomicAdd(&s.hist[wave][key], 1);
                    if (at < LIST) {
                        s.list[wave][at] = key;
                        s.pos[wave][at] = i0 + u * 64 + lane;
                    }
                }
                kept += __popcll(m);
            }
        }
    }
    if (lane == 0) s.below[wave] = below;
    __syncthreads();
    // exclusive places: over the tokens of the range, and for each token over the waves
    int base = 0;
    for (int w = 0; w < SORT_WAVES; w++) base += s.below[w];
    int mine = 0;
    const int t = threadIdx.x;
    if (t < width)
        for (int w = 0; w < SORT_WAVES; w++) {
            const int h = s.hist[w][t];
            s.hist[w][t] = mine;
            mine += h;
        }
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(incl, d, 64);
        if (lane >= d) incl += o;
    }
    if (lane == 63) s.wave_sum[wave] = incl;
    __syncthreads();
    int total = 0, before = 0;
    for (int w = 0; w < SORT_WAVES; w++) {
        if (w < wave) before += s.wave_sum[w];
        total += s.wave_sum[w];
    }
    if (t < width) {
        const int start = base + before + incl - mine;
        for (int w = 0; w < SORT_WAVES; w++) s.hist[w][t] += start;
    }
    if (blockIdx.x == gridDim.x - 1 && t == 0) *count = base + total;
    __syncthreads();
    // place the entries, each wave its own in order
    auto place = [&](bool valid, uint32_t key, int pos) {
        const uint64_t same = same_key(key, valid, range_bits);
        if (valid) {
            const int at = s.hist[wave][key] + __popcll(same & lower);
            sorted_tok[at] = lo + (int)key;
            sorted_pos[at] = pos;
        }
        __builtin_amdgcn_wave_barrier();
        if (valid && !(same & lower)) s.hist[wave][key] += __popcll(same);
        __builtin_amdgcn_wave_barrier();
    };
    if (kept <= LIST) {
        for (int i = 0; i < kept; i += 64) {
            const bool valid = i + lane < kept;
            place(valid, valid ? s.list[wave][i + lane] : 0, valid ? (int)s.pos[wave][i + lane] : 0);
        }
    } else {
        for (int i = first; i < last; i += 64) {
            const int64_t tok = i + lane < last ? token_at(tokens, token_bytes, i + lane) : -1;
            const bool valid = tok >= lo && tok < hi && tok != padding;
            if (__ballot(valid)) place(valid, valid ? (uint32_t)(tok - lo) : 0, i + lane);
        }
    }
    if (!zero) return;
    // rows that no token names: after the placing, a row is empty if the last wave's place is its start
    __syncthreads();
    if (t < width) s.hist[0][t] = mine;
    __syncthreads();
    const int pieces = dim / VEC;
    float nil[VEC] = {};
    for (int r = wave; r < width; r += SORT_WAVES)
        if (s.hist[0][r] == 0)
            for (int p = lane; p < pieces; p += 64) store_n<DWDT, VEC>(dweight, (int64_t)(lo + r) * dweight_stride + p * VEC, nil);
}

// ---------------------------------------------------------------- sums
template <int DWDT, int VEC>
__device__ __forceinline__ void finish_row(void *dweight, int64_t at, float *acc, float scale, bool accumulate)
{
#pragma unroll
    for (int k = 0; k < VEC; k++) acc[k] *= scale;
    if (accumulate) {
        float had[VEC];
        load_n<DWDT, VEC>(dweight, at, had);
#pragma unroll
        for (int k = 0; k < VEC; k++) acc[k] += had[k];
    }
    store_n<DWDT, VEC>(dweight, at, acc);
}

// Wave w of the grid: entries [SEG w, SEG w + SEG), columns [64 VEC blockIdx.x, ...).  `partial`
// [2 chunks][dim]: a chunk's run that began before it, and the run that goes on behind it.  (A run
// that does both is the first kind.)
template <int GDT, int DWDT, int VEC>
__global__ __launch_bounds__(256) void embed_sum_kernel(const int *sorted_tok, const int *sorted_pos, const int *count, const void *grad,
                                                        int64_t grad_stride, int dim, float scale, void *dweight,
                                                        int64_t dweight_stride, bool accumulate, float *partial)
{
    const int lane = threadIdx.x & 63;
    const int chunk = (blockIdx.y + blockIdx.z * 32768) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m = *count;
    const int e0 = chunk * SEG, e1 = min(m, e0 + SEG);
    if (e0 >= m) return;
    const int col = (blockIdx.x * 64 + lane) * VEC;
    const bool live = col < dim;
    float acc[VEC] = {};
    // the chunk's entries, and the tokens on both sides of it (-1: none), one a lane
    const int at = e0 - 1 + lane;
    const int toks = lane <= SEG + 1 && at >= 0 && at < m ? sorted_tok[at] : -1;
    const int poss = lane < SEG && e0 + lane < m ? sorted_pos[e0 + lane] : 0;
    auto token = [&](int i) { return __builtin_amdgcn_readlane(toks, i + 1); };
    const int n = e1 - e0;
    const bool open_front = token(-1) == token(0), open_back = token(n) == token(n - 1);
    bool from_front = open_front;
    constexpr int FLY = 8;                         // rows on their way
    for (int e = 0; e < n; e += FLY) {
        float g[FLY][VEC];
#pragma unroll
        for (int u = 0; u < FLY; u++)
            if (e + u < n && live) load_n<GDT, VEC>(grad, (int64_t)__builtin_amdgcn_readlane(poss, e + u) * grad_stride + col, g[u]);
#pragma unroll
        for (int u = 0; u < FLY; u++) {
            if (e + u >= n) break;
            const int tok = token(e + u);
#pragma unroll
            for (int k = 0; k < VEC; k++) acc[k] += live ? g[u][k] : 0.0f;
            const bool at_end = e + u + 1 == n;
            if (at_end ? open_back : token(e + u + 1) == tok) continue;
            // the run of `tok` ends here
            if (live) {
                if (from_front) store_n<DT_F32, VEC>(partial, (int64_t)(2 * chunk) * dim + col, acc);
                else finish_row<DWDT, VEC>(dweight, (int64_t)tok * dweight_stride + col, acc, scale, accumulate);
            }
            from_front = false;
#pragma unroll
            for (int k = 0; k < VEC; k++) acc[k] = 0.0f;
        }
    }
    if (open_back && live) store_n<DT_F32, VEC>(partial, (int64_t)(2 * chunk + (from_front ? 0 : 1)) * dim + col, acc);
}

// One wave per chunk whose last run goes on behind it and began inside it.
template <int DWDT, int VEC>
__global__ __launch_bounds__(256) void embed_join_kernel(const int *sorted_tok, const int *count, int dim, float scale, void *dweight,
                                                         int64_t dweight_stride, bool accumulate, const float *partial)
{
    const int lane = threadIdx.x & 63;
    const int chunk = (blockIdx.y + blockIdx.z * 32768) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m = *count;
    const int e0 = chunk * SEG, e1 = e0 + SEG;
    if (e1 >= m) return;
    const int tok = sorted_tok[e1 - 1];
    if (sorted_tok[e1] != tok || (sorted_tok[e0] == tok && e0 > 0 && sorted_tok[e0 - 1] == tok)) return;
    const int col = (blockIdx.x * 64 + lane) * VEC;
    const bool live = col < dim;                   // (every lane looks the parts up)
    float acc[VEC] = {};
    if (live) load_n<DT_F32, VEC>(partial, (int64_t)(2 * chunk + 1) * dim + col, acc);
    // the run's parts: the front of each later chunk that starts with this token, 64 looked up at a time
    for (int c0 = chunk + 1;; c0 += 64) {
        const int64_t first = (int64_t)(c0 + lane) * SEG;
        const uint64_t not_mine = ~__ballot(first < m && sorted_tok[first < m ? first : 0] == tok);
        const int parts = not_mine ? __builtin_ctzll(not_mine) : 64;
        for (int i = 0; i < parts; i += 8) {
            float v[8][VEC];
#pragma unroll
            for (int u = 0; u < 8; u++)
                if (i + u < parts && live) load_n<DT_F32, VEC>(partial, (int64_t)(2 * (c0 + i + u)) * dim + col, v[u]);
#pragma unroll
            for (int u = 0; u < 8; u++)
                if (i + u < parts)
#pragma unroll
                    for (int k = 0; k < VEC; k++) acc[k] += live ? v[u][k] : 0.0f;
        }
        if (parts < 64) break;
    }
    if (!live) return;
    finish_row<DWDT, VEC>(dweight, (int64_t)tok * dweight_stride + col, acc, scale, accumulate);
}

bool aligned(const void *p, int64_t stride, int64_t dim, int vec, int size)
{
    const int64_t bytes = vec * size < 16 ? vec * size : 16;
    return (uintptr_t)p % bytes == 0 && (stride * size) % bytes == 0 && dim % vec == 0;
}

int size_of(int dt) { return dt == DT_F32 ? 4 : 2; }

int ranges(int64_t vocab)
{
    // at least one workgroup per CU, and no range wider than the counters
    const int64_t wide = (vocab + 255) / 256;
    return (int)(wide < 1 ? 1 : wide > MAX_RANGE ? MAX_RANGE : wide);
}

int64_t chunks(int64_t n) { return (n + SEG - 1) / SEG; }
int64_t round_up(int64_t x) { return (x + 255) / 256 * 256; }

template <int WDT, int ODT>
void launch_fwd(const EmbedArgs &a, const void *weight, int64_t weight_stride, void *out, hipStream_t stream)
{
    const bool wide = aligned(weight, weight_stride, a.dim, 8, size_of(WDT)) && aligned(out, a.dim, a.dim, 8, size_of(ODT));
    const int pieces = (int)(wide ? a.dim / 8 : a.dim);
    const int rows = pieces >= 1024 ? 1 : 1024 / pieces;
    const int64_t wgs = (a.n + rows - 1) / rows;
    const dim3 grid((unsigned)(wgs < LOOKUP_X ? wgs : LOOKUP_X), (unsigned)((rows * pieces + 1023) / 1024),
                    (unsigned)((wgs + LOOKUP_X - 1) / LOOKUP_X));
    if (wide)
        embed_fwd_kernel<WDT, ODT, 8><<<grid, 256, 0, stream>>>(a.tokens, a.token_bytes, a.n, a.vocab, (int)a.dim, a.scale, weight,
                                                                weight_stride, out, rows, pieces);
    else
        embed_fwd_kernel<WDT, ODT, 1><<<grid, 256, 0, stream>>>(a.tokens, a.token_bytes, a.n, a.vocab, (int)a.dim, a.scale, weight,
                                                                weight_stride, out, rows, pieces);
}

template <int GDT, int DWDT, int VEC>
hipError_t launch_bwd(const EmbedArgs &a, const void *grad, int64_t grad_stride, void *dweight, int64_t dweight_stride, int64_t padding,
                bool accumulate, void *workspace, hipStream_t stream)
{
    int *tok = (int *)workspace;
    int *pos = (int *)((char *)workspace + round_up(a.n * 4));
    int *count = (int *)((char *)pos + round_up(a.n * 4));
    float *partial = (float *)((char *)count + 256);
    const int range = ranges(a.vocab);
    int bits = 0;
    while ((1 << bits) < range) bits++;
    embed_sort_kernel<DWDT, VEC><<<(unsigned)((a.vocab + range - 1) / range), SORT_THREADS, 0, stream>>>(
        a.tokens, a.token_bytes, (int)a.n, (int)a.vocab, range, bits, padding, tok, pos, count, dweight, dweight_stride, (int)a.dim,
        !accumulate);
    // (an error is read before the next launch, whose success would take its place)
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.n == 0) return e;
    const int64_t pieces = a.dim / VEC;
    // (the slices of a chunk's columns side by side: their rows' lines are neighbours in memory)
    const int64_t wgs = (chunks(a.n) + 3) / 4;
    const dim3 grid((unsigned)((pieces + 63) / 64), (unsigned)(wgs < 32768 ? wgs : 32768), (unsigned)((wgs + 32767) / 32768));
    embed_sum_kernel<GDT, DWDT, VEC><<<grid, 256, 0, stream>>>(tok, pos, count, grad, grad_stride, (int)a.dim, a.scale, dweight,
                                                               dweight_stride, accumulate, partial);
    e = hipGetLastError();
    if (e != hipSuccess || a.n <= SEG) return e;
    embed_join_kernel<DWDT, VEC><<<grid, 256, 0, stream>>>(tok, count, (int)a.dim, a.scale, dweight, dweight_stride, accumulate, partial);
    return hipGetLastError();
}

template <int GDT, int DWDT>
hipError_t pick_bwd(const EmbedArgs &a, const void *grad, int64_t gs, void *dw, int64_t dws, int64_t padding, bool acc, void *ws,
              hipStream_t stream)
{
    // 4 columns a lane where a row of fp32 is involved (16 bytes of it), 8 where all are 16-bit
    constexpr int WIDE = GDT == DT_F32 || DWDT == DT_F32 ? 4 : 8;
    if (aligned(grad, gs, a.dim, WIDE, size_of(GDT)) && aligned(dw, dws, a.dim, WIDE, size_of(DWDT)))
        return launch_bwd<GDT, DWDT, WIDE>(a, grad, gs, dw, dws, padding, acc, ws, stream);
    return launch_bwd<GDT, DWDT, 1>(a, grad, gs, dw, dws, padding, acc, ws, stream);
}

}  // namespace

#define LM_TYPE_PAIR(a, b, CALL)                         \
    switch ((a) * 3 + (b)) {                             \
    case 0: CALL(DT_F32, DT_F32); break;                 \
    case 1: CALL(DT_F32, DT_BF16); break;                \
    case 2: CALL(DT_F32, DT_F16); break;                 \
    case 3: CALL(DT_BF16, DT_F32); break;                \
    case 4: CALL(DT_BF16, DT_BF16); break;               \
    case 5: CALL(DT_BF16, DT_F16); break;                \
    case 6: CALL(DT_F16, DT_F32); break;                 \
    case 7: CALL(DT_F16, DT_BF16); break;                \
    default: CALL(DT_F16, DT_F16); break;                \
    }

hipError_t embed_forward(const EmbedArgs &a, const void *weight, int weight_dt, int64_t weight_stride, void *out, int out_dt,
                         hipStream_t stream)
{
#define CALL(W, O) launch_fwd<W, O>(a, weight, weight_stride, out, stream)
    LM_TYPE_PAIR(weight_dt, out_dt, CALL)
#undef CALL
    return hipGetLastError();
}

int64_t embed_backward_workspace(int64_t n, int64_t vocab, int64_t dim)
{
    (void)vocab;
    return 2 * round_up(n * 4) + 256 + 2 * chunks(n) * dim * 4;
}

hipError_t embed_backward(const EmbedArgs &a, const void *grad, int grad_dt, int64_t grad_stride, void *dweight, int dweight_dt,
                          int64_t dweight_stride, int64_t padding, bool accumulate, void *workspace, hipStream_t stream)
{
    hipError_t e = hipSuccess;
#define CALL(G, W) e = pick_bwd<G, W>(a, grad, grad_stride, dweight, dweight_stride, padding, accumulate, workspace, stream)
    LM_TYPE_PAIR(grad_dt, dweight_dt, CALL)
#undef CALL
    return e;
}

}  // namespace lm
