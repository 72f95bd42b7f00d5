// lm_route.hip -- routing of tokens to experts: softmax and top k of a row of logits, the slots sorted by expert, and the
// weighted sum of a token's results.
//
//   p = softmax(z),  chosen: the k largest z (ties: the lowest expert; -inf: never),  w = p, or p / (sum of the chosen p)
//   load[e] = sum over the rows of p[e]
//   dz = p (dl - <p, dl> - [not renormalised] <w, dw>) + [chosen] w (dw - [renormalised] <w, dw>)
//
// Rows are short (experts), so they live in registers: a row's experts are spread over 8 to 64 lanes, several rows a wave
// where they are few.  What bounds these kernels is latency, launches above all: 8192 rows of 64 experts with 6 choices take 8.5
// us for the choices (15 with exchanges through LDS and an exponential a choice), 4 for the load's sums, 10 for the plan
// and 5.6 for the gradient, of 1 MB each way.
#include "lm_common.h"
#include "lm_expert.h"

namespace lm {
namespace {

constexpr int ROUTE_WGS = 1024;           // workgroups at most: each adds a row of partial loads

// A float as an integer of the same order, NaN above all, -0 as 0; 0: absent (-inf, or no expert).
__device__ __forceinline__ uint32_t ordered(float z)
{
    if (z == -__builtin_inff()) return 0;
    if (z != z) return 0xffffffffu;
    const uint32_t u = __float_as_uint(z == 0.0f ? 0.0f : z);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t key)
{
    if (key == 0xffffffffu) return __builtin_nanf("");
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// Over the L lanes of a row without LDS: pairs, quads, halves and rows of 16 mirrored (DPP), then rows and halves of the wave
// swapped.  Both sides of each exchange combine the same two values, so every lane ends with the same bits.
template <int CTRL>
__device__ __forceinline__ uint32_t moved(uint32_t v) { return __builtin_amdgcn_update_dpp(v, v, CTRL, 0xf, 0xf, false); }
template <int L, typename T, typename F>
__device__ __forceinline__ T row_reduce(T v, F op)
{
    auto with = [&](uint32_t other) { return op(v, __builtin_bit_cast(T, other)); };
    v = with(moved<0xb1>(__builtin_bit_cast(uint32_t, v)));
    v = with(moved<0x4e>(__builtin_bit_cast(uint32_t, v)));
    v = with(moved<0x141>(__builtin_bit_cast(uint32_t, v)));
    if constexpr (L >= 16) v = with(moved<0x140>(__builtin_bit_cast(uint32_t, v)));
    if constexpr (L >= 32) {
        const uint32_t w = __builtin_bit_cast(uint32_t, v);
        const auto rows = __builtin_amdgcn_permlane16_swap(w, w, false, false);
        v = op(__builtin_bit_cast(T, (uint32_t)rows[0]), __builtin_bit_cast(T, (uint32_t)rows[1]));
    }
    if constexpr (L >= 64) {
        const uint32_t w = __builtin_bit_cast(uint32_t, v);
        const auto halves = __builtin_amdgcn_permlane32_swap(w, w, false, false);
        v = op(__builtin_bit_cast(T, (uint32_t)halves[0]), __builtin_bit_cast(T, (uint32_t)halves[1]));
    }
    return v;
}
struct MaxKey {
    __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return a > b ? a : b; }
};

// One row's softmax: expert lane + L i in slot i of the lane.  p of a row without experts is 0.
template <int DT, int L, int C>
struct Row {
    float z[C], p[C];
    float top, total;

    __device__ __forceinline__ void read(const RouteArgs &a, int64_t row, int l)
    {
#pragma unroll
        for (int i = 0; i < C; i++) {
            const int e = l + L * i;
            z[i] = row < a.n && e < a.experts ? Elem<DT>::load(a.logits, row * a.stride + e) : -__builtin_inff();
        }
    }
    __device__ __forceinline__ void softmax()
    {
        top = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < C; i++) top = Max()(top, z[i]);
        top = row_reduce<L>(top, Max());
        const float from = top == -__builtin_inff() ? 0.0f : top;
        total = 0.0f;
#pragma unroll
        for (int i = 0; i < C; i++) {
            p[i] = expf(z[i] - from);
            total += p[i];
        }
        total = row_reduce<L>(total, Add());
        const float share = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
        for (int i = 0; i < C; i++) p[i] *= share;
    }
};

template <int DT, int L, int C>
__global__ __launch_bounds__(256) void route_kernel(RouteArgs a)
{
    constexpr int ROWS = 256 / L;
    __shared__ float sums[ROWS][L * C];
    const int lane = threadIdx.x & 63, l = threadIdx.x & (L - 1), r = threadIdx.x / L, first = lane & ~(L - 1);
    float load[C] = {};
    Row<DT, L, C> x, next;
    next.read(a, (int64_t)blockIdx.x * ROWS + r, l);
    for (int64_t row0 = (int64_t)blockIdx.x * ROWS; row0 < a.n; row0 += (int64_t)gridDim.x * ROWS) {
        const int64_t row = row0 + r;
        const bool live = row < a.n;
        x = next;
        next.read(a, row + (int64_t)gridDim.x * ROWS, l);
        x.softmax();
        uint32_t key[C];
#pragma unroll
        for (int i = 0; i < C; i++) {
            key[i] = ordered(x.z[i]);
            load[i] += x.p[i];
        }
        // the k largest in turn; lane j of the row keeps the j-th (as many as 64 of them: a row of 64 lanes)
        uint32_t mine = 0;
        int id = -1;
        for (int j = 0; j < a.k; j++) {
            uint32_t best = 0;
#pragma unroll
            for (int i = 0; i < C; i++) best = MaxKey()(best, key[i]);
            best = row_reduce<L>(best, MaxKey());
            int at = -1;
#pragma unroll
            for (int i = 0; i < C; i++) {
                // the lowest expert of a tie: slot by slot, lane by lane
                uint64_t has = __ballot(key[i] == best && best != 0 && at < 0) >> first;
                if constexpr (L < 64) has &= (1ull << L) - 1;
                if (has) {
                    const int who = __builtin_ctzll(has);
                    at = who + L * i;
                    if (l == who) key[i] = 0;
                }
            }
            if (l == j) {
                mine = best;
                id = at;
            }
        }
        float w = id < 0 ? 0.0f : expf(from_ordered(mine) - x.top) / x.total;
        const float chosen = row_reduce<L>(w, Add());
        if (live && l < a.k) {
            if (a.renormalize && id >= 0) w /= chosen;
            a.weights[row * a.k + l] = w;
            a.ids[row * a.k + l] = id;
        }
    }
    if (!a.load) return;
#pragma unroll
    for (int i = 0; i < C; i++) sums[r][l + L * i] = load[i];
    __syncthreads();
    float *out = gridDim.x == 1 ? a.load : a.partial + (int64_t)blockIdx.x * a.experts;
    for (int e = threadIdx.x; e < a.experts; e += 256) {
        float s = 0.0f;
        for (int i = 0; i < ROWS; i++) s += sums[i][e];
        out[e] = s;
    }
}

// load[e] from the workgroups' sums: 16 experts a workgroup, 16 runs of the sums for each.
__global__ __launch_bounds__(256) void load_kernel(const float *partial, int rows, int experts, float *load)
{
    __shared__ float sums[16][17];
    const int c = threadIdx.x & 15, run = threadIdx.x >> 4, e = blockIdx.x * 16 + c;
    const int each = (rows + 15) / 16, end = min(rows, (run + 1) * each);
    float s = 0.0f;
    if (e < experts)
#pragma unroll 8
        for (int i = run * each; i < end; i++) s += partial[(int64_t)i * experts + e];
    sums[run][c] = s;
    __syncthreads();
    if (run == 0 && e < experts) {
        s = 0.0f;
        for (int i = 0; i < 16; i++) s += sums[i][c];
        load[e] = s;
    }
}

template <int DT, int L, int C>
__global__ __launch_bounds__(256) void route_back_kernel(RouteArgs a)
{
    constexpr int ROWS = 256 / L;
    const int lane = threadIdx.x & 63, l = threadIdx.x & (L - 1), r = threadIdx.x / L, first = lane & ~(L - 1);
    for (int64_t row0 = (int64_t)blockIdx.x * ROWS; row0 < a.n; row0 += (int64_t)gridDim.x * ROWS) {
        const int64_t row = row0 + r;
        const bool live = row < a.n;
        Row<DT, L, C> x;
        x.read(a, row, l);
        x.softmax();
        // lane j: the j-th choice
        int id = -1;
        float w = 0.0f, dw = 0.0f;
        if (live && l < a.k) {
            id = a.ids[row * a.k + l];
            if (id >= 0 && a.dweights) {
                w = a.weights[row * a.k + l];
                dw = a.dweights[row * a.k + l];
            }
        }
        const float inner = row_reduce<L>(w * dw, Add());
        float dl[C], mean = 0.0f;
#pragma unroll
        for (int i = 0; i < C; i++) {
            const int e = l + L * i;
            dl[i] = a.dload && e < a.experts ? a.dload[e] : 0.0f;
            mean += x.p[i] == 0.0f ? 0.0f : x.p[i] * dl[i];
        }
        mean = row_reduce<L>(mean, Add());
        const float all = mean + (a.renormalize ? 0.0f : inner);
        const float own = w * (dw - (a.renormalize ? inner : 0.0f));
        float dz[C];
#pragma unroll
        for (int i = 0; i < C; i++) dz[i] = x.p[i] == 0.0f ? 0.0f : x.p[i] * (dl[i] - all);
        for (int j = 0; j < a.k; j++) {
            const int at = __shfl(id, first + j, 64);
            const float add = __shfl(own, first + j, 64);
#pragma unroll
            for (int i = 0; i < C; i++) dz[i] += at == l + L * i ? add : 0.0f;
        }
        if (live)
#pragma unroll
            for (int i = 0; i < C; i++)
                if (l + L * i < a.experts) Elem<DT>::store(a.dlogits, row * a.dstride + l + L * i, dz[i]);
    }
}

int row_wgs(int64_t n, int rows)
{
    const int64_t wgs = (n + rows - 1) / rows;
    return (int)(wgs < ROUTE_WGS ? wgs : ROUTE_WGS);
}

// f<DT, L, C>() for the type, and the lanes and slots of a row of `experts`.
template <int DT, typename F>
void for_shape(int experts, F f)
{
    if (experts <= 8) f.template operator()<DT, 8, 1>();
    else if (experts <= 16) f.template operator()<DT, 16, 1>();
    else if (experts <= 32) f.template operator()<DT, 32, 1>();
    else if (experts <= 64) f.template operator()<DT, 64, 1>();
    else if (experts <= 128) f.template operator()<DT, 64, 2>();
    else if (experts <= 256) f.template operator()<DT, 64, 4>();
    else f.template operator()<DT, 64, 8>();
}
template <typename F>
void for_type(int dt, int experts, F f)
{
    if (dt == DT_F32) for_shape<DT_F32>(experts, f);
    else if (dt == DT_BF16) for_shape<DT_BF16>(experts, f);
    else for_shape<DT_F16>(experts, f);
}

// ---------------------------------------------------------------- plan
// A stable counting sort by expert.  Each of 16 waves owns a run of the slots: it counts them by expert in LDS, the runs'
// places follow by sums over experts, workgroups and waves, and the wave then places its slots 64 at a time, those of one
// expert found by a ballot for each bit of it.  Few slots take one workgroup, more of them one launch that counts before.
constexpr int PLAN_WAVES = 16, PLAN_EACH = 128;       // slots of a wave (256: 13 us in place of 10 for 49152 slots)
constexpr int PLAN_WGS = 256;

__device__ __forceinline__ int bucket(const void *ids, int bytes, int64_t i, int experts)
{
    const int64_t e = bytes == 8 ? ((const int64_t *)ids)[i] : ((const int32_t *)ids)[i];
    return e >= 0 && e < experts ? (int)e : experts;      // the last one: no expert
}

template <bool COUNT, bool ALONE>
__global__ __launch_bounds__(PLAN_WAVES * 64) void plan_kernel(PlanArgs a, int64_t each)
{
    __shared__ int count[PLAN_WAVES][EXPERT_MAX + 1];
    __shared__ int sums[PLAN_WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, buckets = a.experts + 1;
    for (int i = threadIdx.x; i < PLAN_WAVES * (EXPERT_MAX + 1); i += PLAN_WAVES * 64) (&count[0][0])[i] = 0;
    __syncthreads();
    const int64_t first = min(a.slots, ((int64_t)blockIdx.x * PLAN_WAVES + wave) * each), last = min(a.slots, first + each);
    // (four loads on their way at a time)
    for (int64_t i0 = first + lane; i0 < last; i0 += 4 * 64) {
        int e[4];
#pragma unroll
        for (int u = 0; u < 4; u++) e[u] = i0 + 64 * u < last ? bucket(a.ids, a.id_bytes, i0 + 64 * u, a.experts) : -1;
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (e[u] >= 0) atomicAdd(&count[wave][e[u]], 1);
    }
    __syncthreads();
    const int b = threadIdx.x;
    int here = 0;
    if (b < buckets)
        for (int w = 0; w < PLAN_WAVES; w++) here += count[w][b];
    if constexpr (COUNT) {
        if (b < buckets) a.hist[(int64_t)blockIdx.x * buckets + b] = here;
        return;
    }
    // the slots of this bucket in all workgroups, and in those before this one
    int total = here, before = 0;
    if constexpr (!ALONE) {
        total = 0;
        if (b < buckets)
#pragma unroll 8
            for (int g = 0; g < (int)gridDim.x; g++) {
                const int n = a.hist[(int64_t)g * buckets + b];
                before += g < (int)blockIdx.x ? n : 0;
                total += n;
            }
    }
    int upto = total;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(upto, d, 64);
        if (lane >= d) upto += o;
    }
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    int start = upto - total;
    for (int w = 0; w < wave; w++) start += sums[w];
    if (b < buckets) {
        if (blockIdx.x == 0) a.offsets[b] = start;
        int at = start + before;
        for (int w = 0; w < PLAN_WAVES; w++) {
            const int n = count[w][b];
            count[w][b] = at;
            at += n;
        }
    }
    __syncthreads();
    const int bits = 32 - __builtin_clz(buckets);
    const uint64_t lower = (1ull << lane) - 1;
    for (int64_t i0 = first; i0 < last; i0 += 4 * 64) {
        int e[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int64_t i = i0 + 64 * u + lane;
            e[u] = i < last ? bucket(a.ids, a.id_bytes, i, a.experts) : -1;
        }
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const bool valid = e[u] >= 0;
            uint64_t same = __ballot(valid);
            if (same == 0) break;
            for (int k = 0; k < bits; k++) {
                const uint64_t set = __ballot(valid && (e[u] >> k & 1));
                same &= e[u] >> k & 1 ? set : ~set;
            }
            int at = 0;
            if (valid) at = count[wave][e[u]] + __popcll(same & lower);
            __builtin_amdgcn_wave_barrier();
            if (valid && !(same & lower)) count[wave][e[u]] += __popcll(same);
            __builtin_amdgcn_wave_barrier();
            if (valid) {
                const int64_t i = i0 + 64 * u + lane;
                a.rows[at] = (int)i;
                a.places[i] = at;
            }
        }
    }
}

int64_t plan_each(int64_t slots)
{
    const int64_t most = (int64_t)PLAN_WAVES * PLAN_WGS, each = (slots + most - 1) / most;
    return each <= PLAN_EACH ? PLAN_EACH : (each + 63) / 64 * 64;
}
int plan_wgs(int64_t slots)
{
    const int64_t wg = plan_each(slots) * PLAN_WAVES;
    return (int)((slots + wg - 1) / wg);
}

// ---------------------------------------------------------------- combination
// A wave a token: its k rows of y are read piece by piece, four of them in flight.  Bound by memory: 16384 x 2 rows of 4096 (bf16) 90
// us, 4.3 TB/s, and backward 139, 4.7.  Pieces are taken at any alignment, so that the order of a sum does not go by it.
constexpr int COMBINE_WGS = 1 << 16;

// N elements of a row of dim from column c on: the last piece may be short.
template <int DT, int N>
__device__ __forceinline__ void load_piece(const void *p, int64_t row, int64_t c, int64_t dim, float *v)
{
    if (c + N <= dim) return load_n<DT, N, true>(p, row + c, v);
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = c + i < dim ? Elem<DT>::load(p, row + c + i) : 0.0f;
}
template <int DT, int N>
__device__ __forceinline__ void store_piece(void *p, int64_t row, int64_t c, int64_t dim, const float *v)
{
    if (c + N <= dim) return store_n<DT, N, true>(p, row + c, v);
#pragma unroll
    for (int i = 0; i < N; i++)
        if (c + i < dim) Elem<DT>::store(p, row + c + i, v[i]);
}

template <int YDT, int ODT, int VEC>
__global__ __launch_bounds__(256) void combine_kernel(CombineArgs a)
{
    const int lane = threadIdx.x & 63;
    const int live = (int)min((int64_t)a.offsets[a.experts], a.n * a.k);
    for (int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); t < a.n; t += (int64_t)gridDim.x * 4) {
        int place = -1;
        float weight = 0.0f;
        if (lane < a.k) {
            place = a.places[t * a.k + lane];
            weight = a.weights ? a.weights[t * a.k + lane] : 1.0f;
            if (place < 0 || place >= live) place = -1;
        }
        for (int64_t c = lane * VEC; c < a.dim; c += 64 * VEC) {
            float acc[VEC] = {};
            for (int j0 = 0; j0 < a.k; j0 += 4) {
                float y[4][VEC];
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const int p = j0 + u < a.k ? __builtin_amdgcn_readlane(place, j0 + u) : -1;
                    if (p >= 0) load_piece<YDT, VEC>(a.y, p * a.y_stride, c, a.dim, y[u]);
                }
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    if (j0 + u >= a.k || __builtin_amdgcn_readlane(place, j0 + u) < 0) continue;
                    const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(weight), j0 + u));
#pragma unroll
                    for (int v = 0; v < VEC; v++) acc[v] = fmaf(w, y[u][v], acc[v]);
                }
            }
            store_piece<ODT, VEC>(a.out, t * a.out_stride, c, a.dim, acc);
        }
    }
}

// dy = w dout, dw = <y, dout>; rows of no expert get zeros.  Up to four of a token's rows at a time.
template <int DT, int VEC>
__global__ __launch_bounds__(256) void combine_back_kernel(CombineArgs a)
{
    const int lane = threadIdx.x & 63;
    const int64_t slots = a.n * a.k;
    const int live = (int)min((int64_t)a.offsets[a.experts], slots);
    for (int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); t < a.n; t += (int64_t)gridDim.x * 4) {
        int place = -1;
        float weight = 0.0f, dweight = 0.0f;
        if (lane < a.k) {
            place = a.places[t * a.k + lane];
            weight = a.weights ? a.weights[t * a.k + lane] : 1.0f;
            if (place < 0 || place >= slots) place = -1;
        }
        for (int j0 = 0; j0 < a.k; j0 += 4) {
            float dot[4] = {};
            for (int64_t c = lane * VEC; c < a.dim; c += 64 * VEC) {
                float g[VEC], y[4][VEC];
                load_piece<DT, VEC>(a.dout, t * a.dout_stride, c, a.dim, g);
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const int p = j0 + u < a.k ? __builtin_amdgcn_readlane(place, j0 + u) : -1;
                    if (a.dweights && p >= 0 && p < live) load_piece<DT, VEC>(a.y, p * a.y_stride, c, a.dim, y[u]);
                }
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const int p = j0 + u < a.k ? __builtin_amdgcn_readlane(place, j0 + u) : -1;
                    if (p < 0) continue;
                    const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(weight), j0 + u));
                    float dy[VEC];
#pragma unroll
                    for (int v = 0; v < VEC; v++) dy[v] = p < live ? w * g[v] : 0.0f;
                    store_piece<DT, VEC>(a.dy, p * a.dim, c, a.dim, dy);
                    if (a.dweights && p < live)
#pragma unroll
                        for (int v = 0; v < VEC; v++) dot[u] = fmaf(g[v], y[u][v], dot[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const float d = wave_reduce(dot[u], Add());
                if (lane == j0 + u) dweight = d;
            }
        }
        if (a.dweights && lane < a.k) a.dweights[t * a.k + lane] = dweight;
    }
}

unsigned token_wgs(int64_t n) { return (unsigned)((n + 3) / 4 < COMBINE_WGS ? (n + 3) / 4 : COMBINE_WGS); }

template <int YDT, int ODT>
void launch_combine(const CombineArgs &a, hipStream_t stream)
{
    combine_kernel<YDT, ODT, YDT == DT_F32 ? 4 : 8><<<token_wgs(a.n), 256, 0, stream>>>(a);
}

template <int DT>
void launch_combine_back(const CombineArgs &a, hipStream_t stream)
{
    combine_back_kernel<DT, DT == DT_F32 ? 4 : 8><<<token_wgs(a.n), 256, 0, stream>>>(a);
}

}  // namespace

int64_t route_workspace(int64_t n, int experts)
{
    int wgs = 1;
    for_shape<DT_F32>(experts, [&]<int DT, int L, int C>() { wgs = row_wgs(n, 256 / L); });
    return wgs <= 1 ? 0 : (int64_t)wgs * experts * 4;
}

hipError_t route_forward(const RouteArgs &a, hipStream_t stream)
{
    int wgs = 1;
    for_type(a.dt, a.experts, [&]<int DT, int L, int C>() {
        wgs = a.n ? row_wgs(a.n, 256 / L) : 1;
        route_kernel<DT, L, C><<<wgs, 256, 0, stream>>>(a);
    });
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !a.load || wgs == 1) return e;
    load_kernel<<<(a.experts + 15) / 16, 256, 0, stream>>>(a.partial, wgs, a.experts, a.load);
    return hipGetLastError();
}

hipError_t route_backward(const RouteArgs &a, hipStream_t stream)
{
    if (a.n == 0) return hipSuccess;
    for_type(a.dt, a.experts, [&]<int DT, int L, int C>() {
        const int64_t wgs = (a.n + 256 / L - 1) / (256 / L);
        route_back_kernel<DT, L, C><<<(unsigned)(wgs < 8192 ? wgs : 8192), 256, 0, stream>>>(a);
    });
    return hipGetLastError();
}

int64_t plan_workspace(int64_t slots, int experts)
{
    const int wgs = plan_wgs(slots);
    return wgs <= 1 ? 0 : (int64_t)wgs * (experts + 1) * 4;
}

hipError_t expert_plan(const PlanArgs &a, hipStream_t stream)
{
    const int wgs = plan_wgs(a.slots);
    const int64_t each = plan_each(a.slots);
    if (wgs <= 1) {
        plan_kernel<false, true><<<1, PLAN_WAVES * 64, 0, stream>>>(a, each);
        return hipGetLastError();
    }
    plan_kernel<true, false><<<wgs, PLAN_WAVES * 64, 0, stream>>>(a, each);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    plan_kernel<false, false><<<wgs, PLAN_WAVES * 64, 0, stream>>>(a, each);
    return hipGetLastError();
}

hipError_t combine_forward(const CombineArgs &a, hipStream_t stream)
{
    if (a.n == 0) return hipSuccess;
    if (a.y_dt == DT_F32) {
        if (a.out_dt == DT_F32) launch_combine<DT_F32, DT_F32>(a, stream);
        else if (a.out_dt == DT_BF16) launch_combine<DT_F32, DT_BF16>(a, stream);
        else launch_combine<DT_F32, DT_F16>(a, stream);
    } else if (a.y_dt == DT_BF16) launch_combine<DT_BF16, DT_BF16>(a, stream);
    else launch_combine<DT_F16, DT_F16>(a, stream);
    return hipGetLastError();
}

hipError_t combine_backward(const CombineArgs &a, hipStream_t stream)
{
    if (a.n == 0) return hipSuccess;
    if (a.y_dt == DT_F32) launch_combine_back<DT_F32>(a, stream);
    else if (a.y_dt == DT_BF16) launch_combine_back<DT_BF16>(a, stream);
    else launch_combine_back<DT_F16>(a, stream);
    return hipGetLastError();
}

}  // namespace lm
