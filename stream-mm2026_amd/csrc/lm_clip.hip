// lm_clip.hip -- the global norm of a list of gradients, and the gradients scaled to it.
//
//   norm = sqrt(sum over all tensors of g^2),  out = g min(1, max_norm / (norm + 1e-6))
//
// Squares and sums are doubles: no gradient that is a float overflows or vanishes in them, and the order of the sums does not
// show in a float.  A tensor list travels as kernel arguments, 160 tensors a launch (no table to upload, so a call can
// be captured).  Memory bound: the gradients are read twice, as their norm must be known before the first is written: GPT-2
// small's in fp32 95 us for the norm (5.2 TB/s) and 176 for the scaling (5.7), 1.88 G elements of bf16 680 (5.5) and 1444 (5.2).
// Results are stored past the caches.  What follows decides little: with the gradients written before and the 4-bit optimizer's
// step behind, clipping adds 268-270 us to GPT-2 small's, 91-103 to 30 M parameters and 54-64 to 2.4 M, with ordinary stores 270-272,
// 98-101 and 63-67.  (In a loop of clippings alone, written-back results slow the next norm: 129 us.)
// Every workgroup of the scaling adds up the norm's partial sums for itself, up to 2048 doubles for each launch of the norm: 1.13 G
// elements of bf16 take 1260 us as 160 or 320 tensors, 1310 as 1080, 1590 as 2160 and 2680 as 4320 (the host's side of such a
// list is 4800).
#include "lm_clip.h"
#include "lm_common.h"

namespace lm {
namespace {

constexpr int LIST = 160;                 // tensors of a launch: 3.8 KB of arguments
constexpr int TILE = 32768;               // bytes a workgroup takes at a time, of one tensor (64 KB: the same times)
constexpr int WGS = 2048;                 // workgroups of a launch at most: eight a CU, all resident

struct List {
    const void *grad[LIST];
    void *out[LIST];
    int64_t numel_dt[LIST];               // elements (> 0), and the type in the lowest two bits
    uint32_t tiles;                       // all tiles of the launch
    int count;
};
static_assert(sizeof(List) <= 4000, "kernel arguments");

__host__ __device__ __forceinline__ int tile_of(int dt) { return dt == DT_F32 ? TILE / 4 : TILE / 2; }
__host__ __device__ __forceinline__ uint32_t tiles_of(int64_t numel_dt)
{
    const int tile = tile_of((int)(numel_dt & 3));
    return (uint32_t)(((numel_dt >> 2) + tile - 1) / tile);
}

// Which tensor a tile belongs to: lane l knows the first tiles of tensors l, 64 + l and 128 + l.
struct Starts {
    static constexpr int PARTS = (LIST + 63) / 64;
    uint32_t first[PARTS];
    __device__ __forceinline__ explicit Starts(const List &l)
    {
        const int lane = threadIdx.x & 63;
        uint32_t before = 0;
#pragma unroll
        for (int p = 0; p < PARTS; p++) {
            const int t = 64 * p + lane;
            const uint32_t mine = t < l.count ? tiles_of(l.numel_dt[t]) : 0;
            uint32_t upto = mine;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t o = __shfl_up(upto, d, 64);
                if (lane >= d) upto += o;
            }
            first[p] = t < l.count ? before + upto - mine : 0xffffffffu;
            before += __builtin_amdgcn_readlane(upto, 63);
        }
    }
    // the tensor, and the tile's place in it
    __device__ __forceinline__ int of(uint32_t tile, uint32_t &in) const
    {
        int t = -1;
#pragma unroll
        for (int p = 0; p < PARTS; p++) t += __popcll(__ballot(first[p] <= tile));
        in = tile;
#pragma unroll
        for (int p = 0; p < PARTS; p++)
            if (t >> 6 == p) in -= __builtin_amdgcn_readlane(first[p], t & 63);
        return t;
    }
};

__device__ __forceinline__ double wave_add(double v)
{
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
    return v;
}
__device__ __forceinline__ double group_add(double v, double *buf)
{
    v = wave_add(v);
    if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
    __syncthreads();
    return (buf[0] + buf[1]) + (buf[2] + buf[3]);
}

template <int DT>
__device__ __forceinline__ double squares(const void *p, int64_t at, int n)
{
    constexpr int PER = Elem<DT>::PER16, FLY = 4;
    double s0 = 0.0, s1 = 0.0;
    const int pieces = n / PER;
    for (int i = threadIdx.x; i < pieces; i += 256 * FLY) {
        float v[FLY][PER];
#pragma unroll
        for (int u = 0; u < FLY; u++) {
            if (i + u * 256 < pieces) load_n<DT, PER, true>(p, at + (int64_t)(i + u * 256) * PER, v[u]);
            else
#pragma unroll
                for (int k = 0; k < PER; k++) v[u][k] = 0.0f;
        }
#pragma unroll
        for (int u = 0; u < FLY; u++)
#pragma unroll
            for (int k = 0; k < PER; k += 2) {
                s0 = fma((double)v[u][k], (double)v[u][k], s0);
                s1 = fma((double)v[u][k + 1], (double)v[u][k + 1], s1);
            }
    }
    const int rest = pieces * PER + threadIdx.x;
    if (rest < n) {
        const double v = Elem<DT>::load(p, at + rest);
        s0 = fma(v, v, s0);
    }
    return s0 + s1;
}

__global__ __launch_bounds__(256) void clip_norm_kernel(List l, double *partial)
{
    __shared__ double buf[4];
    const Starts starts(l);
    double s = 0.0;
    for (uint32_t tile = blockIdx.x; tile < l.tiles; tile += gridDim.x) {
        uint32_t in;
        const int t = starts.of(tile, in);
        const int dt = (int)(l.numel_dt[t] & 3), tile_n = tile_of(dt);
        const int64_t numel = l.numel_dt[t] >> 2, at = (int64_t)in * tile_n;
        const int n = (int)(numel - at < tile_n ? numel - at : tile_n);
        if (dt == DT_F32) s += squares<DT_F32>(l.grad[t], at, n);
        else if (dt == DT_BF16) s += squares<DT_BF16>(l.grad[t], at, n);
        else s += squares<DT_F16>(l.grad[t], at, n);
    }
    s = group_add(s, buf);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// The sum of all partial sums, in one order whoever forms it.
__device__ __forceinline__ double all_partials(const double *partial, int64_t count, double *buf)
{
    double s = 0.0;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < count; i += 256) s += partial[i];
    return group_add(s, buf);
}

__global__ __launch_bounds__(256) void clip_finish_kernel(const double *partial, int64_t count, float *norm)
{
    __shared__ double buf[4];
    const double s = all_partials(partial, count, buf);
    if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

// The scale as a float in [0.5, 1] and a power of two: a norm beyond the floats' range makes one that no normal float holds
// (gradients of 3e38 scaled to 1 were off by 1e-5).
struct Scale {
    float m;
    int e;
    __device__ __forceinline__ explicit Scale(double ratio)
    {
        m = 1.0f, e = 0;
        if (ratio >= 1.0) return;
        m = (float)frexp(ratio, &e);
        if (!(fabs(ratio) <= 1.0)) m = (float)ratio, e = 0;      // NaN
    }
    __device__ __forceinline__ bool one() const { return m == 1.0f && e == 0; }
    __device__ __forceinline__ float of(float g) const { return ldexpf(g * m, e); }
};

template <int DT>
__device__ __forceinline__ void scale_tile(const void *p, void *out, int64_t at, int n, Scale c)
{
    constexpr int PER = Elem<DT>::PER16, FLY = 4;
    const int pieces = n / PER;
    for (int i = threadIdx.x; i < pieces; i += 256 * FLY) {
        float v[FLY][PER];
#pragma unroll
        for (int u = 0; u < FLY; u++)
            if (i + u * 256 < pieces) load_n<DT, PER, true>(p, at + (int64_t)(i + u * 256) * PER, v[u]);
#pragma unroll
        for (int u = 0; u < FLY; u++)
            if (i + u * 256 < pieces) {
#pragma unroll
                for (int k = 0; k < PER; k++) v[u][k] = c.of(v[u][k]);
                __builtin_nontemporal_store(Elem<DT>::pack(v[u]), (u32x4_any *)((char *)out + (at + (int64_t)(i + u * 256) * PER) * Elem<DT>::SIZE));
            }
    }
    const int rest = pieces * PER + threadIdx.x;
    if (rest < n) Elem<DT>::store(out, at + rest, c.of(Elem<DT>::load(p, at + rest)));
}

// The tiles from the last to the first: what the norm's pass read last may still be in the last-level cache.
__global__ __launch_bounds__(256) void clip_scale_kernel(List l, const double *partial, int64_t partials, double max_norm, const float *given, float *norm)
{
    __shared__ double buf[4];
    const Starts starts(l);
    const double total = given ? (double)*given : sqrt(all_partials(partial, partials, buf));
    // (a norm above the floats is infinite in *norm alone, and a NaN makes every gradient one)
    const Scale c(max_norm / (total + 1e-6));
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)total;
    for (uint32_t i = blockIdx.x; i < l.tiles; i += gridDim.x) {
        const uint32_t tile = l.tiles - 1 - i;
        uint32_t in;
        const int t = starts.of(tile, in);
        // gradients in place that keep their values need no write
        if (c.one() && l.grad[t] == l.out[t]) continue;
        const int dt = (int)(l.numel_dt[t] & 3), tile_n = tile_of(dt);
        const int64_t numel = l.numel_dt[t] >> 2, at = (int64_t)in * tile_n;
        const int n = (int)(numel - at < tile_n ? numel - at : tile_n);
        if (dt == DT_F32) scale_tile<DT_F32>(l.grad[t], l.out[t], at, n, c);
        else if (dt == DT_BF16) scale_tile<DT_BF16>(l.grad[t], l.out[t], at, n, c);
        else scale_tile<DT_F16>(l.grad[t], l.out[t], at, n, c);
    }
}

// Tensors from `i` on as one launch's list; where the next begins.
int64_t gather(const ClipTensor *t, int64_t count, int64_t i, List &l)
{
    uint32_t tiles = 0;                   // (below 2^31: CLIP_MAX_NUMEL)
    l.count = 0;
    for (; i < count && l.count < LIST; i++) {
        if (t[i].numel == 0) continue;
        const int k = l.count++;
        l.grad[k] = t[i].grad;
        l.out[k] = t[i].out;
        l.numel_dt[k] = t[i].numel << 2 | t[i].dt;
        tiles += tiles_of(l.numel_dt[k]);
    }
    l.tiles = tiles;
    return i;
}
unsigned wgs_of(const List &l) { return l.tiles < WGS ? l.tiles : WGS; }

hipError_t norm_launches(const ClipTensor *t, int64_t count, double *partial, int64_t &partials, hipStream_t stream)
{
    partials = 0;
    List l;
    for (int64_t i = 0; i < count;) {
        i = gather(t, count, i, l);
        if (l.tiles == 0) continue;
        clip_norm_kernel<<<wgs_of(l), 256, 0, stream>>>(l, partial + partials);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        partials += wgs_of(l);
    }
    return hipSuccess;
}

}  // namespace

static_assert((CLIP_MAX_NUMEL * 4 / TILE) * LIST < (1ll << 31), "tiles of a launch");

int64_t clip_workspace(int64_t count) { return ((count + LIST - 1) / LIST * WGS + 1) * 8; }

hipError_t clip_norm(const ClipTensor *t, int64_t count, double *partial, float *norm, hipStream_t stream)
{
    int64_t partials;
    const hipError_t e = norm_launches(t, count, partial, partials, stream);
    if (e != hipSuccess) return e;
    clip_finish_kernel<<<1, 256, 0, stream>>>(partial, partials, norm);
    return hipGetLastError();
}

hipError_t clip_scale(const ClipTensor *t, int64_t count, double max_norm, const float *given, double *partial, float *norm, hipStream_t stream)
{
    int64_t partials = 0;
    if (!given) {
        const hipError_t e = norm_launches(t, count, partial, partials, stream);
        if (e != hipSuccess) return e;
    }
    List l;
    bool any = false;
    for (int64_t i = 0; i < count;) {
        i = gather(t, count, i, l);
        if (l.tiles == 0) continue;
        clip_scale_kernel<<<wgs_of(l), 256, 0, stream>>>(l, partial, partials, max_norm, given, any ? nullptr : norm);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        any = true;
    }
    if (!any && !given) {                 // no gradients: a norm of 0
        clip_finish_kernel<<<1, 256, 0, stream>>>(partial, 0, norm);
        return hipGetLastError();
    }
    return hipSuccess;
}

}  // namespace lm
