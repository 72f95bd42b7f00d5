// lm_norm.hip -- how the residual norms' work is shared out, the addition of the backward pass's
// partial rows, and the choice of the kernels (lm_norm_kernel.h).
#include "lm_common.h"
#include "lm_norm.h"

namespace lm {
namespace {

// Workgroups of the backward pass (each leaves a partial row) and of the forward pass: as many waves as
// the chip holds of each (16 a CU).
int most_wgs(int waves) { return waves <= 4 ? 1024 : waves <= 8 ? 512 : 256; }

// Adds the partial rows: blockIdx.y names the sum (4 and up: the groups of the gate).  64 columns a
// workgroup, its 16 waves take every 16th partial row (without rows there are none: zeros, for any number of
// groups, those beyond GATES_Y along blockIdx.z).  1024 partial rows of 768 4.5 us, 512 of 4096 9.4 us.
constexpr int GATES_Y = 32768;
__global__ __launch_bounds__(1024) void norm_finish_kernel(NormArgs a, NormSplit sp)
{
    __shared__ float buf[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int which = min((int)blockIdx.y, 4);
    void *out = which == 0 ? a.dpre_weight : which == 1 ? a.dpre_bias : which == 2 ? a.dpost_weight : which == 3 ? a.dpost_bias : a.dgate;
    const int64_t group = (int64_t)blockIdx.z * GATES_Y + blockIdx.y - 4;
    if (!out || (which == 4 ? group >= a.groups : blockIdx.z != 0)) return;
    int64_t first = 0, rows = sp.wgs, to = 0;
    if (which == 4) {
        first = group * sp.per_group;
        rows = sp.per_group;
        to = group * a.dim;
    }
    const int64_t col = (int64_t)blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (col < a.dim) {
        const float *p = a.workspace + (which * (int64_t)sp.wgs + first) * a.dim + col;
#pragma unroll 8
        for (int64_t r = wave; r < rows; r += 16) s += p[r * a.dim];
    }
    buf[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && col < a.dim) {
        for (int w = 1; w < 16; w++) s += buf[w][lane];
        store_any(a.weight_dt, out, to + col, s);
    }
}

int size_of(int dt) { return dt == DT_F32 ? 4 : 2; }

NormSplit split_of(int64_t n, int64_t dim, int64_t groups)
{
    NormSplit s;
    const int64_t waves = (dim + 511) / 512;
    s.waves = (int)waves;
    const int rows = waves == 1 ? 4 : waves == 2 ? 2 : 1, most = most_wgs(s.waves);
    s.fwd_wgs = most;
    s.per_group = 0;
    if (groups <= most) {
        const int64_t rpg = n / groups, each = (rpg + rows - 1) / rows;
        int64_t per = most / groups;
        if (per > each) per = each;
        s.per_group = (int)(per < 1 ? 1 : per);
        s.wgs = (int)groups * s.per_group;
    } else {
        const int64_t wgs = (groups + rows - 1) / rows;
        s.wgs = (int)(wgs < most ? wgs : most);
    }
    return s;
}

// Whether every row of every array can be read and written 16 bytes at a time.
bool wide(const NormArgs &a, bool backward)
{
    const int z = size_of(a.dt), vec = 16 / z;
    auto row = [&](const void *p, int64_t stride) { return (uintptr_t)p % 16 == 0 && stride * z % 16 == 0; };
    auto vector = [&](const void *p) { return (uintptr_t)p % 16 == 0; };
    if (a.dim % vec) return false;
    if (!(row(a.x, a.x_stride) && row(a.block, a.block_stride) && vector(a.pre_weight) && vector(a.pre_bias) && vector(a.post_weight) &&
          vector(a.post_bias) && vector(a.gate)))
        return false;
    if (!backward) return row(a.r, a.dim) && row(a.h, a.dim);
    return row(a.dh, a.dh_stride) && row(a.dr, a.dr_stride) && row(a.dx, a.dim) && row(a.dblock, a.dim);
}

hipError_t by_type(const NormArgs &a, bool backward, hipStream_t stream)
{
    // (without rows the sums of no partial rows are written: zeros)
    const NormSplit sp = a.n ? split_of(a.n, a.dim, a.groups) : NormSplit{0, 0, 0, 0};
    const bool ragged = !wide(a, backward);
    hipError_t e = hipSuccess;
    if (a.n)
        e = a.dt == DT_F32                  ? norm_run<DT_F32, true>(a, sp, ragged, backward, stream)
            : a.dt == DT_BF16 && a.weight_dt ? norm_run<DT_BF16, false>(a, sp, ragged, backward, stream)
            : a.dt == DT_BF16                ? norm_run<DT_BF16, true>(a, sp, ragged, backward, stream)
            : a.weight_dt                    ? norm_run<DT_F16, false>(a, sp, ragged, backward, stream)
                                             : norm_run<DT_F16, true>(a, sp, ragged, backward, stream);
    if (e != hipSuccess || !backward) return e;
    const int64_t gates = a.gate && (sp.per_group || !a.n) ? a.groups : 0;
    norm_finish_kernel<<<dim3((unsigned)((a.dim + 63) / 64), 4 + (unsigned)(gates < GATES_Y ? gates : GATES_Y),
                              gates ? (unsigned)((gates + GATES_Y - 1) / GATES_Y) : 1), 1024, 0, stream>>>(a, sp);
    return hipGetLastError();
}

}  // namespace

hipError_t norm_forward(const NormArgs &a, hipStream_t stream) { return by_type(a, false, stream); }

int64_t norm_backward_workspace(int64_t n, int64_t dim, int64_t groups) { return 5ll * split_of(n, dim, groups).wgs * dim * 4; }

hipError_t norm_backward(const NormArgs &a, hipStream_t stream) { return by_type(a, true, stream); }

}  // namespace lm
