// lm_common.h -- what the transformer operators' kernels share: element types, 16-byte pieces of
// a row, wave and workgroup reductions.  gfx950, 64-lane waves.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace lm {

enum { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };   // STQ_FLOAT, STQ_BFLOAT16, STQ_HALF

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <bool B, typename A, typename C>
struct Pick { typedef C T; };
template <typename A, typename C>
struct Pick<true, A, C> { typedef A T; };

// Two floats rounded to nearest even into one word (v_cvt_pk_bf16_f32 / v_cvt_f16_f32).
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b)
{
    const f32x2 v = {a, b};
    if constexpr (DT == DT_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}

template <int DT>
__device__ __forceinline__ f32x2 unpack2(uint32_t w)
{
    if constexpr (DT == DT_BF16)
        return f32x2{__builtin_bit_cast(float, w << 16), __builtin_bit_cast(float, w & 0xffff0000u)};
    else return __builtin_convertvector(__builtin_bit_cast(f16x2, w), f32x2);
}

// Elements of a type: its size, how many of them 16 bytes hold, single loads and stores.
template <int DT>
struct Elem {
    static constexpr int SIZE = DT == DT_F32 ? 4 : 2;
    static constexpr int PER16 = 16 / SIZE;

    static __device__ __forceinline__ float load(const void *p, int64_t i)
    {
        if constexpr (DT == DT_F32) return ((const float *)p)[i];
        else if constexpr (DT == DT_BF16) return __builtin_bit_cast(float, (uint32_t)((const uint16_t *)p)[i] << 16);
        else return (float)((const _Float16 *)p)[i];
    }
    static __device__ __forceinline__ void store(void *p, int64_t i, float v)
    {
        if constexpr (DT == DT_F32) ((float *)p)[i] = v;
        else if constexpr (DT == DT_BF16) ((uint16_t *)p)[i] = __builtin_bit_cast(uint16_t, (__bf16)v);
        else ((_Float16 *)p)[i] = (_Float16)v;
    }
    static __device__ __forceinline__ void unpack(u32x4 w, float *v)
    {
        if constexpr (DT == DT_F32) {
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] = __uint_as_float(w[k]);
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const f32x2 t = unpack2<DT>(w[k]);
                v[2 * k] = t[0];
                v[2 * k + 1] = t[1];
            }
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float *v)
    {
        u32x4 w;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if constexpr (DT == DT_F32) w[k] = __builtin_bit_cast(uint32_t, v[k]);
            else w[k] = pack2<DT>(v[2 * k], v[2 * k + 1]);
        }
        return w;
    }
};

// 16 and 8 bytes at any multiple of the elements' size (global memory takes such accesses; they
// cost what the cache lines that they touch cost).
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));

// N consecutive elements at p + i as floats, and back: one access per 16 bytes (N elements are 2 to
// 32 bytes).  ANY: p + i is aligned to an element only; otherwise to min(16, their bytes).
template <int DT, int N, bool ANY = false>
__device__ __forceinline__ void load_n(const void *p, int64_t i, float *v)
{
    using W4 = typename Pick<ANY, u32x4_any, u32x4>::T;
    using W2 = typename Pick<ANY, u32x2_any, u32x2>::T;
    using E = Elem<DT>;
    const char *a = (const char *)p + i * E::SIZE;
    constexpr int BYTES = N * E::SIZE;
    if constexpr (BYTES >= 16) {
#pragma unroll
        for (int k = 0; k < BYTES / 16; k++) E::unpack(((const W4 *)a)[k], v + k * E::PER16);
    } else if constexpr (N == 1) {
        v[0] = E::load(a, 0);
    } else {
        static_assert(BYTES == 8 && DT != DT_F32, "4 16-bit elements");
        const u32x2 w = *(const W2 *)a;
        const f32x2 t0 = unpack2<DT>(w[0]), t1 = unpack2<DT>(w[1]);
        v[0] = t0[0], v[1] = t0[1], v[2] = t1[0], v[3] = t1[1];
    }
}

template <int DT, int N, bool ANY = false>
__device__ __forceinline__ void store_n(void *p, int64_t i, const float *v)
{
    using W4 = typename Pick<ANY, u32x4_any, u32x4>::T;
    using W2 = typename Pick<ANY, u32x2_any, u32x2>::T;
    using E = Elem<DT>;
    char *a = (char *)p + i * E::SIZE;
    constexpr int BYTES = N * E::SIZE;
    if constexpr (BYTES >= 16) {
#pragma unroll
        for (int k = 0; k < BYTES / 16; k++) ((W4 *)a)[k] = E::pack(v + k * E::PER16);
    } else if constexpr (N == 1) {
        E::store(a, 0, v[0]);
    } else {
        static_assert(BYTES == 8 && DT != DT_F32, "4 16-bit elements");
        *(W2 *)a = u32x2{pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3])};
    }
}

// One element of a type known only at run time (row vectors that are read once).
__device__ __forceinline__ float load_any(int dt, const void *p, int64_t i)
{
    return dt == DT_F32 ? Elem<DT_F32>::load(p, i) : dt == DT_BF16 ? Elem<DT_BF16>::load(p, i) : Elem<DT_F16>::load(p, i);
}
__device__ __forceinline__ void store_any(int dt, void *p, int64_t i, float v)
{
    if (dt == DT_F32) Elem<DT_F32>::store(p, i, v);
    else if (dt == DT_BF16) Elem<DT_BF16>::store(p, i, v);
    else Elem<DT_F16>::store(p, i, v);
}

// Reductions over a wave without LDS: rotations inside the rows of 16 lanes (DPP), then the rows and
// the halves swapped.  Lanes only ever combine the same partial results in one order or its mirror,
// so every lane ends with the same bits, the same ones on every run.
template <int ROR>
__device__ __forceinline__ float rotate16(float v)
{
    const int i = __builtin_bit_cast(int, v);
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, 0x120 + ROR, 0xf, 0xf, false));
}
template <typename F>
__device__ __forceinline__ float wave_reduce(float v, F op)
{
    v = op(v, rotate16<8>(v));
    v = op(v, rotate16<4>(v));
    v = op(v, rotate16<2>(v));
    v = op(v, rotate16<1>(v));
    const uint32_t w = __builtin_bit_cast(uint32_t, v);
    const auto rows = __builtin_amdgcn_permlane16_swap(w, w, false, false);
    v = op(__uint_as_float(rows[0]), __uint_as_float(rows[1]));
    const uint32_t x = __builtin_bit_cast(uint32_t, v);
    const auto halves = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return op(__uint_as_float(halves[0]), __uint_as_float(halves[1]));
}
struct Add {
    __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
// NaN wins, so that a row holding one keeps it.
struct Max {
    __device__ __forceinline__ float operator()(float a, float b) const { return a > b || a != a ? a : b; }
};

// Over the WAVES waves of a workgroup through LDS; `buf` holds WAVES floats and is free again
// after the next barrier.  Every thread gets the result; waves are added in their order.
template <int WAVES, typename F>
__device__ __forceinline__ float group_reduce(float v, F op, float *buf)
{
    v = wave_reduce(v, op);
    if constexpr (WAVES == 1) return v;
    if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = buf[0];
#pragma unroll
    for (int w = 1; w < WAVES; w++) t = op(t, buf[w]);
    return t;
}

}  // namespace lm
