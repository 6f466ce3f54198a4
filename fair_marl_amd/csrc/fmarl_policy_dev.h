// What the policy operators' kernels share (gfx950): element types, four-element loads and stores, MFMA vector types.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/fmarl.h"

namespace fmarl {
namespace policy {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <typename T> struct Vec4;
template <> struct Vec4<float> { typedef f32x4 type; };
template <> struct Vec4<__bf16> { typedef bf16x4 type; };
template <> struct Vec4<_Float16> { typedef f16x4 type; };

// four elements that start anywhere: the memory takes one access of any alignment for them
template <typename T> struct Loose4 { typedef typename Vec4<T>::type type __attribute__((aligned(sizeof(T)))); };

// four consecutive elements at p, zero beyond `left`: one load; where `vec`, p is a multiple of four elements and left one of four, else the row's last ones come one by one
template <typename T>
__device__ __forceinline__ typename Vec4<T>::type load4(const T *p, int left, bool vec) {
    typedef typename Vec4<T>::type V;
    V v = {(T)0.f, (T)0.f, (T)0.f, (T)0.f};
    if (vec) {
        if (left > 0) v = *(const V *)p;
    } else if (left >= 4) {
        v = *(const typename Loose4<T>::type *)p;
    } else {
#pragma unroll
        for (int r = 0; r < 3; ++r) if (r < left) v[r] = p[r];
    }
    return v;
}

template <typename T>
__device__ __forceinline__ void store4(T *p, f32x4 a, int left, bool vec) {
    typedef typename Vec4<T>::type V;
    const V v = {(T)a[0], (T)a[1], (T)a[2], (T)a[3]};   // round to nearest even, once, at the end
    if (vec) {
        if (left > 0) *(V *)p = v;
    } else if (left >= 4) {
        *(typename Loose4<T>::type *)p = v;
    } else {
#pragma unroll
        for (int r = 0; r < 3; ++r) if (r < left) p[r] = v[r];
    }
}

template <typename V> __device__ __forceinline__ f32x4 widen(V v) { return f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]}; }

// LDS of one wave: its writes before this are seen by its reads behind it (the LDS answers a wave in order; this holds the compiler)
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }   // v_exp_f32: 1 ulp, 0 below 2^-126

// v of another lane of the row of 16: a DPP control (0x120 + n: the row turned by n)
template <int CTRL> __device__ __forceinline__ float row_turn(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}

// op over the lanes of a wave whose numbers differ in the bits from FROM (1, 16 or 32) up to below `to`, in all of them: within a row of 16 by DPP (a quad's neighbour, its other pair, a
// half row mirrored -- whose quads hold one value each by then --, the row mirrored), beyond by the swaps of rows and halves.  No LDS pipe: a step is
// a few cycles where ds_bpermute's is over fifty, and a row's norms are chains of such steps.
template <int FROM, typename F> __device__ __forceinline__ float lanes_fold(float v, int to, F op) {
    if (FROM <= 1) {
        if (to > 1) v = op(v, row_turn<0xb1>(v));
        if (to > 2) v = op(v, row_turn<0x4e>(v));
        if (to > 4) v = op(v, row_turn<0x141>(v));
        if (to > 8) v = op(v, row_turn<0x140>(v));
    }
    if (FROM <= 16 && to > 16) {
        const auto p = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
        v = op(__builtin_bit_cast(float, (uint32_t)p[0]), __builtin_bit_cast(float, (uint32_t)p[1]));
    }
    if (to > 32) {
        const auto p = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
        v = op(__builtin_bit_cast(float, (uint32_t)p[0]), __builtin_bit_cast(float, (uint32_t)p[1]));
    }
    return v;
}
template <int FROM> __device__ __forceinline__ float lanes_sum(float v, int to) { return lanes_fold<FROM>(v, to, [](float a, float b) { return a + b; }); }
template <int FROM> __device__ __forceinline__ float lanes_max(float v, int to) { return lanes_fold<FROM>(v, to, [](float a, float b) { return fmaxf(a, b); }); }

}  // namespace policy

int policy_fail(int code, const char *fmt, const char *a = "");   // libfmarl.hip: the text of fmarl_last_error()

}  // namespace fmarl

#define HIP_OK(call)                                                                                        \
    do {                                                                                                    \
        hipError_t e_ = (call);                                                                             \
        if (e_ != hipSuccess) return fmarl::policy_fail(FMARL_EHIP, #call ": %s", hipGetErrorString(e_));   \
    } while (0)

namespace {
inline int elem_bytes(int dtype) { return dtype == FMARL_T_F32 ? 4 : 2; }
inline size_t up256(size_t n) { return (n + 255) / 256 * 256; }
}  // namespace
