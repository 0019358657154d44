// vq_elem.h -- element types and small wave helpers of the beam, norm and gradient kernels (vq_beam.hip, vq_group_norm.hip, vq_grads.hip).
#pragma once

#include "vqhip_internal.h"

#include <math.h>

// Vectors of elements at the ELEMENT's alignment: gfx950 runs with unaligned access on (amdhsa), so a 16-byte load or store needs no
// 16-byte address.  Rows of odd lengths take the same instructions as aligned ones, and an element's lane does not depend on the address.
template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) VqVec { T v[N]; };
template <typename T, int N> __device__ __forceinline__ VqVec<T, N> vq_ldv(const T *p) { return *(const VqVec<T, N> *)p; }
template <typename T, int N> __device__ __forceinline__ void vq_stv(T *p, const VqVec<T, N> &v) { *(VqVec<T, N> *)p = v; }

static inline int vq_elem_bytes(int64_t dtype) { return dtype == VQHIP_F32 ? 4 : (dtype == VQHIP_BF16 || dtype == VQHIP_F16) ? 2 : 0; }

// Reductions over the 64 lanes of a full wave by DPP: each row of 16 to its last lane, then rows 0 -> 1, 2 -> 3, then 1 -> 3; lane 63 holds
// the result and is read into a scalar.  (__shfl_xor goes through LDS: six round trips.)  All 64 lanes must be active.
template <int CTRL, int ROWS, typename T> __device__ __forceinline__ T vq_dpp(T v, T none)
{
    static_assert(sizeof(T) == 4 || sizeof(T) == 8, "");
    if constexpr (sizeof(T) == 4)
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
    else {
        const long long o = __builtin_bit_cast(long long, none), s = __builtin_bit_cast(long long, v);
        const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp((int)o, (int)s, CTRL, ROWS, 0xf, false);
        const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp((int)(o >> 32), (int)(s >> 32), CTRL, ROWS, 0xf, false);
        return __builtin_bit_cast(T, (long long)(((unsigned long long)hi << 32) | lo));
    }
}
template <typename T> __device__ __forceinline__ T vq_lane63(T v)
{
    if constexpr (sizeof(T) == 4)
        return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
    else {
        const long long s = __builtin_bit_cast(long long, v);
        const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)s, 63), hi = (unsigned)__builtin_amdgcn_readlane((int)(s >> 32), 63);
        return __builtin_bit_cast(T, (long long)(((unsigned long long)hi << 32) | lo));
    }
}
template <typename T, typename F> __device__ __forceinline__ T vq_wave_reduce(T v, T none, F &&f)
{
    v = f(v, vq_dpp<0x111, 0xf>(v, none));                    // row_shr 1, 2, 4, 8
    v = f(v, vq_dpp<0x112, 0xf>(v, none));
    v = f(v, vq_dpp<0x114, 0xf>(v, none));
    v = f(v, vq_dpp<0x118, 0xf>(v, none));
    v = f(v, vq_dpp<0x142, 0xa>(v, none));                    // row_bcast 15 into rows 1 and 3, row_bcast 31 into rows 2 and 3
    v = f(v, vq_dpp<0x143, 0xc>(v, none));
    return vq_lane63(v);
}
template <typename T> __device__ __forceinline__ T vq_wave_sum(T v) { return vq_wave_reduce(v, (T)0, [](T a, T b) { return a + b; }); }
__device__ __forceinline__ float vq_wave_max(float v) { return vq_wave_reduce(v, -INFINITY, [](float a, float b) { return fmaxf(a, b); }); }
