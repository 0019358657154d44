// vq_elem.h -- element types and small wave helpers of the beam, norm and gradient kernels (vq_beam.hip, vq_group_norm.hip, vq_grads.hip).
#pragma once

#include "vqhip_internal.h"

// Vectors of elements at the ELEMENT's alignment: gfx950 runs with unaligned access on (amdhsa), so a 16-byte load or store needs no
// 16-byte address.  Rows of odd lengths take the same instructions as aligned ones, and an element's lane does not depend on the address.
template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) VqVec { T v[N]; };
template <typename T, int N> __device__ __forceinline__ VqVec<T, N> vq_ldv(const T *p) { return *(const VqVec<T, N> *)p; }
template <typename T, int N> __device__ __forceinline__ void vq_stv(T *p, const VqVec<T, N> &v) { *(VqVec<T, N> *)p = v; }

// the same past the caches: results that this kernel and the next do not read
template <typename T, int N> __device__ __forceinline__ void vq_stv_nt(T *p, const VqVec<T, N> &v)
{
    if constexpr (sizeof(v) % 4 == 0) {
        typedef unsigned U __attribute__((ext_vector_type(sizeof(v) / 4), aligned(sizeof(T))));
        U u;
        __builtin_memcpy(&u, &v, sizeof(v));
        __builtin_nontemporal_store(u, (U *)p);
    } else
        vq_stv<T, N>(p, v);
}

static inline int vq_elem_bytes(int64_t dtype) { return dtype == VQHIP_F32 ? 4 : (dtype == VQHIP_BF16 || dtype == VQHIP_F16) ? 2 : 0; }

template <typename T> __device__ __forceinline__ T vq_wave_sum(T v)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
