// Runs of neighbouring channels as a thread of the sequence kernels holds them:
// read and written in as few accesses as the run takes, at any element's address.
#pragma once
#include <hip/hip_runtime.h>

#include "device/ormi_device.h"
#include "ormi_hip.h"

namespace ormi_hip {

template <int DT> struct ElemOf { using type = unsigned short; };
template <> struct ElemOf<ORMI_DTYPE_F32> { using type = float; };

template <int DT>
__device__ __forceinline__ float elem_to_f32(typename ElemOf<DT>::type v) {
    if constexpr (DT == ORMI_DTYPE_F32) return v;
    else return DT == ORMI_DTYPE_BF16 ? ormi_bf16_to_f32(v) : ormi_f16_to_f32(v);
}
template <int DT>
__device__ __forceinline__ typename ElemOf<DT>::type elem_from_f32(float v) {
    if constexpr (DT == ORMI_DTYPE_F32) return v;
    else return DT == ORMI_DTYPE_BF16 ? ormi_f32_to_bf16(v) : ormi_f32_to_f16(v);
}

// V elements as they are in memory.
template <int DT, int V>
struct Run {
    using T = typename ElemOf<DT>::type;
    static constexpr int kGroup = 16 / sizeof(T) < V ? 16 / sizeof(T) : V;
    typedef T Vec __attribute__((ext_vector_type(kGroup), aligned(sizeof(T))));
    Vec v[V / kGroup];

    __device__ __forceinline__ float get(int e) const { return elem_to_f32<DT>(v[e / kGroup][e % kGroup]); }
    __device__ __forceinline__ void set(int e, float x) { v[e / kGroup][e % kGroup] = elem_from_f32<DT>(x); }
    __device__ __forceinline__ void fill(float x) {
#pragma unroll
        for (int e = 0; e < V; ++e) set(e, x);
    }
    // Keeps the compiler from holding the elements in fp32 between uses before this
    // and uses after it: for runs that wait long in registers.
    __device__ __forceinline__ void stay_packed() {
        if constexpr (DT == ORMI_DTYPE_F32) return;
        constexpr int kWords = V * sizeof(T) / 4;
        unsigned w[kWords];
        __builtin_memcpy(w, v, sizeof w);
#pragma unroll
        for (int i = 0; i < kWords; ++i) asm volatile("" : "+v"(w[i]));
        __builtin_memcpy(v, w, sizeof w);
    }
    // All V, without a branch.
    __device__ __forceinline__ void load(const void* at) {
#pragma unroll
        for (int i = 0; i < V / kGroup; ++i) v[i] = ((const Vec*)at)[i];
    }
    // The same, past the caches: for results that are not read here again (8 x 2048 x 4096
    // bf16, recurrence and gradient: 2%).
    __device__ __forceinline__ void store_past(void* at) const {
#pragma unroll
        for (int i = 0; i < V / kGroup; ++i) __builtin_nontemporal_store(v[i], (Vec*)at + i);
    }
    // n of the V elements exist; the others become 0.
    __device__ __forceinline__ void load(const void* at, int n) {
        if (n == V) {
#pragma unroll
            for (int i = 0; i < V / kGroup; ++i)
                v[i] = ((const Vec*)at)[i];
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) v[e / kGroup][e % kGroup] = e < n ? ((const T*)at)[e] : T(0);
        }
    }
    __device__ __forceinline__ void store(void* at, int n) const {
        if (n == V) {
#pragma unroll
            for (int i = 0; i < V / kGroup; ++i) ((Vec*)at)[i] = v[i];
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (e < n) ((T*)at)[e] = v[e / kGroup][e % kGroup];
        }
    }
};

}  // namespace ormi_hip
