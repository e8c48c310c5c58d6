// typed.h -- tensors of float, bfloat16 and half elements in kernels that
// compute in float.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/dressi_hip.h"

namespace dressi {

using bf16 = __bf16;
using f16 = _Float16;

template <typename T>
__device__ __forceinline__ float to_float(T x) {
    return (float)x;
}
// Rounded to nearest, ties to even.
template <typename T>
__device__ __forceinline__ T from_float(float x) {
    return (T)x;
}

template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
    T v[V];
};

// V neighbours in one load or store; `p` aligned to all of them.
template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float* x) {
    const Pack<T, V> a = *(const Pack<T, V>*)p;
#pragma unroll
    for (int i = 0; i < V; i++) {
        x[i] = to_float(a.v[i]);
    }
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float* x) {
    Pack<T, V> a;
#pragma unroll
    for (int i = 0; i < V; i++) {
        a.v[i] = from_float<T>(x[i]);
    }
    *(Pack<T, V>*)p = a;
}

inline size_t type_bytes(uint32_t type) { return type == DRESSI_F32 ? 4 : 2; }

}  // namespace dressi
