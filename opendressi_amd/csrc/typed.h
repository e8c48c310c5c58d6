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

// V neighbours in one load, as they lie in memory: held so, 16 bytes take four
// registers where floats take eight. `p` aligned to all of them.
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
    return *(const Pack<T, V>*)p;
}
template <typename T, int V>
__device__ __forceinline__ void unpack(const Pack<T, V>& a, float (&x)[V]) {
#pragma unroll
    for (int i = 0; i < V; i++) {
        x[i] = to_float(a.v[i]);
    }
}

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

// The same for what is not read again soon: it goes past the caches.
template <typename T, int V>
__device__ __forceinline__ void stream_vec(T* p, const float* x) {
    Pack<T, V> a;
#pragma unroll
    for (int i = 0; i < V; i++) {
        a.v[i] = from_float<T>(x[i]);
    }
    using Word = std::conditional_t<sizeof(a) % 4 == 0, uint32_t, uint16_t>;
    constexpr int kWords = sizeof(a) / sizeof(Word);
    typedef Word Words __attribute__((ext_vector_type(kWords)));
    Words w;
    __builtin_memcpy(&w, &a, sizeof(a));
    __builtin_nontemporal_store(w, (Words*)p);
}

inline size_t type_bytes(uint32_t type) { return type == DRESSI_F32 ? 4 : 2; }

}  // namespace dressi
