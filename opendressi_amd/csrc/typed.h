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

// The widest words that make up N bytes.
template <size_t N>
using Words = std::conditional_t<N % 4 == 0, uint32_t, std::conditional_t<N % 2 == 0, uint16_t, uint8_t>>
    __attribute__((ext_vector_type(N % 4 == 0 ? N / 4 : N % 2 == 0 ? N / 2 : N)));

// Memory that is not used again soon (`STREAM`) goes past the caches, so that it
// does not drive out what is.
template <bool STREAM, typename P>
__device__ __forceinline__ P load_as(const P* p) {
    if constexpr (STREAM) {
        const Words<sizeof(P)> w = __builtin_nontemporal_load((const Words<sizeof(P)>*)p);
        P a;
        __builtin_memcpy(&a, &w, sizeof(P));
        return a;
    } else {
        return *p;
    }
}
template <bool STREAM, typename P>
__device__ __forceinline__ void store_as(P* p, const P& a) {
    if constexpr (STREAM) {
        Words<sizeof(P)> w;
        __builtin_memcpy(&w, &a, sizeof(P));
        __builtin_nontemporal_store(w, (Words<sizeof(P)>*)p);
    } else {
        *p = a;
    }
}

// V neighbours in one load, as they lie in memory: held so, 16 bytes take four
// registers where floats take eight. `p` aligned to all of them.
template <typename T, int V, bool STREAM = false>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
    return load_as<STREAM>((const Pack<T, V>*)p);
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
    const Pack<T, V> a = load_pack<T, V>(p);
#pragma unroll
    for (int i = 0; i < V; i++) {
        x[i] = to_float(a.v[i]);
    }
}
template <typename T, int V, bool STREAM = false>
__device__ __forceinline__ void store_vec(T* p, const float* x) {
    Pack<T, V> a;
#pragma unroll
    for (int i = 0; i < V; i++) {
        a.v[i] = from_float<T>(x[i]);
    }
    store_as<STREAM>((Pack<T, V>*)p, a);
}

inline size_t type_bytes(uint32_t type) { return type == DRESSI_F32 ? 4 : 2; }

}  // namespace dressi
