// norm_core.h -- what the normalisation layers share: activations and their
// slopes, and the affine step's weight and bias in any of the three types.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "typed.h"

namespace dressi {

__device__ __forceinline__ float sigmoid(float z) {
    return __builtin_amdgcn_rcpf(1.f + __expf(-z));  // an ulp of each
}
// The normal distribution's Phi(z) and e = exp(-z^2 / 2), its tail beyond |z| being
// e times a smooth function of |z|, for 16-bit images Abramowitz and Stegun's
// 7.1.26: erf to 1.5e-7, a rounding of a float near 1 (group norm of 2 x 512 x 512 x
// 88 float16, backward: 116 us, 153 with a library erf beside the exponential).
template <typename T>
__device__ __forceinline__ void gauss(float z, float& cdf, float& e) {
    e = __expf(-0.5f * z * z);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f * 0.70710678f, fabsf(z), 1.f));
    float q = fmaf(1.061405429f, t, -1.453152027f);
    q = fmaf(q, t, 1.421413741f);
    q = fmaf(q, t, -0.284496736f);
    q = fmaf(q, t, 0.254829592f);
    q *= 0.5f * t * e;
    cdf = z < 0.f ? q : 1.f - q;
}
// For float images 1/2 + s P(s), s = a / (1 + a), a = 0.26 |z|: P fitted to the least
// relative error over |z| < 14 (7e-9; past it e is zero), its coefficients rounded
// one after the other. Near z = 0, where a function of t = 1 / (1 + a) takes every
// rounding of t, little is added to the 1/2. The error of z Phi(z) over normal z is
// 2.2e-8 (7.1.26: 5.6e-8; 0.5 (1 + erf) in floats: 2.5e-8), of its slope 2.6e-8
// (6.6e-8, 2.7e-8). Group norm of 2 x 512 x 512 x 88 takes 109 and 183 us with it, 104 and 181
// with 7.1.26; with it float16 images would take 78 and 130, not 70 and 118.
template <>
__device__ __forceinline__ void gauss<float>(float z, float& cdf, float& e) {
    e = __expf(-0.5f * z * z);
    const float a = 0.26f * fminf(fabsf(z), 14.f);
    const float s = a * __builtin_amdgcn_rcpf(1.f + a);
    float q = fmaf(-0.0338316262f, s, 0.134448603f);
    q = fmaf(q, s, -0.147560731f);
    q = fmaf(q, s, -0.0892333016f);
    q = fmaf(q, s, 0.168799251f);
    q = fmaf(q, s, 0.542275906f);
    q = fmaf(q, s, -1.70436502f);
    q = fmaf(q, s, 2.16385388f);
    q = fmaf(q, s, -1.53439391f);
    q = fmaf(q, s, 0.5f);
    cdf = z < 0.f ? q * e : fmaf(-q, e, 1.f);
}

template <typename T, int V>
__device__ __forceinline__ void act_values(uint32_t act, float (&z)[V]) {
    switch (act) {
        case DRESSI_ACT_RELU:
#pragma unroll
            for (int j = 0; j < V; j++) {
                z[j] = z[j] < 0.f ? 0.f : z[j];
            }
            break;
        case DRESSI_ACT_SILU:
#pragma unroll
            for (int j = 0; j < V; j++) {
                z[j] *= sigmoid(z[j]);
            }
            break;
        case DRESSI_ACT_GELU:
#pragma unroll
            for (int j = 0; j < V; j++) {
                float cdf, e;
                gauss<T>(z[j], cdf, e);
                z[j] *= cdf;
            }
            break;
        default:
            break;
    }
}

// g times the activation's slope at z
template <typename T, int V>
__device__ __forceinline__ void act_slopes(uint32_t act, const float (&z)[V], float (&g)[V]) {
    switch (act) {
        case DRESSI_ACT_RELU:
#pragma unroll
            for (int j = 0; j < V; j++) {
                g[j] = z[j] > 0.f ? g[j] : 0.f;  // an infinity or a NaN is masked too
            }
            break;
        case DRESSI_ACT_SILU:
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float e = sigmoid(z[j]);
                g[j] *= e * fmaf(z[j], 1.f - e, 1.f);
            }
            break;
        case DRESSI_ACT_GELU:
#pragma unroll
            for (int j = 0; j < V; j++) {
                float cdf, e;
                gauss<T>(z[j], cdf, e);
                g[j] *= fmaf(z[j] * 0.39894228f, e, cdf);
            }
            break;
        default:
            break;
    }
}

__device__ __forceinline__ void store_one(void* p, uint32_t type, size_t i, float x) {
    if (type == DRESSI_F32) {
        ((float*)p)[i] = x;
    } else if (type == DRESSI_BF16) {
        ((bf16*)p)[i] = from_float<bf16>(x);
    } else {
        ((f16*)p)[i] = from_float<f16>(x);
    }
}

struct Affine {
    const void* weight;  // null: 1
    const void* bias;    // null: 0
    uint32_t type;
};

// One branch for all V, so that their loads are on their way together.
template <int V>
__device__ __forceinline__ void load_channels(const void* p, uint32_t type, uint32_t ch,
                                              float absent, float (&w)[V]) {
    if (!p) {
#pragma unroll
        for (int j = 0; j < V; j++) {
            w[j] = absent;
        }
    } else if (type == DRESSI_F32) {
#pragma unroll
        for (int j = 0; j < V; j++) {
            w[j] = ((const float*)p)[ch + j];
        }
    } else if (type == DRESSI_BF16) {
#pragma unroll
        for (int j = 0; j < V; j++) {
            w[j] = to_float(((const bf16*)p)[ch + j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; j++) {
            w[j] = to_float(((const f16*)p)[ch + j]);
        }
    }
}
template <int V>
__device__ __forceinline__ void load_affine(const Affine& a, uint32_t ch, float (&w)[V],
                                            float (&b)[V]) {
    load_channels<V>(a.weight, a.type, ch, 1.f, w);
    load_channels<V>(a.bias, a.type, ch, 0.f, b);
}

}  // namespace dressi
