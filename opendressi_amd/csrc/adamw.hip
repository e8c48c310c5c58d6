// adamw.hip -- one AdamW step over many parameter tensors at once
// (dressi_adamw_step), with moments in 32 or in 8 bits.
//
// Per element, every operation rounded to float once and in this order, so
// that the result does not depend on how the work is cut:
//
//   g' = g c                     c = min(1, max_norm / (|g|_2 + 1e-6))
//   m' = m b1 + g' (1 - b1)
//   v' = v b2 + (g' g') (1 - b2)
//   p' = p (1 - lr wd) - (m' / (sqrt(v') / sqrt(1 - b2^t) + eps)) (lr / (1 - b1^t))
//
// Moments in 8 bits. 32 neighbours share the largest exponent field E of
// their magnitudes (8 bits). With up = max(E, T) - T the scaled magnitude
// f = |x| 2^-up has exponent fields of at most T, and its code is
// (bits(f) + r) >> 20: a float of three mantissa bits with gradual underflow,
// because the code's subnormals are float's own. T is 14 for the first moment
// (4 exponent bits and a sign) and 30 for the second (5 exponent bits): one
// field is left for a rounding that carries. r is uniform in [0, 2^20), a hash
// of (element, step): the rounding is right on average, without which a second
// moment that moves by 0.1 % a step would stay where it is, half a step of the
// code being 3 to 6 %. A second moment above zero never becomes zero: the
// update would divide by eps. E = 255 (an infinity or a NaN among the 32)
// makes all 32 NaN. The update itself uses m' and v' as computed, before they
// are rounded.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "internal.h"
#include "typed.h"

namespace dressi {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kLaneElems = 4;  // neighbours of a lane: 16 bytes of float
constexpr uint32_t kBlock = 32;     // elements that share an exponent
constexpr int kTop1 = 14, kTop2 = 30;
constexpr uint32_t kMaxTensors = 64, kMaxSets = 16;
constexpr uint32_t kMaxPartials = 1024;

struct TensorArg {
    void* param;
    const void* grad;
    float* master;         // of 16-bit parameters, or null
    uint64_t n;
    uint64_t state;        // element offset in the flat state buffers
    uint32_t first_chunk;  // of this launch
    uint16_t type, set;
};
struct SetArg {
    float b1, omb1, b2, omb2, eps, decay, step_size, inv_bc2;
    uint32_t key;
};
// A launch's tensors: in the kernel arguments, so that no copy to the device
// and no wait stands between a step's gradients and its kernel. 4 KB at most.
struct Table {
    TensorArg t[kMaxTensors];
    SetArg set[kMaxSets];
    uint32_t n_tensors, n_chunks;
};
static_assert(sizeof(Table) <= 3800, "with the pointers beside it within 4 KB of arguments");

struct State {
    const SetArg* sets;  // on the device, or null: the table's
    void* m;
    void* v;
    uint8_t* m_scale;
    uint8_t* v_scale;
    const double* partials;  // of the squared norm; null: no clipping
    uint32_t n_partials;
    float max_norm;
    float* norm;
};

// The tensor that holds `chunk`: the last whose first chunk is not past it.
// A lane per tensor, one load deep.
__device__ __forceinline__ uint32_t find_tensor(const Table& tb, uint32_t chunk) {
    static_assert(kMaxTensors == 64, "a tensor a lane");
    const uint32_t lane = threadIdx.x & 63u;
    const bool at = lane < tb.n_tensors && tb.t[lane].first_chunk <= chunk;
    return __builtin_amdgcn_readfirstlane((uint32_t)__popcll(__ballot(at)) - 1);
}

// ---------------------------------------------------------------------------
// the squared norm of all gradients
// ---------------------------------------------------------------------------

// The workgroup's sum of `s`, valid in thread 0.
__device__ __forceinline__ double block_sum(double s) {
    __shared__ double part[kThreads / 64];
    for (int o = 32; o > 0; o >>= 1) {
        s += __shfl_xor(s, o);
    }
    if ((threadIdx.x & 63u) == 0) {
        part[threadIdx.x >> 6] = s;
    }
    __syncthreads();
    s = part[0];
    for (uint32_t i = 1; i < kThreads / 64; i++) {
        s += part[i];
    }
    return s;
}

template <typename T, int ITER>
__device__ __forceinline__ double chunk_squares(const TensorArg& t, uint64_t at) {
    const T* g = (const T*)t.grad;
    double s = 0.0;
    constexpr uint32_t kStep = kThreads * kLaneElems;
    const bool vec = ((uintptr_t)g & (kLaneElems * sizeof(T) - 1)) == 0;
    if (vec && at + (uint64_t)ITER * kStep <= t.n) {
        float x[ITER][kLaneElems];
#pragma unroll
        for (int k = 0; k < ITER; k++) {
            load_vec<T, kLaneElems>(g + at + (uint64_t)k * kStep + threadIdx.x * kLaneElems, x[k]);
        }
#pragma unroll
        for (int k = 0; k < ITER; k++) {
#pragma unroll
            for (uint32_t j = 0; j < kLaneElems; j++) {
                s = fma((double)x[k][j], (double)x[k][j], s);
            }
        }
    } else {
        const uint64_t end = std::min<uint64_t>(t.n, at + (uint64_t)ITER * kStep);
        for (uint64_t i = at + threadIdx.x; i < end; i += kThreads) {
            const double x = (double)to_float(g[i]);
            s = fma(x, x, s);
        }
    }
    return s;
}

// A workgroup's share of sum g^2, in double: a float's square may not be one.
// One read of the gradients.
template <int ITER>
__global__ __launch_bounds__(256) void k_adamw_squares(const Table tb, double* partials) {
    double s = 0.0;
    for (uint32_t c = blockIdx.x; c < tb.n_chunks; c += gridDim.x) {
        const TensorArg& t = tb.t[find_tensor(tb, c)];
        const uint64_t at = (uint64_t)(c - t.first_chunk) * (ITER * kThreads * kLaneElems);
        switch (t.type) {
            case DRESSI_F32:
                s += chunk_squares<float, ITER>(t, at);
                break;
            case DRESSI_BF16:
                s += chunk_squares<bf16, ITER>(t, at);
                break;
            default:
                s += chunk_squares<f16, ITER>(t, at);
        }
    }
    s = block_sum(s);
    if (threadIdx.x == 0) {
        partials[blockIdx.x] = s;
    }
}

// ---------------------------------------------------------------------------
// 8-bit moments
// ---------------------------------------------------------------------------

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The largest of the 8 lanes that hold a block.
__device__ __forceinline__ uint32_t block_max(uint32_t x) {
    x = std::max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xb1, 0xf, 0xf, true));   // lane ^ 1
    x = std::max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4e, 0xf, 0xf, true));   // lane ^ 2
    x = std::max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x141, 0xf, 0xf, true));  // 7 - lane
    return x;
}

__device__ __forceinline__ int scale_shift(uint32_t field, int top) {
    return std::max((int)field, top) - top;
}

__device__ __forceinline__ float decode(uint32_t code, uint32_t field, int top) {
    const float f = __builtin_ldexpf(__uint_as_float(code << 20), scale_shift(field, top));
    return field == 255u ? __uint_as_float(0x7fc00000u) : f;
}

__device__ __forceinline__ uint32_t encode(float x, int up, uint32_t r) {
    return (__float_as_uint(__builtin_ldexpf(__uint_as_float(abs_bits(x)), -up)) + r) >> 20;
}

// 32 bits of element i at a step. Folds of 16, 15 and 16 bits around products with
// 0x7feb352d and 0x846ca68b are the 32-bit hash that C. Wellons found and published
// (2018, by a search for the least bias); the factor of the high word is the first
// of A. Appleby's published 32-bit finalizer (2008).
__device__ __forceinline__ uint32_t noise(uint64_t i, uint32_t key) {
    uint32_t x = (uint32_t)i ^ key ^ ((uint32_t)(i >> 32) * 0x85ebca6bu);
    x = (x ^ (x >> 16)) * 0x7feb352du;
    x = (x ^ (x >> 15)) * 0x846ca68bu;
    return x ^ (x >> 16);
}

struct Moments {
    float m[kLaneElems], v[kLaneElems];
};

// A lane's moments as they lie in memory.
template <bool Q8>
struct RawMoments {
    Pack<float, kLaneElems> m, v;
    template <bool STREAM>
    __device__ __forceinline__ void load(const State& st, uint64_t i) {
        m = load_pack<float, kLaneElems, STREAM>((const float*)st.m + i);
        v = load_pack<float, kLaneElems, STREAM>((const float*)st.v + i);
    }
    __device__ __forceinline__ void clear() { m = v = {}; }
    __device__ __forceinline__ Moments values() const {
        Moments o;
        unpack(m, o.m);
        unpack(v, o.v);
        return o;
    }
};
template <>
struct RawMoments<true> {
    uint32_t m, v;  // four codes each
    uint8_t m_scale, v_scale;
    template <bool STREAM>
    __device__ __forceinline__ void load(const State& st, uint64_t i) {
        m = load_as<STREAM>((const uint32_t*)((const uint8_t*)st.m + i));
        v = load_as<STREAM>((const uint32_t*)((const uint8_t*)st.v + i));
        m_scale = st.m_scale[i / kBlock];
        v_scale = st.v_scale[i / kBlock];
    }
    __device__ __forceinline__ void clear() { m = v = m_scale = v_scale = 0; }
    __device__ __forceinline__ Moments values() const {
        Moments o;
#pragma unroll
        for (uint32_t j = 0; j < kLaneElems; j++) {
            const uint32_t c = (m >> (8 * j)) & 255u;
            o.m[j] = __uint_as_float(__float_as_uint(decode(c & 127u, m_scale, kTop1)) |
                                     ((c & 128u) << 24));
            o.v[j] = decode((v >> (8 * j)) & 255u, v_scale, kTop2);
        }
        return o;
    }
};

// All 64 lanes call this together (the block's maximum crosses lanes); `live`
// says which hold elements.
template <bool Q8, bool STREAM>
__device__ __forceinline__ void store_moments(const State& st, uint64_t i, const Moments& o,
                                              uint32_t key, bool live) {
    if constexpr (Q8) {
        uint32_t am = 0, av = 0;
#pragma unroll
        for (uint32_t j = 0; j < kLaneElems; j++) {
            am = std::max(am, abs_bits(o.m[j]));
            av = std::max(av, abs_bits(o.v[j]));
        }
        const uint32_t fm = block_max(am) >> 23, fv = block_max(av) >> 23;
        const int um = scale_shift(fm, kTop1), uv = scale_shift(fv, kTop2);
        uint32_t cm = 0, cv = 0;
#pragma unroll
        for (uint32_t j = 0; j < kLaneElems; j++) {
            const uint32_t r = noise(i + j, key);
            uint32_t a = encode(o.m[j], um, ((r & 0xffffu) << 4) + 8u);
            uint32_t b = encode(o.v[j], uv, ((r >> 16) << 4) + 8u);
            b = o.v[j] > 0.f ? std::max(b, 1u) : b;
            a = fm == 255u ? 0u : a;
            b = fv == 255u ? 0u : b;
            cm |= (a | ((__float_as_uint(o.m[j]) >> 24) & 128u)) << (8 * j);
            cv |= b << (8 * j);
        }
        if (live) {
            store_as<STREAM>((uint32_t*)((uint8_t*)st.m + i), cm);
            store_as<STREAM>((uint32_t*)((uint8_t*)st.v + i), cv);
            if ((threadIdx.x & 7u) == 0) {
                st.m_scale[i / kBlock] = (uint8_t)fm;
                st.v_scale[i / kBlock] = (uint8_t)fv;
            }
        }
    } else if (live) {
        store_vec<float, kLaneElems, STREAM>((float*)st.m + i, o.m);
        store_vec<float, kLaneElems, STREAM>((float*)st.v + i, o.v);
    }
}

// ---------------------------------------------------------------------------
// the step
// ---------------------------------------------------------------------------

__device__ __forceinline__ void update(const SetArg& h, float coef, bool clip, const float* g,
                                       float* p, Moments& o) {
#pragma unroll
    for (uint32_t j = 0; j < kLaneElems; j++) {
        const float x = clip ? g[j] * coef : g[j];
        o.m[j] = o.m[j] * h.b1 + x * h.omb1;
        o.v[j] = o.v[j] * h.b2 + (x * x) * h.omb2;
        const float den = sqrtf(o.v[j]) * h.inv_bc2 + h.eps;
        p[j] = p[j] * h.decay - (o.m[j] / den) * h.step_size;
    }
}

// A parameter's value: its master's, unless it is no longer the master's
// rounding. Then someone else has written it since the last step (a clamp, a
// checkpoint) and it counts.
template <typename T>
__device__ __forceinline__ float newest(float param, float master) {
    return to_float(from_float<T>(master)) == param ? master : param;
}

// A chunk of one tensor. FULL: all of its elements are there and aligned for
// a lane's vector loads, which are all issued before the first is used. STREAM:
// a FULL chunk's go past the caches.
template <typename T, bool Q8, int ITER, bool FULL, bool STREAM>
__device__ __forceinline__ void step_chunk(const TensorArg& t, const SetArg& h, const State& st,
                                           uint64_t at, float coef, bool clip) {
    constexpr uint32_t kStep = kThreads * kLaneElems;
    T* p = (T*)t.param;
    const T* g = (const T*)t.grad;
    const bool wide = !std::is_same<T, float>::value && t.master != nullptr;
    const uint64_t padded = (t.n + kBlock - 1) / kBlock * kBlock;
    Pack<T, kLaneElems> gv[ITER], pv[ITER];
    Pack<float, kLaneElems> mv[ITER];
    RawMoments<Q8> raw[ITER];
#pragma unroll
    for (int k = 0; k < ITER; k++) {
        const uint64_t i = at + (uint64_t)k * kStep + threadIdx.x * kLaneElems;
        if (FULL) {
            gv[k] = load_pack<T, kLaneElems, STREAM>(g + i);
            pv[k] = load_pack<T, kLaneElems, STREAM>(p + i);
            if (wide) {
                mv[k] = load_pack<float, kLaneElems, STREAM>(t.master + i);
            }
            raw[k].template load<STREAM>(st, t.state + i);
        } else {
#pragma unroll
            for (uint32_t j = 0; j < kLaneElems; j++) {
                const bool in = i + j < t.n;
                gv[k].v[j] = in ? g[i + j] : (T)0.f;
                pv[k].v[j] = in ? p[i + j] : (T)0.f;
                mv[k].v[j] = in && wide ? t.master[i + j] : 0.f;
            }
            raw[k].clear();
            if (i < padded) {  // a share is padded with zeros to whole blocks
                raw[k].template load<false>(st, t.state + i);
            }
        }
    }
#pragma unroll
    for (int k = 0; k < ITER; k++) {
        const uint64_t i = at + (uint64_t)k * kStep + threadIdx.x * kLaneElems;
        float gx[kLaneElems], px[kLaneElems];
        unpack(gv[k], gx);
        unpack(pv[k], px);
#pragma unroll
        for (uint32_t j = 0; wide && j < kLaneElems; j++) {
            px[j] = newest<T>(px[j], mv[k].v[j]);
        }
        Moments o = raw[k].values();
        update(h, coef, clip, gx, px, o);
        if (!FULL) {
#pragma unroll
            for (uint32_t j = 0; j < kLaneElems; j++) {
                if (i + j >= t.n) {
                    o.m[j] = o.v[j] = 0.f;  // the padding stays zero
                }
            }
        }
        store_moments<Q8, STREAM>(st, t.state + i, o, h.key, FULL || i < padded);
        if (FULL) {
            store_vec<T, kLaneElems, STREAM>(p + i, px);
            if (wide) {
                store_vec<float, kLaneElems, STREAM>(t.master + i, px);
            }
        } else {
#pragma unroll
            for (uint32_t j = 0; j < kLaneElems; j++) {
                if (i + j < t.n) {
                    p[i + j] = from_float<T>(px[j]);
                    if (wide) {
                        t.master[i + j] = px[j];
                    }
                }
            }
        }
    }
}

template <typename T, bool Q8, int ITER, bool STREAM>
__device__ __forceinline__ void step_tensor(const TensorArg& t, const SetArg& h, const State& st,
                                            uint64_t at, float coef, bool clip) {
    constexpr uintptr_t kMask = kLaneElems * sizeof(T) - 1;
    const bool vec = (((uintptr_t)t.param | (uintptr_t)t.grad) & kMask) == 0;
    if (vec && at + (uint64_t)ITER * kThreads * kLaneElems <= t.n) {
        step_chunk<T, Q8, ITER, true, STREAM>(t, h, st, at, coef, clip);
    } else {
        step_chunk<T, Q8, ITER, false, false>(t, h, st, at, coef, clip);
    }
}

// A workgroup per chunk of 1024 ITER elements of one tensor: everything is
// read and written once, so memory bounds it. 2^28 float32 elements take 1302 us
// with moments in 32 bits (28 bytes each, 5.8 TB/s) and 734 in 8 (16.1 bytes, 5.9
// TB/s; counters: 2.72 GB read, 1.63 written, which is what there is); 2 million,
// clipped, 5.4 us for the norm and 11.2 for the step; three small tensors 3.2.
template <bool Q8, int ITER, bool STREAM>
__global__ __launch_bounds__(256) void k_adamw_step(const Table tb, const State st) {
    float coef = 1.f;
    const bool clip = st.partials != nullptr;
    if (clip) {
        // every workgroup adds the few partials itself: no launch between
        double s = 0.0;
        for (uint32_t i = threadIdx.x; i < st.n_partials; i += kThreads) {
            s += st.partials[i];
        }
        const float norm = (float)sqrt(block_sum(s));
        const float q = st.max_norm / (norm + 1e-6f);
        coef = q > 1.f ? 1.f : q;  // a NaN stays one
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            *st.norm = norm;
        }
    }
    const TensorArg& t = tb.t[find_tensor(tb, blockIdx.x)];
    const SetArg h = st.sets ? st.sets[t.set] : tb.set[t.set];
    const uint64_t at = (uint64_t)(blockIdx.x - t.first_chunk) * (ITER * kThreads * kLaneElems);
    switch (t.type) {
        case DRESSI_F32:
            step_tensor<float, Q8, ITER, STREAM>(t, h, st, at, coef, clip);
            break;
        case DRESSI_BF16:
            step_tensor<bf16, Q8, ITER, STREAM>(t, h, st, at, coef, clip);
            break;
        default:
            step_tensor<f16, Q8, ITER, STREAM>(t, h, st, at, coef, clip);
    }
}

// What follows from a set's rates at step t.
__host__ __device__ inline SetArg set_arg(const dressi_adamw_set& s, uint64_t step, uint32_t seed) {
    SetArg a;
    a.b1 = (float)s.beta1;
    a.omb1 = (float)(1.0 - s.beta1);
    a.b2 = (float)s.beta2;
    a.omb2 = (float)(1.0 - s.beta2);
    a.eps = (float)s.eps;
    a.decay = (float)(1.0 - s.lr * s.weight_decay);
    a.step_size = (float)(s.lr / (1.0 - pow(s.beta1, (double)step)));
    a.inv_bc2 = (float)(1.0 / sqrt(1.0 - pow(s.beta2, (double)step)));
    a.key = (uint32_t)step * 0x9e3779b9u + seed * 0x632be5abu + 0x7f4a7c15u;
    return a;
}

// Steps that a graph may repeat: their count is on the device. One thread, a
// launch for each set: it is counted once, before the step's kernels read it.
__global__ __launch_bounds__(64) void k_adamw_tick(const dressi_adamw_set set, uint32_t seed,
                                                   uint64_t* step, SetArg* out) {
    if (threadIdx.x == 0) {
        *step += 1;
        *out = set_arg(set, *step, seed);
    }
}

// The values that 8-bit moments stand for, as bfloat16 (which holds them all:
// three mantissa bits). Two times 4 elements a lane; the values go past the caches
// (2^23 elements and a sum of both after them: 19.5 us, 20 through the caches), and
// so do the codes if they are too many for one (`STREAM`): 2^28 elements take 254
// us so (6.4 TB/s), 289 through them and 331 with 4 elements a lane; 2^26, whose
// codes a cache holds, 64 us past it and 59 through it.
constexpr uint32_t kValuesIter = 2;
template <bool STREAM>
__global__ __launch_bounds__(256) void k_adamw_values(const State st, uint64_t n, bf16* m,
                                                      bf16* v) {
    constexpr uint32_t kStep = kThreads * kLaneElems;
    const uint64_t at = (uint64_t)blockIdx.x * (kStep * kValuesIter) + threadIdx.x * kLaneElems;
    RawMoments<true> raw[kValuesIter];
#pragma unroll
    for (uint32_t k = 0; k < kValuesIter; k++) {
        if (at + k * kStep < n) {
            raw[k].load<STREAM>(st, at + k * kStep);
        }
    }
#pragma unroll
    for (uint32_t k = 0; k < kValuesIter; k++) {
        const uint64_t i = at + k * kStep;
        if (i < n) {
            const Moments o = raw[k].values();
            store_vec<bf16, kLaneElems, true>(m + i, o.m);
            store_vec<bf16, kLaneElems, true>(v + i, o.v);
        }
    }
}

// Elements up to which a workgroup takes 1024 of them, else 4096 (8-bit moments,
// which take more registers: 2048): more workgroups against more loads in flight
// in each. 8-bit moments take 25.7 us so and 27.8 with 4096 at 2^23 elements, and
// the two are level at 2^28; 32-bit ones are at 2^22, and 4096 leaves a quarter
// of the sums of a clipped norm (61 and 54 us at 2^23, both through the caches).
constexpr uint64_t kSmallTotal = 1ull << 20, kSmallTotal8 = 1ull << 23;

// Bytes of a step from which they go past the caches (256 MB the last), which hold
// less and less of them for the next one. Past them and through them: 117 MB 21.8
// and 19.4 us, 235 MB clipped 46.7 and 54.0, 940 MB 157 and 175, 7.5 GB 1315 and
// 1396; bfloat16 with 2^27 elements, 32-bit moments and clipped 730 and 829, 8-bit
// 422 and 446.
constexpr uint64_t kStreamBytes = 160ull << 20;

int check_tensors(const dressi_adamw_tensor* t, uint32_t n, uint32_t n_sets, uint64_t state_elems) {
    for (uint32_t i = 0; i < n; i++) {
        DRESSI_REQUIRE(t[i].n == 0 || (t[i].param && t[i].grad), "adamw: tensor %u has a NULL pointer", i);
        DRESSI_REQUIRE(t[i].type <= DRESSI_F16, "adamw: tensor %u has unknown type %u", i, t[i].type);
        DRESSI_REQUIRE(t[i].set < n_sets, "adamw: tensor %u names set %u of %u", i, t[i].set, n_sets);
        DRESSI_REQUIRE(t[i].state % kBlock == 0, "adamw: tensor %u's state is not at a multiple of %u",
                       i, kBlock);
        const size_t size = t[i].type == DRESSI_F32 ? 4 : 2;
        DRESSI_REQUIRE(((uintptr_t)t[i].param | (uintptr_t)t[i].grad) % size == 0,
                       "adamw: tensor %u is not aligned to its type", i);
        DRESSI_REQUIRE(((uintptr_t)t[i].master & 15) == 0,
                       "adamw: tensor %u's master is not aligned", i);
        DRESSI_REQUIRE(t[i].n <= (1ull << 40), "adamw: tensor %u is too large", i);
        const uint64_t padded = (t[i].n + kBlock - 1) / kBlock * kBlock;
        DRESSI_REQUIRE(t[i].state <= state_elems && padded <= state_elems - t[i].state,
                       "adamw: tensor %u's share ends past the state buffers", i);
    }
    return DRESSI_OK;
}

int check_set(const dressi_adamw_set& s, uint32_t i, bool on_device) {
    DRESSI_REQUIRE(s.lr >= 0.0 && std::isfinite(s.lr), "adamw: lr %g of set %u", s.lr, i);
    DRESSI_REQUIRE(s.beta1 >= 0.0 && s.beta1 < 1.0, "adamw: beta1 %g of set %u", s.beta1, i);
    DRESSI_REQUIRE(s.beta2 >= 0.0 && s.beta2 < 1.0, "adamw: beta2 %g of set %u", s.beta2, i);
    DRESSI_REQUIRE(s.eps >= 0.0 && std::isfinite(s.eps), "adamw: eps %g of set %u", s.eps, i);
    DRESSI_REQUIRE(s.weight_decay >= 0.0 && std::isfinite(s.weight_decay),
                   "adamw: weight_decay %g of set %u", s.weight_decay, i);
    DRESSI_REQUIRE(on_device || s.step >= 1, "adamw: step 0 of set %u (the first is 1)", i);
    return DRESSI_OK;
}

// Calls f(table) for each launch. on_device: the entries keep their sets' own
// numbers.
template <typename F>
int for_batches(const dressi_adamw_tensor* t, uint32_t n, const dressi_adamw_set* sets,
                bool on_device, uint32_t seed, uint32_t chunk_elems, F&& f) {
    Table tb;
    uint32_t set_of[kMaxSets];
    uint32_t n_sets = 0;
    tb.n_tensors = tb.n_chunks = 0;
    for (uint32_t i = 0; i < n; i++) {
        if (t[i].n == 0) {
            continue;
        }
        // a tensor's chunks of one launch: more go into further entries
        uint64_t done = 0;
        while (done < t[i].n) {
            uint32_t s = 0;
            while (!on_device && s < n_sets && set_of[s] != t[i].set) {
                s++;
            }
            if (tb.n_tensors == kMaxTensors || s == kMaxSets || tb.n_chunks == (1u << 23)) {
                if (int rc = f(tb)) {
                    return rc;
                }
                tb.n_tensors = tb.n_chunks = n_sets = 0;
                continue;
            }
            if (on_device) {
                s = t[i].set;
            } else if (s == n_sets) {
                set_of[n_sets++] = t[i].set;
                tb.set[s] = set_arg(sets[t[i].set], sets[t[i].set].step, seed);
            }
            const uint64_t room = (uint64_t)((1u << 23) - tb.n_chunks) * chunk_elems;
            const uint64_t take = std::min<uint64_t>(room, t[i].n - done);
            const size_t size = t[i].type == DRESSI_F32 ? 4 : 2;
            TensorArg& a = tb.t[tb.n_tensors++];
            a.param = (char*)t[i].param + done * size;
            a.grad = (const char*)t[i].grad + done * size;
            a.master = t[i].master ? t[i].master + done : nullptr;
            a.n = take;
            a.state = t[i].state + done;
            a.first_chunk = tb.n_chunks;
            a.type = (uint16_t)t[i].type;
            a.set = (uint16_t)s;
            tb.n_chunks += (uint32_t)((take + chunk_elems - 1) / chunk_elems);
            done += take;
        }
    }
    return tb.n_tensors ? f(tb) : DRESSI_OK;
}

}  // namespace
}  // namespace dressi

using namespace dressi;

extern "C" {

size_t dressi_adamw_set_bytes(void) { return sizeof(SetArg); }

size_t dressi_adamw_scratch(void) { return kMaxPartials * sizeof(double); }

int dressi_adamw_step(dressi_ctx* ctx, const dressi_adamw_tensor* tensors, uint32_t n_tensors,
                      const dressi_adamw_set* sets, uint32_t n_sets, uint32_t state_bits,
                      uint64_t state_elems, void* exp_avg, void* exp_avg_sq,
                      uint8_t* exp_avg_scale, uint8_t* exp_avg_sq_scale, uint32_t seed,
                      float max_norm, void* scratch, float* norm, uint64_t* steps,
                      void* device_sets) {
    DRESSI_REQUIRE(ctx, "NULL context");
    if (n_tensors == 0) {
        return DRESSI_OK;
    }
    DRESSI_REQUIRE(tensors && sets && n_sets > 0, "adamw: bad arguments");
    DRESSI_REQUIRE(state_bits == 8 || state_bits == 32, "adamw: state_bits %u is not 8 or 32",
                   state_bits);
    DRESSI_REQUIRE((exp_avg && exp_avg_sq) || state_elems == 0, "adamw: NULL state");
    const bool q8 = state_bits == 8;
    DRESSI_REQUIRE(!q8 || (exp_avg_scale && exp_avg_sq_scale) || state_elems == 0,
                   "adamw: 8-bit moments need their scales");
    const uintptr_t mask = q8 ? 3 : 15;
    DRESSI_REQUIRE((((uintptr_t)exp_avg | (uintptr_t)exp_avg_sq) & mask) == 0,
                   "adamw: the state buffers are not aligned");
    DRESSI_REQUIRE(!steps == !device_sets && n_sets <= 65536, "adamw: bad sets");
    const bool on_device = steps != nullptr;
    DRESSI_REQUIRE(max_norm >= 0.f, "adamw: max_norm %g", (double)max_norm);
    const bool clip = max_norm > 0.f;
    DRESSI_REQUIRE(!clip || (scratch && norm), "adamw: clipping needs scratch and norm");
    if (int rc = check_tensors(tensors, n_tensors, n_sets, state_elems)) {
        return rc;
    }
    uint64_t total = 0, bytes = 0;  // elements, and what is read and written of them
    for (uint32_t i = 0; i < n_tensors; i++) {
        total += tensors[i].n;
        const bool wide = tensors[i].type != DRESSI_F32 && tensors[i].master;
        bytes += tensors[i].n * (3 * type_bytes(tensors[i].type) + (wide ? 8 : 0) + (q8 ? 4 : 16));
    }
    for (uint32_t i = 0; i < n_sets; i++) {
        if (int rc = check_set(sets[i], i, steps != nullptr)) {
            return rc;
        }
    }
    if (total == 0) {
        return clip ? launch_zero(ctx->stream, norm, sizeof(float)) : DRESSI_OK;
    }
    const bool small = total <= (q8 ? kSmallTotal8 : kSmallTotal);
    const bool stream = bytes >= kStreamBytes;
    const uint32_t iter = small ? 1 : q8 ? 2 : 4;
    const uint32_t chunk = kThreads * kLaneElems * iter;
    State st{(const SetArg*)device_sets, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, nullptr, 0, max_norm, norm};
    if (clip) {
        uint32_t launches = 0;
        for_batches(tensors, n_tensors, sets, on_device, seed, chunk, [&](const Table&) {
            launches++;
            return (int)DRESSI_OK;
        });
        DRESSI_REQUIRE(launches <= kMaxPartials, "adamw: too many tensors to clip (%u launches)",
                       launches);
        const uint32_t share = launches ? kMaxPartials / launches : 1;
        uint32_t used = 0;
        const int rc = for_batches(
            tensors, n_tensors, sets, on_device, seed, chunk, [&](const Table& tb) -> int {
                const uint32_t grid = std::min(tb.n_chunks, std::min(share, 512u));
                double* out = (double*)scratch + used;
                const auto squares = iter == 1   ? k_adamw_squares<1>
                                     : iter == 2 ? k_adamw_squares<2>
                                                 : k_adamw_squares<4>;
                hipLaunchKernelGGL(squares, dim3(grid), dim3(kThreads), 0, ctx->stream, tb, out);
                DRESSI_CHECK_LAUNCH();
                used += grid;
                return DRESSI_OK;
            });
        if (rc) {
            return rc;
        }
        st.partials = (const double*)scratch;
        st.n_partials = used;
    }
    // after all that may be refused: a step that is not taken does not count
    for (uint32_t i = 0; on_device && i < n_sets; i++) {
        hipLaunchKernelGGL(k_adamw_tick, dim3(1), dim3(64), 0, ctx->stream, sets[i], seed,
                           steps + i, (SetArg*)device_sets + i);
        DRESSI_CHECK_LAUNCH();
    }
    return for_batches(tensors, n_tensors, sets, on_device, seed, chunk, [&](const Table& tb) -> int {
        const auto step =
            q8 ? (small ? k_adamw_step<true, 1, false>
                  : stream ? k_adamw_step<true, 2, true> : k_adamw_step<true, 2, false>)
               : (small ? k_adamw_step<false, 1, false>
                  : stream ? k_adamw_step<false, 4, true> : k_adamw_step<false, 4, false>);
        hipLaunchKernelGGL(step, dim3(tb.n_chunks), dim3(kThreads), 0, ctx->stream, tb, st);
        DRESSI_CHECK_LAUNCH();
        return DRESSI_OK;
    });
}

int dressi_adamw_values(dressi_ctx* ctx, uint64_t n, const void* exp_avg, const void* exp_avg_sq,
                        const uint8_t* exp_avg_scale, const uint8_t* exp_avg_sq_scale,
                        void* exp_avg_bf16, void* exp_avg_sq_bf16) {
    DRESSI_REQUIRE(ctx, "NULL context");
    if (n == 0) {
        return DRESSI_OK;
    }
    DRESSI_REQUIRE(exp_avg && exp_avg_sq && exp_avg_scale && exp_avg_sq_scale && exp_avg_bf16 &&
                       exp_avg_sq_bf16,
                   "adamw: bad arguments");
    DRESSI_REQUIRE(n % kBlock == 0, "adamw: %llu elements are not whole blocks of %u",
                   (unsigned long long)n, kBlock);
    DRESSI_REQUIRE((((uintptr_t)exp_avg | (uintptr_t)exp_avg_sq) & 3) == 0 &&
                       (((uintptr_t)exp_avg_bf16 | (uintptr_t)exp_avg_sq_bf16) & 7) == 0,
                   "adamw: the buffers are not aligned");
    State st{nullptr, (void*)exp_avg, (void*)exp_avg_sq, (uint8_t*)exp_avg_scale,
             (uint8_t*)exp_avg_sq_scale, nullptr, 0, 0.f, nullptr};
    const auto values = 2 * n >= kStreamBytes ? k_adamw_values<true> : k_adamw_values<false>;
    // within the launch limit, in whole blocks
    constexpr uint64_t kShare = kThreads * kLaneElems * kValuesIter;
    constexpr uint64_t kPiece = kLaunchThreads / kThreads * kShare;
    for (uint64_t at = 0; at < n; at += kPiece) {
        const uint64_t take = std::min(kPiece, n - at);
        State s = st;
        s.m = (uint8_t*)st.m + at;
        s.v = (uint8_t*)st.v + at;
        s.m_scale = st.m_scale + at / kBlock;
        s.v_scale = st.v_scale + at / kBlock;
        const uint32_t blocks = (uint32_t)((take + kShare - 1) / kShare);
        hipLaunchKernelGGL(values, dim3(blocks), dim3(kThreads), 0, ctx->stream, s, take,
                           (bf16*)exp_avg_bf16 + at, (bf16*)exp_avg_sq_bf16 + at);
        DRESSI_CHECK_LAUNCH();
    }
    return DRESSI_OK;
}

}  // extern "C"
