// clip.hip -- the norm of many tensors together, and their elements scaled down
// to a largest one (dressi_clip_norm).
//
//   |g| = (sum g^2)^(1/2), or the largest |g|, over all elements of all tensors
//   g = g min(1, max_norm / (|g| + 1e-6))
//
// Squares are added in double: a float's may not be one. The factor is rounded to
// float once, each product once to the tensor's type. Memory bounds it, launches
// where there is little: three operations an element. All of a small set lies in
// the registers of one workgroup, in one launch. Else two launches read the
// elements: the first leaves each workgroup's share of the norm, the second joins
// the shares, every workgroup for itself, and scales, backwards and each part on
// the die that read it, so that it finds what was read last in a cache. Where the
// norm is below max_norm the second ends there.
//
// 2^28 float32 elements: 158 us for the norm, 6.8 TB/s, and 375 for the scaling,
// 5.7 TB/s over the 2.1 GB that it reads and writes; 2^28 of 16 bits 83 and 178,
// 6.0 TB/s; 2^24 float32 17 and 21; three small tensors 3.4 in all. These times and
// those below are of graphs of some calls, from 48 MB of gradients on of others
// each time, as a training step has: over the same ones again a cache would still
// hold what the call before wrote last (2^28 float32 522 us in place of 533).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <new>
#include <vector>

#include "internal.h"
#include "typed.h"

namespace dressi {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kMaxTensors = 128;     // of a launch
constexpr uint32_t kMaxPartials = 4096;   // of a call
constexpr uint32_t kBytes = 16;           // a lane's neighbours
constexpr uint32_t kSmallThreads = 1024;  // of the one workgroup that holds a small set
constexpr uint32_t kSmallVecs = 8;        // of a thread of it

struct TensorArg {
    void* data;
    uint64_t n;
    uint32_t first;  // of the launch's chunks, or vectors
    uint32_t type;
};
// A launch's tensors: in the kernel arguments, so that no copy to the device
// stands before it. 4 KB at most (a table of 16 saves 0.2 us of a launch's 4 on
// the host).
struct Table {
    TensorArg t[kMaxTensors];
    uint32_t n_tensors, n_chunks;
    uint32_t keep;  // the last chunks, which a cache keeps from the first pass to the second
};
static_assert(sizeof(Table) <= 3800, "with the pointers beside it within 4 KB of arguments");

// The tensor that holds `chunk`: the last whose first chunk is not past it.
// Lanes look at two tensors each, one load deep.
__device__ __forceinline__ uint32_t find_tensor(const Table& tb, uint32_t chunk) {
    static_assert(kMaxTensors == 128, "two tensors a lane");
    const uint32_t lane = threadIdx.x & 63u;
    const bool a = lane < tb.n_tensors && tb.t[lane].first <= chunk;
    const bool b = lane + 64 < tb.n_tensors && tb.t[lane + 64].first <= chunk;
    return __builtin_amdgcn_readfirstlane(
        (uint32_t)(__popcll(__ballot(a)) + __popcll(__ballot(b))) - 1);
}

// A norm's sum, of squares or of magnitudes' bits: the bits of a larger magnitude
// are larger, and a NaN's larger than all others.
template <bool LARGEST>
struct Sum;
template <>
struct Sum<false> {
    double s = 0.0;
    __device__ __forceinline__ void add(float x) { s = fma((double)x, (double)x, s); }
    __device__ __forceinline__ void join(double x) { s += x; }
    __device__ __forceinline__ double value() const { return s; }
    __device__ __forceinline__ double norm() const { return sqrt(s); }
};
template <>
struct Sum<true> {
    uint32_t s = 0;
    __device__ __forceinline__ void add(float x) {
        s = std::max(s, __float_as_uint(x) & 0x7fffffffu);
    }
    __device__ __forceinline__ void join(double x) { add((float)x); }
    __device__ __forceinline__ double value() const { return (double)__uint_as_float(s); }
    __device__ __forceinline__ double norm() const { return value(); }
};

// A workgroup's sum, in all threads.
template <bool LARGEST, uint32_t THREADS>
__device__ __forceinline__ void block_join(Sum<LARGEST>& s) {
    __shared__ double part[THREADS / 64];
    for (int o = 32; o > 0; o >>= 1) {
        s.join(__shfl_xor(s.value(), o));
    }
    if ((threadIdx.x & 63u) == 0) {
        part[threadIdx.x >> 6] = s.value();
    }
    __syncthreads();
    s = Sum<LARGEST>();
    for (uint32_t i = 0; i < THREADS / 64; i++) {
        s.join(part[i]);
    }
}

// The factor of a norm; 1 where the elements stay as they are.
__device__ __forceinline__ float factor(double norm, double max_norm) {
    if (isinf(max_norm)) {
        return 1.f;
    }
    const float c = (float)(max_norm / (norm + 1e-6));
    return c > 1.f ? 1.f : c;  // a NaN stays one
}

// A chunk of ITER vectors a thread: f(number, its elements as they lie in memory,
// how many of them there are), loads first. PAST: past the caches.
template <typename T, int ITER, bool PAST, typename F>
__device__ __forceinline__ void for_chunk(const T* g, uint64_t at, uint64_t n, F&& f) {
    constexpr uint32_t V = kBytes / sizeof(T), kStep = kThreads * V;
    const T* p = g + at + threadIdx.x * V;
    Pack<T, V> x[ITER];
    if (at + (uint64_t)ITER * kStep <= n) {
#pragma unroll
        for (int k = 0; k < ITER; k++) {
            x[k] = load_loose<T, V, PAST>(p + k * kStep);
        }
#pragma unroll
        for (int k = 0; k < ITER; k++) {
            f(p + k * kStep, x[k], V);
        }
        return;
    }
    for (uint32_t k = 0; k < ITER; k++) {
        const uint64_t i = at + k * kStep + threadIdx.x * V;
        const uint32_t count = i >= n ? 0 : n - i < V ? (uint32_t)(n - i) : V;
        for (uint32_t j = 0; j < V; j++) {
            x[0].v[j] = j < count ? g[i + j] : (T)0.f;
        }
        f(p + k * kStep, x[0], count);
    }
}

template <typename F>
__device__ __forceinline__ void for_type(uint32_t type, F&& f) {
    switch (type) {
        case DRESSI_F32:
            f((float*)nullptr);
            break;
        case DRESSI_BF16:
            f((bf16*)nullptr);
            break;
        default:
            f((f16*)nullptr);
    }
}

// Calls f(tensor, first element of the chunk, whether it is read past the caches)
// for the workgroup's chunks: every gridDim.x-th, forwards or backwards.
template <int ITER, bool BACK, typename F>
__device__ __forceinline__ void for_chunks(const Table& tb, F&& f) {
    const uint32_t rounds = (tb.n_chunks - blockIdx.x + gridDim.x - 1) / gridDim.x;
    TensorArg t{};
    uint32_t end = 0;  // chunks of t: first .. end
    for (uint32_t r = 0; r < rounds; r++) {
        const uint32_t c = blockIdx.x + (BACK ? rounds - 1 - r : r) * gridDim.x;
        if (c < t.first || c >= end) {
            t = tb.t[find_tensor(tb, c)];
            const uint32_t size = t.type == DRESSI_F32 ? 4 : 2;
            const uint64_t elems = (uint64_t)ITER * kThreads * kBytes / size;
            end = t.first + (uint32_t)((t.n + elems - 1) / elems);
        }
        f(t, c - t.first, c + tb.keep < tb.n_chunks);
    }
}

// A workgroup's share of the norm.
template <bool LARGEST, int ITER>
__global__ __launch_bounds__(kThreads) void k_clip_norm(const Table tb, double* partials) {
    Sum<LARGEST> s;
    for_chunks<ITER, false>(tb, [&](const TensorArg& t, uint32_t chunk, bool past) {
        for_type(t.type, [&](auto* type) {
            using T = std::remove_pointer_t<decltype(type)>;
            const uint64_t at = (uint64_t)chunk * (ITER * kThreads * kBytes / sizeof(T));
            const auto add = [&](const T*, const auto& x, uint32_t) {
#pragma unroll
                for (uint32_t j = 0; j < kBytes / sizeof(T); j++) {
                    s.add(to_float(x.v[j]));
                }
            };
            if (past) {
                asm volatile("");  // or the two become one branch, through the caches
                for_chunk<T, ITER, true>((const T*)t.data, at, t.n, add);
                asm volatile("");
            } else {
                for_chunk<T, ITER, false>((const T*)t.data, at, t.n, add);
            }
        });
    });
    block_join<LARGEST, kThreads>(s);
    if (threadIdx.x == 0) {
        partials[blockIdx.x] = s.value();
    }
}

// Joins the shares (every workgroup for itself: no launch between) and scales.
template <bool LARGEST, int ITER>
__global__ __launch_bounds__(kThreads) void k_clip_scale(const Table tb, const double* partials,
                                                         uint32_t n_partials, double max_norm,
                                                         float* norm_out) {
    Sum<LARGEST> s;
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < n_partials; i += kThreads) {
        s.join(partials[i]);
    }
    block_join<LARGEST, kThreads>(s);
    const double norm = s.norm();
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        *norm_out = (float)norm;
    }
    const float coef = factor(norm, max_norm);
    if (coef == 1.f) {
        return;
    }
    for_chunks<ITER, true>(tb, [&](const TensorArg& t, uint32_t chunk, bool past) {
        for_type(t.type, [&](auto* type) {
            using T = std::remove_pointer_t<decltype(type)>;
            constexpr uint32_t V = kBytes / sizeof(T);
            const uint64_t at = (uint64_t)chunk * (ITER * kThreads * V);
            const auto scale = [&](const T* p, const auto& x, uint32_t count) {
                float v[V];
                unpack(x, v);
#pragma unroll
                for (uint32_t j = 0; j < V; j++) {
                    v[j] *= coef;
                }
                if (count == V) {
                    store_loose<T, V, true>((T*)p, v);
                    return;
                }
#pragma unroll
                for (uint32_t j = 0; j < V; j++) {
                    if (j < count) {
                        ((T*)p)[j] = from_float<T>(v[j]);
                    }
                }
            };
            if (past) {
                asm volatile("");
                for_chunk<T, ITER, true>((const T*)t.data, at, t.n, scale);
                asm volatile("");
            } else {
                for_chunk<T, ITER, false>((const T*)t.data, at, t.n, scale);
            }
        });
    });
}

// A small set: norm and scaling by one workgroup that holds all vectors.
// `n_chunks` and `first` count vectors. 1930 elements 3.4 us, 30000 8.1: two
// launches over 40000 take 5.6, but 4 us more of the host, which is what counts
// outside of a graph.
template <bool LARGEST>
__global__ __launch_bounds__(kSmallThreads) void k_clip_small(const Table tb, double max_norm,
                                                              float* norm_out) {
    __shared__ TensorArg list[kMaxTensors];
    if (threadIdx.x < tb.n_tensors) {
        list[threadIdx.x] = tb.t[threadIdx.x];
    }
    __syncthreads();
    struct Vec {
        uint4 x;
        char* p;
        uint32_t type, count;
    } v[kSmallVecs];
    Sum<LARGEST> s;
#pragma unroll
    for (uint32_t k = 0; k < kSmallVecs; k++) {
        const uint32_t i = k * kSmallThreads + threadIdx.x;
        v[k].count = 0;
        if (i < tb.n_chunks) {
            uint32_t lo = 0, hi = tb.n_tensors;  // the last tensor that begins at i or before
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) / 2;
                (list[mid].first <= i ? lo : hi) = mid;
            }
            const TensorArg t = list[lo];
            const uint32_t size = t.type == DRESSI_F32 ? 4 : 2, per = kBytes / size;
            const uint64_t at = (uint64_t)(i - t.first) * per;
            v[k].type = t.type;
            v[k].count = (uint32_t)std::min<uint64_t>(t.n - at, per);
            v[k].p = (char*)t.data + at * size;
            for_type(t.type, [&](auto* type) {
                using T = std::remove_pointer_t<decltype(type)>;
                constexpr uint32_t V = kBytes / sizeof(T);
                const T* p = (const T*)v[k].p;
                Pack<T, V> x;
                if (v[k].count == V) {
                    x = load_loose<T, V>(p);
                } else {
#pragma unroll
                    for (uint32_t j = 0; j < V; j++) {
                        x.v[j] = j < v[k].count ? p[j] : (T)0.f;
                    }
                }
                __builtin_memcpy(&v[k].x, &x, kBytes);
            });
        }
    }
#pragma unroll
    for (uint32_t k = 0; k < kSmallVecs; k++) {
        if (v[k].count > 0) {
            for_type(v[k].type, [&](auto* type) {
                using T = std::remove_pointer_t<decltype(type)>;
                Pack<T, kBytes / sizeof(T)> x;
                __builtin_memcpy(&x, &v[k].x, kBytes);
#pragma unroll
                for (uint32_t j = 0; j < kBytes / sizeof(T); j++) {
                    s.add(to_float(x.v[j]));
                }
            });
        }
    }
    block_join<LARGEST, kSmallThreads>(s);
    const double norm = s.norm();
    if (threadIdx.x == 0) {
        *norm_out = (float)norm;
    }
    const float coef = factor(norm, max_norm);
    if (coef == 1.f) {
        return;
    }
#pragma unroll
    for (uint32_t k = 0; k < kSmallVecs; k++) {
        if (v[k].count > 0) {
            for_type(v[k].type, [&](auto* type) {
                using T = std::remove_pointer_t<decltype(type)>;
                constexpr uint32_t V = kBytes / sizeof(T);
                Pack<T, V> x;
                __builtin_memcpy(&x, &v[k].x, kBytes);
                float f[V];
                unpack(x, f);
#pragma unroll
                for (uint32_t j = 0; j < V; j++) {
                    f[j] *= coef;
                }
                if (v[k].count == V) {
                    store_loose<T, V>((T*)v[k].p, f);
                    return;
                }
#pragma unroll
                for (uint32_t j = 0; j < V; j++) {
                    if (j < v[k].count) {
                        ((T*)v[k].p)[j] = from_float<T>(f[j]);
                    }
                }
            });
        }
    }
}

// Bytes of all tensors up to which a chunk is 4 KB and not 16: more workgroups (42
// tensors of 588000 bfloat16 in all 7.5 us, 10.0 with chunks of 16 KB; 2^22 bfloat16
// 8.2 with those, 9.4 with 4 KB).
constexpr uint64_t kFewBytes = 4ull << 20;

// Bytes that the second pass may find in the last-level cache (256 MB); the rest
// goes past it both times. With more, what the cache held from before has to leave
// it in between: 2^28 float32 533 us (550 with 224 MB kept, 527 with none), 2^26
// 125 (142, 129), 2^24 38 (38, 37), and 32 where they were written just before (32,
// 35).
constexpr uint64_t kKeepBytes = 96ull << 20;

// Workgroups of a launch: four a compute unit (2^28 float32 533 us, the norm alone
// 158; 541 and 186 with half of them, 527 and 167 with twice as many, but 2^24 41
// where these take 38).
constexpr uint32_t kGroups = 1024;

int check_tensors(const dressi_clip_tensor* t, uint32_t n, bool written) {
    std::vector<std::pair<uintptr_t, uint32_t>> order;  // by address
    try {
        order.reserve(n);
    } catch (const std::bad_alloc&) {
        set_error("clip_norm: out of host memory for %u tensors", n);
        return DRESSI_ERR_INVALID;
    }
    for (uint32_t i = 0; i < n; i++) {
        DRESSI_REQUIRE(t[i].type <= DRESSI_F16, "clip_norm: tensor %u has unknown type %u", i,
                       t[i].type);
        DRESSI_REQUIRE(t[i].n == 0 || t[i].data, "clip_norm: tensor %u has a NULL pointer", i);
        DRESSI_REQUIRE((uintptr_t)t[i].data % type_bytes(t[i].type) == 0,
                       "clip_norm: tensor %u is not aligned to its type", i);
        DRESSI_REQUIRE(t[i].n <= (1ull << 40), "clip_norm: tensor %u is too large", i);
        if (t[i].n > 0 && written) {
            order.emplace_back((uintptr_t)t[i].data, i);
        }
    }
    std::sort(order.begin(), order.end());
    for (size_t k = 1; k < order.size(); k++) {
        const dressi_clip_tensor& a = t[order[k - 1].second];
        const uintptr_t end = order[k - 1].first + (uintptr_t)a.n * type_bytes(a.type);
        DRESSI_REQUIRE(end <= order[k].first, "clip_norm: tensors %u and %u share memory",
                       std::min(order[k - 1].second, order[k].second),
                       std::max(order[k - 1].second, order[k].second));
    }
    return DRESSI_OK;
}

// How much there is, and whether one workgroup takes it.
struct Size {
    uint64_t bytes = 0;
    bool small;
    Size(const dressi_clip_tensor* t, uint32_t n) {
        uint64_t vecs = 0;
        uint32_t some = 0;  // tensors with elements
        for (uint32_t i = 0; i < n; i++) {
            const uint64_t b = t[i].n * type_bytes(t[i].type);
            bytes += b;
            vecs += (b + kBytes - 1) / kBytes;
            some += b > 0;
        }
        small = some <= kMaxTensors && vecs <= kSmallThreads * kSmallVecs;
    }
};

// Calls f(table) for each launch, in chunks of so many bytes.
template <typename F>
int for_batches(const dressi_clip_tensor* t, uint32_t n, uint32_t chunk_bytes, F&& f) {
    constexpr uint32_t kMostChunks = 1u << 30;
    Table tb;
    tb.n_tensors = tb.n_chunks = 0;
    const auto flush = [&]() -> int {
        tb.keep = (uint32_t)std::min<uint64_t>(tb.n_chunks, kKeepBytes / chunk_bytes);
        return f(tb);
    };
    for (uint32_t i = 0; i < n; i++) {
        const uint32_t size = (uint32_t)type_bytes(t[i].type), chunk = chunk_bytes / size;
        uint64_t done = 0;
        while (done < t[i].n) {
            if (tb.n_tensors == kMaxTensors || tb.n_chunks == kMostChunks) {
                if (int rc = flush()) {
                    return rc;
                }
                tb.n_tensors = tb.n_chunks = 0;
            }
            const uint64_t room = (uint64_t)(kMostChunks - tb.n_chunks) * chunk;
            const uint64_t take = std::min<uint64_t>(room, t[i].n - done);
            tb.t[tb.n_tensors++] =
                TensorArg{(char*)t[i].data + done * size, take, tb.n_chunks, t[i].type};
            tb.n_chunks += (uint32_t)((take + chunk - 1) / chunk);
            done += take;
        }
    }
    return tb.n_tensors ? flush() : DRESSI_OK;
}

template <bool LARGEST, int ITER>
int clip_in_two(hipStream_t s, const dressi_clip_tensor* tensors, uint32_t n_tensors,
                double max_norm, double* scratch, float* norm) {
    constexpr uint32_t kChunkBytes = ITER * kThreads * kBytes;
    uint32_t launches = 0;
    for_batches(tensors, n_tensors, kChunkBytes, [&](const Table&) {
        launches++;
        return (int)DRESSI_OK;
    });
    DRESSI_REQUIRE(launches <= kMaxPartials, "clip_norm: too many tensors (%u launches)", launches);
    const uint32_t most = std::min(kGroups, kMaxPartials / launches);
    uint32_t used = 0;
    int rc = for_batches(tensors, n_tensors, kChunkBytes, [&](const Table& tb) -> int {
        const uint32_t grid = std::min(tb.n_chunks, most);
        hipLaunchKernelGGL((k_clip_norm<LARGEST, ITER>), dim3(grid), dim3(kThreads), 0, s, tb,
                           scratch + used);
        DRESSI_CHECK_LAUNCH();
        used += grid;
        return DRESSI_OK;
    });
    if (rc) {
        return rc;
    }
    const auto scale = [&](const Table& tb) -> int {
        const uint32_t grid = std::max(1u, std::min(tb.n_chunks, most));
        hipLaunchKernelGGL((k_clip_scale<LARGEST, ITER>), dim3(grid), dim3(kThreads), 0, s, tb,
                           (const double*)scratch, used, max_norm, norm);
        DRESSI_CHECK_LAUNCH();
        return DRESSI_OK;
    };
    if (std::isinf(max_norm)) {  // the norm alone
        Table none;
        none.n_tensors = none.n_chunks = none.keep = 0;
        return scale(none);
    }
    return for_batches(tensors, n_tensors, kChunkBytes, scale);
}

template <bool LARGEST>
int clip(hipStream_t s, const Size& size, const dressi_clip_tensor* tensors, uint32_t n_tensors,
         double max_norm, double* scratch, float* norm) {
    if (!size.small) {
        const auto run = size.bytes <= kFewBytes ? clip_in_two<LARGEST, 1>
                                                 : clip_in_two<LARGEST, 4>;
        return run(s, tensors, n_tensors, max_norm, scratch, norm);
    }
    return for_batches(tensors, n_tensors, kBytes, [&](const Table& tb) -> int {
        hipLaunchKernelGGL((k_clip_small<LARGEST>), dim3(1), dim3(kSmallThreads), 0, s, tb,
                           max_norm, norm);
        DRESSI_CHECK_LAUNCH();
        return DRESSI_OK;
    });
}

}  // namespace
}  // namespace dressi

using namespace dressi;

extern "C" {

size_t dressi_clip_norm_scratch(const dressi_clip_tensor* tensors, uint32_t n_tensors) {
    return Size(tensors, n_tensors).small ? 0 : kMaxPartials * sizeof(double);
}

int dressi_clip_norm(dressi_ctx* ctx, const dressi_clip_tensor* tensors, uint32_t n_tensors,
                     uint32_t kind, double max_norm, void* scratch, float* norm) {
    DRESSI_REQUIRE(ctx, "NULL context");
    DRESSI_REQUIRE((tensors || n_tensors == 0) && norm, "clip_norm: bad arguments");
    DRESSI_REQUIRE(kind <= DRESSI_NORM_LARGEST, "clip_norm: unknown norm %u", kind);
    DRESSI_REQUIRE(max_norm >= 0.0, "clip_norm: max_norm %g", max_norm);
    if (int rc = check_tensors(tensors, n_tensors, std::isfinite(max_norm))) {
        return rc;
    }
    const Size size(tensors, n_tensors);
    DRESSI_REQUIRE(size.small || (scratch && ((uintptr_t)scratch & 7) == 0),
                   "clip_norm: bad scratch");
    const DeviceScope scope(ctx->device);
    DRESSI_TRY_HIP(scope.error());
    if (size.bytes == 0) {
        return launch_zero(ctx->stream, norm, sizeof(float));
    }
    const bool largest = kind == DRESSI_NORM_LARGEST;
    return (largest ? clip<true> : clip<false>)(ctx->stream, size, tensors, n_tensors, max_norm,
                                                (double*)scratch, norm);
}

}  // extern "C"
