// clip.hip -- the norm of many tensors together, and their elements scaled down
// to a largest one (dressi_clip_norm).
//
//   |g| = (sum g^2)^(1/2), or the largest |g|, over all elements of all tensors
//   g = g min(1, max_norm / (|g| + 1e-6))
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
constexpr uint32_t kMaxTensors = 128;    // of a launch
constexpr uint32_t kMaxPartials = 4096;  // of a call
constexpr uint32_t kChunk = 4096;        // elements

struct TensorArg {
    void* data;
    uint64_t n;
    uint32_t first_chunk, type;
};
// A launch's tensors: in the kernel arguments, so that no copy to the device
// stands before it. 4 KB at most.
struct Table {
    TensorArg t[kMaxTensors];
    uint32_t n_tensors, n_chunks;
};
static_assert(sizeof(Table) <= 3800, "with the pointers beside it within 4 KB of arguments");

// The tensor that holds `chunk`: the last whose first chunk is not past it.
// Lanes look at two tensors each, one load deep.
__device__ __forceinline__ uint32_t find_tensor(const Table& tb, uint32_t chunk) {
    static_assert(kMaxTensors == 128, "two tensors a lane");
    const uint32_t lane = threadIdx.x & 63u;
    const bool a = lane < tb.n_tensors && tb.t[lane].first_chunk <= chunk;
    const bool b = lane + 64 < tb.n_tensors && tb.t[lane + 64].first_chunk <= chunk;
    return __builtin_amdgcn_readfirstlane(
        (uint32_t)(__popcll(__ballot(a)) + __popcll(__ballot(b))) - 1);
}

// Of the 2-norm sums, in double: a float's square may not be one. Of the largest
// magnitude the larger, and a NaN stays.
template <bool LARGEST>
__device__ __forceinline__ double joined(double a, double b) {
    return !LARGEST ? a + b : a > b || a != a ? a : b;
}
template <bool LARGEST>
__device__ __forceinline__ double with(double a, float x) {
    return LARGEST ? joined<true>(a, (double)fabsf(x)) : fma((double)x, (double)x, a);
}

// The workgroup's, in all threads.
template <bool LARGEST>
__device__ __forceinline__ double block_join(double s) {
    __shared__ double part[kThreads / 64];
    for (int o = 32; o > 0; o >>= 1) {
        s = joined<LARGEST>(s, __shfl_xor(s, o));
    }
    if ((threadIdx.x & 63u) == 0) {
        part[threadIdx.x >> 6] = s;
    }
    __syncthreads();
    s = part[0];
    for (uint32_t i = 1; i < kThreads / 64; i++) {
        s = joined<LARGEST>(s, part[i]);
    }
    return s;
}

template <typename T, bool LARGEST>
__device__ __forceinline__ double chunk_norm(const T* g, uint64_t at, uint64_t end, double s) {
    for (uint64_t i = at + threadIdx.x; i < end; i += kThreads) {
        s = with<LARGEST>(s, to_float(g[i]));
    }
    return s;
}
template <typename T>
__device__ __forceinline__ void chunk_scale(T* g, uint64_t at, uint64_t end, float coef) {
    for (uint64_t i = at + threadIdx.x; i < end; i += kThreads) {
        g[i] = from_float<T>(to_float(g[i]) * coef);
    }
}

// A workgroup's share of the norm.
template <bool LARGEST>
__global__ __launch_bounds__(kThreads) void k_clip_norm(const Table tb, double* partials) {
    double s = 0.0;
    for (uint32_t c = blockIdx.x; c < tb.n_chunks; c += gridDim.x) {
        const TensorArg& t = tb.t[find_tensor(tb, c)];
        const uint64_t at = (uint64_t)(c - t.first_chunk) * kChunk;
        const uint64_t end = std::min<uint64_t>(t.n, at + kChunk);
        s = t.type == DRESSI_F32    ? chunk_norm<float, LARGEST>((const float*)t.data, at, end, s)
            : t.type == DRESSI_BF16 ? chunk_norm<bf16, LARGEST>((const bf16*)t.data, at, end, s)
                                    : chunk_norm<f16, LARGEST>((const f16*)t.data, at, end, s);
    }
    s = block_join<LARGEST>(s);
    if (threadIdx.x == 0) {
        partials[blockIdx.x] = s;
    }
}

// Joins the shares (every workgroup for itself: no launch between) and scales.
template <bool LARGEST>
__global__ __launch_bounds__(kThreads) void k_clip_scale(const Table tb, const double* partials,
                                                         uint32_t n_partials, double max_norm,
                                                         float* norm_out) {
    double s = 0.0;
    for (uint32_t i = threadIdx.x; i < n_partials; i += kThreads) {
        s = joined<LARGEST>(s, partials[i]);
    }
    s = block_join<LARGEST>(s);
    const double norm = LARGEST ? s : sqrt(s);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        *norm_out = (float)norm;
    }
    const float coef = (float)(max_norm / (norm + 1e-6));
    if (coef >= 1.f || isinf(max_norm)) {  // a NaN scales
        return;
    }
    for (uint32_t c = blockIdx.x; c < tb.n_chunks; c += gridDim.x) {
        const TensorArg& t = tb.t[find_tensor(tb, c)];
        const uint64_t at = (uint64_t)(c - t.first_chunk) * kChunk;
        const uint64_t end = std::min<uint64_t>(t.n, at + kChunk);
        switch (t.type) {
            case DRESSI_F32:
                chunk_scale((float*)t.data, at, end, coef);
                break;
            case DRESSI_BF16:
                chunk_scale((bf16*)t.data, at, end, coef);
                break;
            default:
                chunk_scale((f16*)t.data, at, end, coef);
        }
    }
}

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

// Calls f(table) for each launch.
template <typename F>
int for_batches(const dressi_clip_tensor* t, uint32_t n, F&& f) {
    constexpr uint32_t kMostChunks = 1u << 30;
    Table tb;
    tb.n_tensors = tb.n_chunks = 0;
    for (uint32_t i = 0; i < n; i++) {
        uint64_t done = 0;
        while (done < t[i].n) {
            if (tb.n_tensors == kMaxTensors || tb.n_chunks == kMostChunks) {
                if (int rc = f(tb)) {
                    return rc;
                }
                tb.n_tensors = tb.n_chunks = 0;
            }
            const uint64_t room = (uint64_t)(kMostChunks - tb.n_chunks) * kChunk;
            const uint64_t take = std::min<uint64_t>(room, t[i].n - done);
            tb.t[tb.n_tensors++] = TensorArg{(char*)t[i].data + done * type_bytes(t[i].type), take,
                                             tb.n_chunks, t[i].type};
            tb.n_chunks += (uint32_t)((take + kChunk - 1) / kChunk);
            done += take;
        }
    }
    return tb.n_tensors ? f(tb) : DRESSI_OK;
}

}  // namespace
}  // namespace dressi

using namespace dressi;

extern "C" {

size_t dressi_clip_norm_scratch(void) { return kMaxPartials * sizeof(double); }

int dressi_clip_norm(dressi_ctx* ctx, const dressi_clip_tensor* tensors, uint32_t n_tensors,
                     uint32_t kind, double max_norm, void* scratch, float* norm) {
    DRESSI_REQUIRE(ctx, "NULL context");
    DRESSI_REQUIRE((tensors || n_tensors == 0) && norm, "clip_norm: bad arguments");
    DRESSI_REQUIRE(kind <= DRESSI_NORM_LARGEST, "clip_norm: unknown norm %u", kind);
    DRESSI_REQUIRE(max_norm >= 0.0, "clip_norm: max_norm %g", max_norm);
    if (int rc = check_tensors(tensors, n_tensors, std::isfinite(max_norm))) {
        return rc;
    }
    uint32_t launches = 0;
    for_batches(tensors, n_tensors, [&](const Table&) {
        launches++;
        return (int)DRESSI_OK;
    });
    const DeviceScope scope(ctx->device);
    DRESSI_TRY_HIP(scope.error());
    if (launches == 0) {
        return launch_zero(ctx->stream, norm, sizeof(float));
    }
    DRESSI_REQUIRE(launches <= kMaxPartials, "clip_norm: too many tensors (%u launches)", launches);
    DRESSI_REQUIRE(scratch && ((uintptr_t)scratch & 7) == 0, "clip_norm: bad scratch");
    const uint32_t share = kMaxPartials / launches;
    const bool largest = kind == DRESSI_NORM_LARGEST;
    uint32_t used = 0;
    int rc = for_batches(tensors, n_tensors, [&](const Table& tb) -> int {
        const uint32_t grid = std::min({tb.n_chunks, share, 1024u});
        hipLaunchKernelGGL(largest ? k_clip_norm<true> : k_clip_norm<false>, dim3(grid),
                           dim3(kThreads), 0, ctx->stream, tb, (double*)scratch + used);
        DRESSI_CHECK_LAUNCH();
        used += grid;
        return DRESSI_OK;
    });
    if (rc) {
        return rc;
    }
    return for_batches(tensors, n_tensors, [&](const Table& tb) -> int {
        hipLaunchKernelGGL(largest ? k_clip_scale<true> : k_clip_scale<false>,
                           dim3(std::min(tb.n_chunks, 2048u)), dim3(kThreads), 0, ctx->stream, tb,
                           (const double*)scratch, used, max_norm, norm);
        DRESSI_CHECK_LAUNCH();
        return DRESSI_OK;
    });
}

}  // extern "C"
