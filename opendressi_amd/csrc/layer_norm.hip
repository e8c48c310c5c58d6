// layer_norm.hip -- layer normalisation of rows (the channels of each pixel)
// with an activation, forward and backward (dressi_layer_norm,
// dressi_layer_norm_bwd).
//
// A row of C values:
//
//   mu = mean x, s = 1 / sqrt(mean (x - mu)^2 + eps), xh = (x - mu) s
//   z = xh w + b, y = act(z)
//   gz = gy act'(z), gb = sum gz, gw = sum gz xh (over rows)
//   gx = s (w gz - mean(w gz) - xh mean(w gz xh))
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "internal.h"
#include "norm_core.h"
#include "typed.h"

namespace dressi {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kSumRows = 256;  // workgroups that share the rows of gw and gb

// Where rows lie: n_px to an item.
struct Rows {
    uint64_t n, n_px;
    uint64_t item_stride, px_stride;  // of x, in elements
    uint32_t n_ch;
    __device__ __forceinline__ size_t at(uint64_t row) const {
        const uint64_t item = row / n_px;
        return (size_t)(item * item_stride + (row - item * n_px) * px_stride);
    }
};

// A workgroup's sum, in all threads.
__device__ __forceinline__ float2 block_sum(float2 s) {
    __shared__ float2 part[kThreads / 64];
    for (int o = 1; o < 64; o <<= 1) {
        s.x += __shfl_xor(s.x, o);
        s.y += __shfl_xor(s.y, o);
    }
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) {
        part[threadIdx.x >> 6] = s;
    }
    __syncthreads();
    s = part[0];
    for (uint32_t i = 1; i < kThreads / 64; i++) {
        s.x += part[i].x;
        s.y += part[i].y;
    }
    return s;
}

// The row's value and channel's weight and bias: xh and z.
template <typename T>
__device__ __forceinline__ void value(const T* x, const Affine& aff, uint32_t ch, float mean,
                                      float rstd, float& xh, float (&w)[1], float (&z)[1]) {
    float b[1];
    load_affine<1>(aff, ch, w, b);
    xh = (to_float(x[ch]) - mean) * rstd;
    z[0] = fmaf(xh, w[0], b[0]);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void k_ln_forward(const T* x, const Rows rows,
                                                         const Affine aff, float eps, uint32_t act,
                                                         T* y, float* mean_out, float* rstd_out) {
    const float inv = 1.f / (float)rows.n_ch;
    for (uint64_t row = blockIdx.x; row < rows.n; row += gridDim.x) {
        const T* p = x + rows.at(row);
        float2 s = make_float2(0.f, 0.f);
        for (uint32_t c = threadIdx.x; c < rows.n_ch; c += kThreads) {
            s.x += to_float(p[c]);
        }
        const float m = block_sum(s).x * inv;
        s = make_float2(0.f, 0.f);
        for (uint32_t c = threadIdx.x; c < rows.n_ch; c += kThreads) {
            const float d = to_float(p[c]) - m;
            s.x += d;
            s.y = fmaf(d, d, s.y);
        }
        s = block_sum(s);
        const float off = s.x * inv, mean = m + off;
        const float var = fmaf(-off, off, s.y * inv);
        const float rstd = 1.f / sqrtf((var < 0.f ? 0.f : var) + eps);  // a NaN stays one
        for (uint32_t c = threadIdx.x; c < rows.n_ch; c += kThreads) {
            float xh, w[1], z[1];
            value(p, aff, c, mean, rstd, xh, w, z);
            act_values<T, 1>(act, z);
            y[row * rows.n_ch + c] = from_float<T>(z[0]);
        }
        if (threadIdx.x == 0 && mean_out) {
            mean_out[row] = mean;
            rstd_out[row] = rstd;
        }
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void k_ln_backward(const T* gy, const T* x, const Rows rows,
                                                          const Affine aff, uint32_t act,
                                                          const float* mean, const float* rstd,
                                                          T* gx) {
    const float inv = 1.f / (float)rows.n_ch;
    for (uint64_t row = blockIdx.x; row < rows.n; row += gridDim.x) {
        const T* p = x + rows.at(row);
        const T* q = gy + row * rows.n_ch;
        const float mu = mean[row], rs = rstd[row];
        float2 s = make_float2(0.f, 0.f);
        for (uint32_t c = threadIdx.x; c < rows.n_ch; c += kThreads) {
            float xh, w[1], z[1], g[1] = {to_float(q[c])};
            value(p, aff, c, mu, rs, xh, w, z);
            act_slopes<T, 1>(act, z, g);
            const float t = g[0] * w[0];
            s.x += t;
            s.y = fmaf(t, xh, s.y);
        }
        s = block_sum(s);
        for (uint32_t c = threadIdx.x; c < rows.n_ch; c += kThreads) {
            float xh, w[1], z[1], g[1] = {to_float(q[c])};
            value(p, aff, c, mu, rs, xh, w, z);
            act_slopes<T, 1>(act, z, g);
            gx[row * rows.n_ch + c] =
                from_float<T>(rs * (g[0] * w[0] - s.x * inv - xh * (s.y * inv)));
        }
    }
}

// Sums of gz and gz xh over the rows of a workgroup's share, a column a thread.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_ln_sums(const T* gy, const T* x, const Rows rows,
                                                      const Affine aff, uint32_t act,
                                                      const float* mean, const float* rstd,
                                                      float* part) {
    for (uint32_t c = blockIdx.y * kThreads + threadIdx.x; c < rows.n_ch;
         c += gridDim.y * kThreads) {
        float sw = 0.f, sb = 0.f;
        for (uint64_t row = blockIdx.x; row < rows.n; row += gridDim.x) {
            float xh, w[1], z[1], g[1] = {to_float(gy[row * rows.n_ch + c])};
            value(x + rows.at(row), aff, c, mean[row], rstd[row], xh, w, z);
            act_slopes<T, 1>(act, z, g);
            sw = fmaf(g[0], xh, sw);
            sb += g[0];
        }
        float* out = part + (size_t)blockIdx.x * 2 * rows.n_ch;
        out[c] = sw;
        out[rows.n_ch + c] = sb;
    }
}

// The shares' sums, in their order. n 0: sums of nothing.
__global__ __launch_bounds__(kThreads) void k_ln_params(const float* part, uint32_t n,
                                                        uint32_t n_ch, uint32_t type, void* gw,
                                                        void* gb) {
    for (uint32_t c = blockIdx.x * kThreads + threadIdx.x; c < n_ch; c += gridDim.x * kThreads) {
        float sw = 0.f, sb = 0.f;
        for (uint32_t i = 0; i < n; i++) {
            sw += part[(size_t)i * 2 * n_ch + c];
            sb += part[(size_t)i * 2 * n_ch + n_ch + c];
        }
        if (gw) {
            store_one(gw, type, c, sw);
        }
        if (gb) {
            store_one(gb, type, c, sb);
        }
    }
}

uint32_t grid_of(uint64_t n) { return (uint32_t)std::min<uint64_t>(n, 4096); }

int check_shape(const char* what, uint32_t type, uint64_t n_items, uint64_t n_px, uint32_t n_ch,
                uint64_t px_stride, uint32_t act, const Affine& aff) {
    DRESSI_REQUIRE(type <= DRESSI_F16, "%s: unknown type %u", what, type);
    DRESSI_REQUIRE(aff.type <= DRESSI_F16, "%s: unknown type %u of the weight", what, aff.type);
    DRESSI_REQUIRE(act <= DRESSI_ACT_GELU, "%s: unknown activation %u", what, act);
    DRESSI_REQUIRE(n_ch > 0 && n_ch <= (1u << 24), "%s: %u channels are not 1 to 2^24", what, n_ch);
    DRESSI_REQUIRE(n_px <= (1ull << 40) && n_items <= (1ull << 40) &&
                       (n_px == 0 || n_items <= (1ull << 40) / n_px),
                   "%s: too many rows", what);
    DRESSI_REQUIRE(px_stride >= n_ch || n_px <= 1, "%s: pixels overlap", what);
    return DRESSI_OK;
}

// f(a null pointer of the element type)
template <typename F>
int for_type(uint32_t type, F&& f) {
    return type == DRESSI_F32 ? f((float*)nullptr)
                              : type == DRESSI_BF16 ? f((bf16*)nullptr) : f((f16*)nullptr);
}

}  // namespace
}  // namespace dressi

using namespace dressi;

extern "C" {

size_t dressi_layer_norm_scratch(uint32_t type, uint64_t n_items, uint64_t n_px, uint32_t n_ch,
                                 int backward) {
    (void)type;
    const uint64_t rows = n_items * n_px;
    return backward ? std::min<uint64_t>(rows, kSumRows) * 2 * n_ch * sizeof(float) : 0;
}

int dressi_layer_norm(dressi_ctx* ctx, const void* x, uint32_t type, uint64_t n_items,
                      uint64_t n_px, uint32_t n_ch, uint64_t item_stride, uint64_t px_stride,
                      const void* weight, const void* bias, uint32_t affine_type, float eps,
                      uint32_t activation, void* scratch, size_t scratch_bytes, void* y,
                      float* mean, float* rstd) {
    DRESSI_REQUIRE(ctx, "NULL context");
    const Affine aff{weight, bias, affine_type};
    if (int rc = check_shape("layer_norm", type, n_items, n_px, n_ch, px_stride, activation, aff)) {
        return rc;
    }
    DRESSI_REQUIRE(eps >= 0.f && std::isfinite(eps), "layer_norm: eps %g", (double)eps);
    if (n_items == 0 || n_px == 0) {
        return DRESSI_OK;
    }
    DRESSI_REQUIRE(x && y && !mean == !rstd, "layer_norm: bad arguments");
    DRESSI_REQUIRE(((uintptr_t)x | (uintptr_t)y) % type_bytes(type) == 0,
                   "layer_norm: not aligned to its type");
    DRESSI_REQUIRE(
        scratch_bytes >= dressi_layer_norm_scratch(type, n_items, n_px, n_ch, 0),
        "layer_norm: scratch too small");
    (void)scratch;
    const DeviceScope scope(ctx->device);
    DRESSI_TRY_HIP(scope.error());
    const Rows rows{n_items * n_px, n_px, item_stride, px_stride, n_ch};
    return for_type(type, [&](auto* t) -> int {
        using T = std::remove_pointer_t<decltype(t)>;
        hipLaunchKernelGGL((k_ln_forward<T>), dim3(grid_of(rows.n)), dim3(kThreads), 0, ctx->stream,
                           (const T*)x, rows, aff, eps, activation, (T*)y, mean, rstd);
        DRESSI_CHECK_LAUNCH();
        return DRESSI_OK;
    });
}

int dressi_layer_norm_bwd(dressi_ctx* ctx, const void* gy, const void* x, uint32_t type,
                          uint64_t n_items, uint64_t n_px, uint32_t n_ch, uint64_t item_stride,
                          uint64_t px_stride, const void* weight, const void* bias,
                          uint32_t affine_type, uint32_t activation, const float* mean,
                          const float* rstd, void* scratch, size_t scratch_bytes, void* gx,
                          void* gw, void* gb) {
    DRESSI_REQUIRE(ctx, "NULL context");
    const Affine aff{weight, bias, affine_type};
    if (int rc = check_shape("layer_norm_bwd", type, n_items, n_px, n_ch, px_stride, activation,
                             aff)) {
        return rc;
    }
    if (!gx && !gw && !gb) {
        return DRESSI_OK;
    }
    const DeviceScope scope(ctx->device);
    DRESSI_TRY_HIP(scope.error());
    const Rows rows{n_items * n_px, n_px, item_stride, px_stride, n_ch};
    const uint32_t shares = (uint32_t)std::min<uint64_t>(rows.n, kSumRows);
    const uint32_t blocks = std::min(div_up(n_ch, kThreads), 1024u);
    if (rows.n > 0) {
        DRESSI_REQUIRE(gy && x && mean && rstd, "layer_norm_bwd: bad arguments");
        DRESSI_REQUIRE(((uintptr_t)gy | (uintptr_t)x | (uintptr_t)gx) % type_bytes(type) == 0,
                       "layer_norm_bwd: not aligned to its type");
        DRESSI_REQUIRE(scratch && scratch_bytes >= dressi_layer_norm_scratch(type, n_items, n_px,
                                                                             n_ch, 1),
                       "layer_norm_bwd: scratch too small");
        const int rc = for_type(type, [&](auto* t) -> int {
            using T = std::remove_pointer_t<decltype(t)>;
            if (gx) {
                hipLaunchKernelGGL((k_ln_backward<T>), dim3(grid_of(rows.n)), dim3(kThreads), 0,
                                   ctx->stream, (const T*)gy, (const T*)x, rows, aff, activation,
                                   mean, rstd, (T*)gx);
                DRESSI_CHECK_LAUNCH();
            }
            if (gw || gb) {
                hipLaunchKernelGGL((k_ln_sums<T>), dim3(shares, blocks), dim3(kThreads), 0,
                                   ctx->stream, (const T*)gy, (const T*)x, rows, aff, activation,
                                   mean, rstd, (float*)scratch);
                DRESSI_CHECK_LAUNCH();
            }
            return DRESSI_OK;
        });
        if (rc) {
            return rc;
        }
    }
    if (gw || gb) {
        hipLaunchKernelGGL(k_ln_params, dim3(blocks), dim3(kThreads), 0, ctx->stream,
                           (const float*)scratch, shares, n_ch, affine_type, gw, gb);
        DRESSI_CHECK_LAUNCH();
    }
    return DRESSI_OK;
}

}  // extern "C"
