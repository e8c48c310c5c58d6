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
//
// Memory bounds it: about 12 operations a value forward and 20 backward, 5 (with
// gelu 20) of them an exponential's. So a row is read once and held in registers
// until its sums are known: by a few lanes of a wave, by a wave, or by a
// workgroup, as its length asks; only rows beyond a workgroup's registers are
// read twice. A lane holds vectors of 16 bytes wherever they begin (rows of an
// odd number of channels need no narrower ones), and a row's last vector, where
// it would end past the row, is moved back into it: its first values are the
// vector's before, count once in the sums, and are written twice with the same
// bits.
//
// The mean is taken twice: of x, then of x less that, whose sum comes with that
// of the squares. So a mean many deviations from zero is as exact as a float can
// be, and the variance is that about it.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "internal.h"
#include "norm_core.h"
#include "typed.h"

namespace dressi {
namespace {

constexpr uint32_t kThreads = 256;  // of a workgroup that takes several rows

// Where rows lie: n_px to an item.
struct Rows {
    uint64_t n, n_px;
    uint64_t item_stride, px_stride;  // of x, in elements
    uint32_t n_ch;
    float inv;  // 1 / n_ch
    __device__ __forceinline__ size_t at(uint64_t row) const {
        if (n_px == n) {
            return (size_t)(row * px_stride);
        }
        const uint64_t item = row / n_px;
        return (size_t)(item * item_stride + (row - item * n_px) * px_stride);
    }
};

// Vector `vec` of a row: where it begins, and how many of its values count in
// the vector before (all, past the end).
template <int V>
struct Span {
    uint32_t first, skip;
    __device__ __forceinline__ Span(uint32_t vec, uint32_t n_ch) {
        const uint32_t at = vec * V;
        first = at + V <= n_ch ? at : n_ch - V;
        skip = at - first < V ? at - first : V;
    }
};

// x where value j counts, else 0. WHOLE: all do.
template <bool WHOLE>
__device__ __forceinline__ float counted(float x, uint32_t j, uint32_t skip) {
    return WHOLE || j >= skip ? x : 0.f;
}

template <int V>
__device__ __forceinline__ void load_params(const void* p, uint32_t type, uint32_t ch, float absent,
                                            float (&w)[V]) {
    if (!p) {
#pragma unroll
        for (int j = 0; j < V; j++) {
            w[j] = absent;
        }
    } else if (type == DRESSI_F32) {
        unpack(load_loose<float, V>((const float*)p + ch), w);
    } else if (type == DRESSI_BF16) {
        unpack(load_loose<bf16, V>((const bf16*)p + ch), w);
    } else {
        unpack(load_loose<f16, V>((const f16*)p + ch), w);
    }
}

// The sum over L lanes side by side, in each of them.
template <uint32_t L>
__device__ __forceinline__ float lane_sum(float x) {
    const auto dpp = [](float v, auto c) {
        return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), decltype(c)::value, 0xf,
                                                       0xf, true));
    };
    if constexpr (L >= 2) {
        x += dpp(x, std::integral_constant<int, 0xb1>());  // lane ^ 1
    }
    if constexpr (L >= 4) {
        x += dpp(x, std::integral_constant<int, 0x4e>());  // lane ^ 2
    }
    if constexpr (L >= 8) {
        x += dpp(x, std::integral_constant<int, 0x141>());  // 7 - lane
    }
    if constexpr (L >= 16) {
        x += dpp(x, std::integral_constant<int, 0x140>());  // 15 - lane
    }
    if constexpr (L >= 32) {
        const uint32_t u = __float_as_uint(x);
        const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if constexpr (L >= 64) {
        const uint32_t u = __float_as_uint(x);
        const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return x;
}

// The sum over a workgroup, in all threads, through part[waves]: one barrier, so
// that the next sum goes through another part.
__device__ __forceinline__ float wide_sum(float x, float* part) {
    x = lane_sum<64>(x);
    if ((threadIdx.x & 63u) == 0) {
        part[threadIdx.x >> 6] = x;
    }
    __syncthreads();
    const uint32_t waves = blockDim.x >> 6;
    x = part[0];
    for (uint32_t i = 1; i < waves; i++) {
        x += part[i];
    }
    return x;
}
__device__ __forceinline__ float2 wide_sum(float2 x, float2* part) {
    x = make_float2(lane_sum<64>(x.x), lane_sum<64>(x.y));
    if ((threadIdx.x & 63u) == 0) {
        part[threadIdx.x >> 6] = x;
    }
    __syncthreads();
    const uint32_t waves = blockDim.x >> 6;
    x = part[0];
    for (uint32_t i = 1; i < waves; i++) {
        x.x += part[i].x;
        x.y += part[i].y;
    }
    return x;
}

// 1 / deviation from the sums s of x - m and q of its squares, and the mean.
__device__ __forceinline__ float finish(float m, float s, float q, float inv, float eps,
                                        float& mean) {
    const float off = s * inv;
    mean = m + off;
    const float var = fmaf(-off, off, q * inv);
    return 1.f / sqrtf((var < 0.f ? 0.f : var) + eps);  // a NaN stays one
}

// y of a vector.
template <typename T, int V, bool STREAM>
__device__ __forceinline__ void write_y(const Pack<T, V>& x, float mean, float rstd,
                                        const float (&w)[V], const float (&b)[V], uint32_t act,
                                        T* y) {
    float z[V];
    unpack(x, z);
#pragma unroll
    for (int j = 0; j < V; j++) {
        z[j] = fmaf((z[j] - mean) * rstd, w[j], b[j]);
    }
    act_values<T, V>(act, z);
    store_loose<T, V, STREAM>(y, z);
}

struct Forward {
    const void* x;
    void* y;
    float* mean;  // or null, and rstd too
    float* rstd;
    Rows rows;
    Affine aff;
    float eps;
    uint32_t act;
};

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------

// Rows that a lane has in flight, of K vectors each.
template <int V, int K>
constexpr int kInFlight = K == 1 ? 4 : K == 2 ? 2 : 1;

// L lanes hold a row, K vectors each.
template <typename T, int V, int L, int K, bool WHOLE, bool STREAM>
__global__ __launch_bounds__(kThreads) void k_ln_rows(const Forward a) {
    constexpr int R = kInFlight<V, K>;
    constexpr uint32_t kSlots = kThreads / L;
    const uint32_t lane = threadIdx.x % L, slot = threadIdx.x / L;
    const Rows& rows = a.rows;
    uint32_t first[K], skip[K];
    float w[K][V], b[K][V];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const Span<V> sp(k * L + lane, rows.n_ch);
        first[k] = sp.first;
        skip[k] = sp.skip;
        load_params<V>(a.aff.weight, a.aff.type, sp.first, 1.f, w[k]);
        load_params<V>(a.aff.bias, a.aff.type, sp.first, 0.f, b[k]);
    }
    const T* x = (const T*)a.x;
    T* y = (T*)a.y;
    for (uint64_t r0 = (uint64_t)blockIdx.x * (kSlots * R); r0 < rows.n;
         r0 += (uint64_t)gridDim.x * (kSlots * R)) {
        Pack<T, V> v[R][K];
#pragma unroll
        for (int i = 0; i < R; i++) {
            const uint64_t row = r0 + i * kSlots + slot;
            const T* p = x + rows.at(row < rows.n ? row : rows.n - 1);
#pragma unroll
            for (int k = 0; k < K; k++) {
                v[i][k] = load_loose<T, V, STREAM>(p + first[k]);
            }
        }
        float m[R], s[R], q[R];
#pragma unroll
        for (int i = 0; i < R; i++) {
            m[i] = 0.f;
#pragma unroll
            for (int k = 0; k < K; k++) {
#pragma unroll
                for (int j = 0; j < V; j++) {
                    m[i] += counted<WHOLE>(to_float(v[i][k].v[j]), j, skip[k]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < R; i++) {
            m[i] = lane_sum<L>(m[i]) * rows.inv;
            s[i] = q[i] = 0.f;
#pragma unroll
            for (int k = 0; k < K; k++) {
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float d = counted<WHOLE>(to_float(v[i][k].v[j]) - m[i], j, skip[k]);
                    s[i] += d;
                    q[i] = fmaf(d, d, q[i]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < R; i++) {
            const uint64_t row = r0 + i * kSlots + slot;
            float mean;
            const float rstd = finish(m[i], lane_sum<L>(s[i]), lane_sum<L>(q[i]), rows.inv, a.eps,
                                      mean);
            if (row < rows.n) {
                T* out = y + row * rows.n_ch;
#pragma unroll
                for (int k = 0; k < K; k++) {
                    if (WHOLE || skip[k] < V) {
                        write_y<T, V, STREAM>(v[i][k], mean, rstd, w[k], b[k], a.act,
                                              out + first[k]);
                    }
                }
                if (lane == 0 && a.mean) {
                    a.mean[row] = mean;
                    a.rstd[row] = rstd;
                }
            }
        }
    }
}

// A workgroup holds a row, K vectors a thread. HOLD: weight and bias stay in
// registers between rows.
template <typename T, int V, int K, uint32_t THREADS, bool HOLD, bool WHOLE, bool STREAM>
__global__ __launch_bounds__(THREADS) void k_ln_wide(const Forward a) {
    __shared__ float part1[THREADS / 64];
    __shared__ float2 part2[THREADS / 64];
    const Rows& rows = a.rows;
    uint32_t first[K], skip[K];
    float w[K][V], b[K][V];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const Span<V> sp(k * blockDim.x + threadIdx.x, rows.n_ch);
        first[k] = sp.first;
        skip[k] = sp.skip;
        if (HOLD) {
            load_params<V>(a.aff.weight, a.aff.type, sp.first, 1.f, w[k]);
            load_params<V>(a.aff.bias, a.aff.type, sp.first, 0.f, b[k]);
        }
    }
    for (uint64_t row = blockIdx.x; row < rows.n; row += gridDim.x) {
        const T* p = (const T*)a.x + rows.at(row);
        Pack<T, V> v[K];
#pragma unroll
        for (int k = 0; k < K; k++) {
            v[k] = load_loose<T, V, STREAM>(p + first[k]);
        }
        float m = 0.f;
#pragma unroll
        for (int k = 0; k < K; k++) {
#pragma unroll
            for (int j = 0; j < V; j++) {
                m += counted<WHOLE>(to_float(v[k].v[j]), j, skip[k]);
            }
        }
        m = wide_sum(m, part1) * rows.inv;
        float2 s = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < K; k++) {
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float d = counted<WHOLE>(to_float(v[k].v[j]) - m, j, skip[k]);
                s.x += d;
                s.y = fmaf(d, d, s.y);
            }
        }
        s = wide_sum(s, part2);
        float mean;
        const float rstd = finish(m, s.x, s.y, rows.inv, a.eps, mean);
        T* out = (T*)a.y + row * rows.n_ch;
#pragma unroll
        for (int k = 0; k < K; k++) {
            if (WHOLE || skip[k] < V) {
                if (!HOLD) {
                    load_params<V>(a.aff.weight, a.aff.type, first[k], 1.f, w[k]);
                    load_params<V>(a.aff.bias, a.aff.type, first[k], 0.f, b[k]);
                }
                write_y<T, V, STREAM>(v[k], mean, rstd, w[k], b[k], a.act, out + first[k]);
            }
        }
        if (threadIdx.x == 0 && a.mean) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
    }
}

// Rows beyond a workgroup's registers go in chunks of kChunkVecs vectors, a
// workgroup each, in two passes: one leaves every chunk's (mean, squares about
// it), the other joins those of its row, every workgroup for itself.
constexpr uint32_t kChunkIter = 4;
constexpr uint32_t kChunkVecs = kChunkIter * kThreads;

// A thread's vectors of a chunk.
template <int V>
struct ChunkSpan {
    uint32_t first[kChunkIter], skip[kChunkIter], count;  // count: of the chunk
    __device__ __forceinline__ ChunkSpan(uint32_t chunk, uint32_t n_ch) {
#pragma unroll
        for (uint32_t k = 0; k < kChunkIter; k++) {
            const Span<V> sp(chunk * kChunkVecs + k * kThreads + threadIdx.x, n_ch);
            first[k] = sp.first;
            skip[k] = sp.skip;
        }
        count = std::min(n_ch - chunk * (kChunkVecs * V), kChunkVecs * V);
    }
};

template <typename T, int V>
__global__ __launch_bounds__(kThreads) void k_ln_chunk_stats(const Forward a, uint32_t chunks,
                                                             float2* part) {
    __shared__ float part1[kThreads / 64];
    __shared__ float2 part2[kThreads / 64];
    for (uint64_t u = blockIdx.x; u < a.rows.n * chunks; u += gridDim.x) {
        const uint64_t row = u / chunks;
        const ChunkSpan<V> sp((uint32_t)(u - row * chunks), a.rows.n_ch);
        const T* p = (const T*)a.x + a.rows.at(row);
        Pack<T, V> v[kChunkIter];
#pragma unroll
        for (uint32_t k = 0; k < kChunkIter; k++) {
            v[k] = load_loose<T, V>(p + sp.first[k]);
        }
        float m = 0.f;
#pragma unroll
        for (uint32_t k = 0; k < kChunkIter; k++) {
#pragma unroll
            for (int j = 0; j < V; j++) {
                m += counted<false>(to_float(v[k].v[j]), j, sp.skip[k]);
            }
        }
        const float inv = 1.f / (float)sp.count;
        m = wide_sum(m, part1) * inv;
        float2 s = make_float2(0.f, 0.f);
#pragma unroll
        for (uint32_t k = 0; k < kChunkIter; k++) {
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float d = counted<false>(to_float(v[k].v[j]) - m, j, sp.skip[k]);
                s.x += d;
                s.y = fmaf(d, d, s.y);
            }
        }
        s = wide_sum(s, part2);
        if (threadIdx.x == 0) {
            const float off = s.x * inv;
            part[u] = make_float2(m + off, fmaf(-off, s.x, s.y));
        }
    }
}

// A row's sums over its chunks' entries, in double, in all threads.
template <typename F>
__device__ __forceinline__ double2 join_chunks(const float2* part, uint32_t chunks, F&& f) {
    __shared__ double2 sums[kThreads / 64];
    double2 s = make_double2(0.0, 0.0);
    for (uint32_t i = threadIdx.x; i < chunks; i += kThreads) {
        f(i, part[i], s);
    }
    for (int o = 1; o < 64; o <<= 1) {
        s.x += __shfl_xor(s.x, o);
        s.y += __shfl_xor(s.y, o);
    }
    __syncthreads();  // those of before have been read
    if ((threadIdx.x & 63u) == 0) {
        sums[threadIdx.x >> 6] = s;
    }
    __syncthreads();
    s = sums[0];
    for (uint32_t i = 1; i < kThreads / 64; i++) {
        s.x += sums[i].x;
        s.y += sums[i].y;
    }
    return s;
}

template <typename T, int V>
__global__ __launch_bounds__(kThreads) void k_ln_chunk_apply(const Forward a, uint32_t chunks,
                                                             const float2* part) {
    const uint32_t n_ch = a.rows.n_ch;
    const double full = kChunkVecs * V, last = n_ch - (chunks - 1) * full;
    for (uint64_t u = blockIdx.x; u < a.rows.n * chunks; u += gridDim.x) {
        const uint64_t row = u / chunks;
        const ChunkSpan<V> sp((uint32_t)(u - row * chunks), n_ch);
        const T* p = (const T*)a.x + a.rows.at(row);
        Pack<T, V> v[kChunkIter];
#pragma unroll
        for (uint32_t k = 0; k < kChunkIter; k++) {
            v[k] = load_loose<T, V>(p + sp.first[k]);
        }
        // about the first chunk's mean: their difference loses nothing
        const float2* entries = part + row * chunks;
        const double pivot = (double)entries[0].x;
        const double2 s = join_chunks(entries, chunks, [&](uint32_t i, float2 e, double2& t) {
            const double n = i + 1 == chunks ? last : full, d = (double)e.x - pivot;
            t.x = fma(n, d, t.x);
            t.y += fma(n * d, d, (double)e.y);
        });
        const double d = s.x / n_ch, var = s.y / n_ch - d * d;
        const float mean = (float)(pivot + d);
        const float rstd = 1.f / sqrtf((float)(var < 0.0 ? 0.0 : var) + a.eps);
        T* out = (T*)a.y + row * n_ch;
#pragma unroll
        for (uint32_t k = 0; k < kChunkIter; k++) {
            if (sp.skip[k] < V) {
                float w[V], b[V];
                load_params<V>(a.aff.weight, a.aff.type, sp.first[k], 1.f, w);
                load_params<V>(a.aff.bias, a.aff.type, sp.first[k], 0.f, b);
                write_y<T, V, false>(v[k], mean, rstd, w, b, a.act, out + sp.first[k]);
            }
        }
        if (u == row * chunks && threadIdx.x == 0 && a.mean) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
    }
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------

struct Backward {
    const void* gy;
    const void* x;
    const float* mean;
    const float* rstd;
    void* gx;  // or null
    // of gw and gb: each workgroup's sums [2][n_ch] at a distance of part_stride,
    // or, where it is alone, the gradients themselves
    float* part;
    size_t part_stride;
    void* gw;
    void* gb;
    Rows rows;
    Affine aff;
    uint32_t act;
};

// xh and t = w gz of a vector, and gz added to the sums of a column.
template <typename T, int V>
__device__ __forceinline__ void slopes(const Pack<T, V>& xv, const Pack<T, V>& gv, float mean,
                                       float rstd, const float (&w)[V], const float (&b)[V],
                                       uint32_t act, float (&xh)[V], float (&t)[V], float (&gw)[V],
                                       float (&gb)[V]) {
    float z[V];
    unpack(xv, xh);
    unpack(gv, t);
#pragma unroll
    for (int j = 0; j < V; j++) {
        xh[j] = (xh[j] - mean) * rstd;
        z[j] = fmaf(xh[j], w[j], b[j]);
    }
    act_slopes<T, V>(act, z, t);
#pragma unroll
    for (int j = 0; j < V; j++) {
        gb[j] += t[j];
        gw[j] = fmaf(t[j], xh[j], gw[j]);
        t[j] *= w[j];
    }
}

template <int V, bool WHOLE>
__device__ __forceinline__ void add_row(const float (&xh)[V], const float (&t)[V], uint32_t skip,
                                        float2& s) {
#pragma unroll
    for (int j = 0; j < V; j++) {
        const float c = counted<WHOLE>(t[j], j, skip);
        s.x += c;
        s.y += counted<WHOLE>(t[j] * xh[j], j, skip);
    }
}

// gx of a vector, a and c the means of t and t xh.
template <typename T, int V, bool STREAM>
__device__ __forceinline__ void write_gx(const float (&xh)[V], const float (&t)[V], float rstd,
                                         float a, float c, T* gx) {
    float g[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        g[j] = rstd * ((t[j] - a) - xh[j] * c);
    }
    store_loose<T, V, STREAM>(gx, g);
}

__device__ __forceinline__ void write_sums(const Backward& a, uint32_t ch, float gw, float gb) {
    if (a.part) {
        float* p = a.part + blockIdx.x * a.part_stride;
        p[ch] = gw;
        p[a.rows.n_ch + ch] = gb;
        return;
    }
    if (a.gw) {
        store_one(a.gw, a.aff.type, ch, gw);
    }
    if (a.gb) {
        store_one(a.gb, a.aff.type, ch, gb);
    }
}

template <int V, int K>
constexpr int kInFlightBwd = K == 1 ? 2 : 1;

template <typename T, int V, int L, int K, bool WHOLE, bool STREAM>
__global__ __launch_bounds__(kThreads) void k_ln_bwd_rows(const Backward a) {
    constexpr int R = kInFlightBwd<V, K>;
    constexpr uint32_t kSlots = kThreads / L, kWaves = kThreads / 64;
    __shared__ float2 red[kWaves][L * K * V];
    const uint32_t lane = threadIdx.x % L, slot = threadIdx.x / L;
    const Rows& rows = a.rows;
    uint32_t first[K], skip[K];
    float w[K][V], b[K][V], gw[K][V], gb[K][V];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const Span<V> sp(k * L + lane, rows.n_ch);
        first[k] = sp.first;
        skip[k] = sp.skip;
        load_params<V>(a.aff.weight, a.aff.type, sp.first, 1.f, w[k]);
        load_params<V>(a.aff.bias, a.aff.type, sp.first, 0.f, b[k]);
#pragma unroll
        for (int j = 0; j < V; j++) {
            gw[k][j] = gb[k][j] = 0.f;
        }
    }
    const T* x = (const T*)a.x;
    const T* gy = (const T*)a.gy;
    T* gx = (T*)a.gx;
    for (uint64_t r0 = (uint64_t)blockIdx.x * (kSlots * R); r0 < rows.n;
         r0 += (uint64_t)gridDim.x * (kSlots * R)) {
        Pack<T, V> xv[R][K], gv[R][K];
        float mean[R], rstd[R];
#pragma unroll
        for (int i = 0; i < R; i++) {
            const uint64_t at = r0 + i * kSlots + slot, row = at < rows.n ? at : rows.n - 1;
            const T* p = x + rows.at(row);
            const T* q = gy + row * rows.n_ch;
            mean[i] = a.mean[row];
            rstd[i] = a.rstd[row];
#pragma unroll
            for (int k = 0; k < K; k++) {
                xv[i][k] = load_loose<T, V, STREAM>(p + first[k]);
                gv[i][k] = load_loose<T, V, STREAM>(q + first[k]);
            }
        }
#pragma unroll
        for (int i = 0; i < R; i++) {
            const uint64_t row = r0 + i * kSlots + slot;
            const bool live = row < rows.n;
            float xh[K][V], t[K][V];
            float2 s = make_float2(0.f, 0.f);
            if (live) {
#pragma unroll
                for (int k = 0; k < K; k++) {
                    slopes<T, V>(xv[i][k], gv[i][k], mean[i], rstd[i], w[k], b[k], a.act, xh[k],
                                 t[k], gw[k], gb[k]);
                    add_row<V, WHOLE>(xh[k], t[k], skip[k], s);
                }
            }
            s.x = lane_sum<L>(s.x) * rows.inv;
            s.y = lane_sum<L>(s.y) * rows.inv;
            if (live && gx) {
#pragma unroll
                for (int k = 0; k < K; k++) {
                    if (WHOLE || skip[k] < V) {
                        write_gx<T, V, STREAM>(xh[k], t[k], rstd[i], s.x, s.y,
                                               gx + row * rows.n_ch + first[k]);
                    }
                }
            }
        }
    }
    if (!a.part && !a.gw && !a.gb) {
        return;
    }
    // a column's sums over the slots: of a wave, then of the waves
    const uint32_t wave = threadIdx.x >> 6;
#pragma unroll
    for (int k = 0; k < K; k++) {
#pragma unroll
        for (int j = 0; j < V; j++) {
            for (int o = L; o < 64; o <<= 1) {
                gw[k][j] += __shfl_xor(gw[k][j], o);
                gb[k][j] += __shfl_xor(gb[k][j], o);
            }
            if ((threadIdx.x & 63u) < L) {
                red[wave][(k * V + j) * L + lane] = make_float2(gw[k][j], gb[k][j]);
            }
        }
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < L * K * V; e += kThreads) {
        const uint32_t vec = e / (L * V) * L + e % L, j = e / L % V;
        const Span<V> sp(vec, rows.n_ch);
        if (j >= sp.skip) {
            float2 s = red[0][e];
#pragma unroll
            for (uint32_t i = 1; i < kWaves; i++) {
                s.x += red[i][e].x;
                s.y += red[i][e].y;
            }
            write_sums(a, sp.first + j, s.x, s.y);
        }
    }
}

template <typename T, int V, int K, uint32_t THREADS, bool HOLD, bool WHOLE, bool STREAM>
__global__ __launch_bounds__(THREADS) void k_ln_bwd_wide(const Backward a) {
    __shared__ float2 part[2][THREADS / 64];
    const Rows& rows = a.rows;
    uint32_t first[K], skip[K];
    float w[K][V], b[K][V], gw[K][V], gb[K][V];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const Span<V> sp(k * blockDim.x + threadIdx.x, rows.n_ch);
        first[k] = sp.first;
        skip[k] = sp.skip;
        if (HOLD) {
            load_params<V>(a.aff.weight, a.aff.type, sp.first, 1.f, w[k]);
            load_params<V>(a.aff.bias, a.aff.type, sp.first, 0.f, b[k]);
        }
#pragma unroll
        for (int j = 0; j < V; j++) {
            gw[k][j] = gb[k][j] = 0.f;
        }
    }
    uint32_t turn = 0;
    for (uint64_t row = blockIdx.x; row < rows.n; row += gridDim.x, turn ^= 1) {
        const T* p = (const T*)a.x + rows.at(row);
        const T* q = (const T*)a.gy + row * rows.n_ch;
        const float mean = a.mean[row], rstd = a.rstd[row];
        Pack<T, V> xv[K], gv[K];
#pragma unroll
        for (int k = 0; k < K; k++) {
            xv[k] = load_loose<T, V, STREAM>(p + first[k]);
            gv[k] = load_loose<T, V, STREAM>(q + first[k]);
        }
        float xh[K][V], t[K][V];
        float2 s = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < K; k++) {
            if (!HOLD) {
                load_params<V>(a.aff.weight, a.aff.type, first[k], 1.f, w[k]);
                load_params<V>(a.aff.bias, a.aff.type, first[k], 0.f, b[k]);
            }
            slopes<T, V>(xv[k], gv[k], mean, rstd, w[k], b[k], a.act, xh[k], t[k], gw[k], gb[k]);
            add_row<V, WHOLE>(xh[k], t[k], skip[k], s);
        }
        s = wide_sum(s, part[turn]);
        if (a.gx) {
            T* out = (T*)a.gx + row * rows.n_ch;
#pragma unroll
            for (int k = 0; k < K; k++) {
                if (WHOLE || skip[k] < V) {
                    write_gx<T, V, STREAM>(xh[k], t[k], rstd, s.x * rows.inv, s.y * rows.inv,
                                           out + first[k]);
                }
            }
        }
    }
    if (!a.part && !a.gw && !a.gb) {
        return;
    }
#pragma unroll
    for (int k = 0; k < K; k++) {
#pragma unroll
        for (int j = 0; j < V; j++) {
            if (j >= skip[k]) {
                write_sums(a, first[k] + j, gw[k][j], gb[k][j]);
            }
        }
    }
}

// Longer rows, in chunks: a workgroup takes one chunk of every gridDim.x-th row.
// The first pass leaves the chunk's sums of t and t xh of each row, and the
// columns' over its rows.
template <typename T, int V>
__global__ __launch_bounds__(kThreads) void k_ln_bwd_chunk_sums(const Backward a, uint32_t chunks,
                                                                float2* row_part) {
    __shared__ float2 part[2][kThreads / 64];
    const Rows& rows = a.rows;
    const uint32_t chunk = blockIdx.y;
    const ChunkSpan<V> sp(chunk, rows.n_ch);
    float gw[kChunkIter][V], gb[kChunkIter][V];
#pragma unroll
    for (uint32_t k = 0; k < kChunkIter; k++) {
#pragma unroll
        for (int j = 0; j < V; j++) {
            gw[k][j] = gb[k][j] = 0.f;
        }
    }
    uint32_t turn = 0;
    for (uint64_t row = blockIdx.x; row < rows.n; row += gridDim.x, turn ^= 1) {
        const T* p = (const T*)a.x + rows.at(row);
        const T* q = (const T*)a.gy + row * rows.n_ch;
        const float mean = a.mean[row], rstd = a.rstd[row];
        float2 s = make_float2(0.f, 0.f);
#pragma unroll
        for (uint32_t k = 0; k < kChunkIter; k++) {
            float w[V], b[V], xh[V], t[V];
            load_params<V>(a.aff.weight, a.aff.type, sp.first[k], 1.f, w);
            load_params<V>(a.aff.bias, a.aff.type, sp.first[k], 0.f, b);
            slopes<T, V>(load_loose<T, V>(p + sp.first[k]), load_loose<T, V>(q + sp.first[k]), mean,
                         rstd, w, b, a.act, xh, t, gw[k], gb[k]);
            add_row<V, false>(xh, t, sp.skip[k], s);
        }
        s = wide_sum(s, part[turn]);
        if (threadIdx.x == 0) {
            row_part[row * chunks + chunk] = s;
        }
    }
    if (!a.part && !a.gw && !a.gb) {
        return;
    }
#pragma unroll
    for (uint32_t k = 0; k < kChunkIter; k++) {
#pragma unroll
        for (int j = 0; j < V; j++) {
            if (j >= sp.skip[k]) {
                write_sums(a, sp.first[k] + j, gw[k][j], gb[k][j]);
            }
        }
    }
}

template <typename T, int V>
__global__ __launch_bounds__(kThreads) void k_ln_bwd_chunk_apply(const Backward a, uint32_t chunks,
                                                                 const float2* row_part) {
    const uint32_t n_ch = a.rows.n_ch;
    for (uint64_t u = blockIdx.x; u < a.rows.n * chunks; u += gridDim.x) {
        const uint64_t row = u / chunks;
        const ChunkSpan<V> sp((uint32_t)(u - row * chunks), n_ch);
        const T* p = (const T*)a.x + a.rows.at(row);
        const T* q = (const T*)a.gy + row * n_ch;
        const float mean = a.mean[row], rstd = a.rstd[row];
        const double2 s = join_chunks(row_part + row * chunks, chunks,
                                      [](uint32_t, float2 e, double2& t) {
                                          t.x += (double)e.x;
                                          t.y += (double)e.y;
                                      });
        const float ma = (float)(s.x / n_ch), mc = (float)(s.y / n_ch);
#pragma unroll
        for (uint32_t k = 0; k < kChunkIter; k++) {
            if (sp.skip[k] < V) {
                float w[V], b[V], xh[V], t[V], gw[V] = {}, gb[V] = {};
                load_params<V>(a.aff.weight, a.aff.type, sp.first[k], 1.f, w);
                load_params<V>(a.aff.bias, a.aff.type, sp.first[k], 0.f, b);
                slopes<T, V>(load_loose<T, V>(p + sp.first[k]), load_loose<T, V>(q + sp.first[k]),
                             mean, rstd, w, b, a.act, xh, t, gw, gb);
                write_gx<T, V, false>(xh, t, rstd, ma, mc, (T*)a.gx + row * n_ch + sp.first[k]);
            }
        }
    }
}

// Adds the workgroups' sums of gw and gb, in their order: 16 columns of the
// 2 n_ch a workgroup, four a lane, over 256 lanes. n 0: sums of nothing.
constexpr uint32_t kParamThreads = 1024, kParamCols = 16;

__global__ __launch_bounds__(kParamThreads) void k_ln_params(const float* part, size_t stride,
                                                             uint32_t n, uint32_t n_ch,
                                                             uint32_t type, void* gw, void* gb) {
    __shared__ float red[kParamThreads / 64][kParamCols];
    const uint32_t col = threadIdx.x & 3u, r0 = threadIdx.x >> 2;
    const uint32_t c0 = blockIdx.x * kParamCols + col * 4;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (c0 < 2 * n_ch) {  // the stride is a multiple of four
#pragma unroll 4
        for (uint32_t r = r0; r < n; r += kParamThreads / 4) {
            float v[4];
            load_vec<float, 4>(part + r * stride + c0, v);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                s[j] += v[j];
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
        for (int o = 4; o < 64; o <<= 1) {
            s[j] += __shfl_xor(s[j], o);
        }
        if ((threadIdx.x & 63u) < 4) {
            red[threadIdx.x >> 6][col * 4 + j] = s[j];
        }
    }
    __syncthreads();
    const uint32_t c = blockIdx.x * kParamCols + threadIdx.x;
    if (threadIdx.x >= kParamCols || c >= 2 * n_ch) {
        return;
    }
    float sum = red[0][threadIdx.x];
    for (uint32_t i = 1; i < kParamThreads / 64; i++) {
        sum += red[i][threadIdx.x];
    }
    if (c < n_ch && gw) {
        store_one(gw, type, c, sum);
    } else if (c >= n_ch && gb) {
        store_one(gb, type, c - n_ch, sum);
    }
}

// ---------------------------------------------------------------------------
// how a call is cut
// ---------------------------------------------------------------------------

// A type's vectors, and a single value where a row is shorter.
constexpr uint32_t vec_of(uint32_t type, uint32_t n_ch) {
    const uint32_t v = type == DRESSI_F32 ? 4 : 8;
    return n_ch >= v ? v : 1;
}

// Vectors of a row up to which a wave, then a workgroup of 1024, holds it, forward and backward.
constexpr uint32_t kWaveVecs = 256, kWaveVecsBwd = 128;
constexpr uint32_t kHoldElems = 32768, kHoldElemsBwd = 16384;

// Bytes of results from which they go past the caches.
constexpr uint64_t kStreamBytes = 32ull << 20;

struct Plan {
    uint32_t v, vecs;  // of a row
    bool chunked, wide, whole, stream;
    uint32_t lanes, iter;  // of a row; wide: lanes = the workgroup's threads
    uint32_t chunks;       // of a row
    uint32_t groups;       // workgroups whose sums of gw and gb are added
};

Plan make_plan(uint32_t type, uint64_t rows, uint32_t n_ch, bool backward) {
    Plan p{};
    p.v = vec_of(type, n_ch);
    p.vecs = div_up(n_ch, p.v);
    p.stream = rows * n_ch * type_bytes(type) >= kStreamBytes;
    const uint32_t most = backward ? kWaveVecsBwd : kWaveVecs;
    if (n_ch > (backward ? kHoldElemsBwd : kHoldElems)) {
        p.chunked = true;
        p.chunks = div_up(p.vecs, kChunkVecs);
        p.groups = (uint32_t)std::min<uint64_t>(rows, std::max(1u, 1024 / p.chunks));
    } else if (p.vecs > most) {
        p.wide = true;
        const uint32_t elems = backward ? 16 : 32;  // a thread's at most
        p.iter = 1;
        while (p.iter * p.v < elems && p.vecs > p.iter * 256) {
            p.iter *= 2;
        }
        p.lanes = div_up(div_up(p.vecs, p.iter), 64) * 64;
        p.whole = n_ch == p.lanes * p.iter * p.v;
        p.groups = (uint32_t)std::min<uint64_t>(rows, 512);
    } else {
        p.lanes = 1;
        while (p.lanes < 64 && p.lanes < p.vecs) {
            p.lanes *= 2;
        }
        p.iter = 1;
        while (p.iter * p.lanes < p.vecs) {
            p.iter *= 2;
        }
        p.whole = n_ch == p.lanes * p.iter * p.v;
        const uint64_t slots = kThreads / p.lanes * (p.iter == 1 ? 2 : 1);
        p.groups = (uint32_t)std::min<uint64_t>((rows + slots - 1) / slots, 1024);
    }
    return p;
}

size_t part_stride(uint32_t n_ch) { return (2 * (size_t)n_ch + 3) / 4 * 4; }

// Bytes of the chunks' sums, and of the workgroups' of gw and gb after them.
size_t row_bytes(const Plan& p, uint64_t rows) {
    return p.chunked ? (rows * p.chunks * sizeof(float2) + 15) / 16 * 16 : 0;
}
size_t scratch_bytes_of(const Plan& p, uint64_t rows, uint32_t n_ch, bool backward) {
    const size_t sums = backward && p.groups > 1 ? p.groups * part_stride(n_ch) * sizeof(float) : 0;
    return row_bytes(p, rows) + sums;
}

template <typename A>
int launch(void (*kernel)(A), uint32_t grid, uint32_t threads, hipStream_t s, const A& a) {
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(threads), 0, s, a);
    DRESSI_CHECK_LAUNCH();
    return DRESSI_OK;
}

// f(integral_constant)s of a truth value, and of a power of two up to MOST.
template <typename F>
auto for_bool(bool x, F&& f) {
    return x ? f(std::true_type()) : f(std::false_type());
}
template <int MOST, int LEAST = 1, typename F>
int for_power(uint32_t x, F&& f) {
    if constexpr (LEAST < MOST) {
        if (x > LEAST) {
            return for_power<MOST, LEAST * 2>(x, f);
        }
    }
    return f(std::integral_constant<int, LEAST>());
}

template <typename T, int V>
int forward(hipStream_t s, const Plan& p, const Forward& a, void* scratch) {
    const uint64_t n = a.rows.n;
    if (p.chunked) {
        const uint32_t grid = (uint32_t)std::min<uint64_t>(n * p.chunks, 1u << 20);
        hipLaunchKernelGGL((k_ln_chunk_stats<T, V>), dim3(grid), dim3(kThreads), 0, s, a, p.chunks,
                           (float2*)scratch);
        DRESSI_CHECK_LAUNCH();
        hipLaunchKernelGGL((k_ln_chunk_apply<T, V>), dim3(grid), dim3(kThreads), 0, s, a, p.chunks,
                           (const float2*)scratch);
        DRESSI_CHECK_LAUNCH();
        return DRESSI_OK;
    }
    return for_bool(p.whole, [&](auto whole) {
        return for_bool(p.stream, [&](auto stream) {
            constexpr bool W = decltype(whole)::value, S = decltype(stream)::value;
            if constexpr (V > 1) {
                if (p.wide) {
                    const uint32_t grid = (uint32_t)std::min<uint64_t>(n, 256 * (2048 / p.lanes));
                    return for_power<32 / V, 2>(p.iter, [&](auto iter) {
                        constexpr int K = decltype(iter)::value;
                        return p.lanes <= 256
                                   ? launch(k_ln_wide<T, V, K, 256, true, W, S>, grid, p.lanes, s, a)
                                   : launch(k_ln_wide<T, V, K, 1024, false, W, S>, grid, p.lanes, s, a);
                    });
                }
                if (p.lanes == 64 && p.iter > 1) {
                    return for_power<4, 2>(p.iter, [&](auto iter) {
                        constexpr int K = decltype(iter)::value;
                        const uint64_t take = kThreads / 64 * kInFlight<V, K>;
                        return launch(k_ln_rows<T, V, 64, K, W, S>,
                                      (uint32_t)std::min<uint64_t>((n + take - 1) / take, 2048),
                                      kThreads, s, a);
                    });
                }
            }
            return for_power<(V > 1 ? 64 : 8)>(p.lanes, [&](auto lanes) {
                constexpr int L = decltype(lanes)::value;
                const uint64_t take = kThreads / L * kInFlight<V, 1>;
                return launch(k_ln_rows<T, V, L, 1, W, S>,
                              (uint32_t)std::min<uint64_t>((n + take - 1) / take, 2048), kThreads,
                              s, a);
            });
        });
    });
}

template <typename T, int V>
int backward(hipStream_t s, const Plan& p, const Backward& a, float2* row_part) {
    const uint64_t n = a.rows.n;
    if (p.chunked) {
        hipLaunchKernelGGL((k_ln_bwd_chunk_sums<T, V>), dim3(p.groups, p.chunks), dim3(kThreads), 0,
                           s, a, p.chunks, row_part);
        DRESSI_CHECK_LAUNCH();
        if (a.gx) {
            hipLaunchKernelGGL((k_ln_bwd_chunk_apply<T, V>),
                               dim3((uint32_t)std::min<uint64_t>(n * p.chunks, 1u << 20)),
                               dim3(kThreads), 0, s, a, p.chunks, (const float2*)row_part);
            DRESSI_CHECK_LAUNCH();
        }
        return DRESSI_OK;
    }
    return for_bool(p.whole, [&](auto whole) {
        return for_bool(p.stream, [&](auto stream) {
            constexpr bool W = decltype(whole)::value, S = decltype(stream)::value;
            if constexpr (V > 1) {
                if (p.wide) {
                    return for_power<16 / V>(p.iter, [&](auto iter) {
                        constexpr int K = decltype(iter)::value;
                        return p.lanes <= 256
                                   ? launch(k_ln_bwd_wide<T, V, K, 256, true, W, S>, p.groups,
                                            p.lanes, s, a)
                                   : launch(k_ln_bwd_wide<T, V, K, 1024, false, W, S>, p.groups,
                                            p.lanes, s, a);
                    });
                }
                if (p.lanes == 64 && p.iter == 2) {
                    return launch(k_ln_bwd_rows<T, V, 64, 2, W, S>, p.groups, kThreads, s, a);
                }
            }
            return for_power<(V > 1 ? 64 : 8)>(p.lanes, [&](auto lanes) {
                return launch(k_ln_bwd_rows<T, V, decltype(lanes)::value, 1, W, S>, p.groups,
                              kThreads, s, a);
            });
        });
    });
}

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

Rows make_rows(uint64_t n_items, uint64_t n_px, uint32_t n_ch, uint64_t item_stride,
               uint64_t px_stride) {
    Rows r{n_items * n_px, n_px, item_stride, px_stride, n_ch, 1.f / (float)n_ch};
    if (n_px == 1) {
        r.px_stride = item_stride;
    }
    if (n_items == 1 || n_px == 1 || item_stride == n_px * px_stride) {
        r.n_px = r.n;
    }
    return r;
}

// f(a vector's type)
template <typename F>
int for_vec(uint32_t type, uint32_t v, F&& f) {
    switch (type) {
        case DRESSI_F32:
            return v == 1 ? f(Pack<float, 1>()) : f(Pack<float, 4>());
        case DRESSI_BF16:
            return v == 1 ? f(Pack<bf16, 1>()) : f(Pack<bf16, 8>());
        default:
            return v == 1 ? f(Pack<f16, 1>()) : f(Pack<f16, 8>());
    }
}

}  // namespace
}  // namespace dressi

using namespace dressi;

extern "C" {

size_t dressi_layer_norm_scratch(uint32_t type, uint64_t n_items, uint64_t n_px, uint32_t n_ch,
                                 int backward) {
    if (type > DRESSI_F16 || n_ch == 0 || n_items == 0 || n_px == 0) {
        return 0;
    }
    const uint64_t rows = n_items * n_px;
    return scratch_bytes_of(make_plan(type, rows, n_ch, backward != 0), rows, n_ch, backward != 0);
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
    const Rows rows = make_rows(n_items, n_px, n_ch, item_stride, px_stride);
    const Plan p = make_plan(type, rows.n, n_ch, false);
    const size_t need = scratch_bytes_of(p, rows.n, n_ch, false);
    DRESSI_REQUIRE(need == 0 || (scratch && ((uintptr_t)scratch & 15) == 0 && scratch_bytes >= need),
                   "layer_norm: scratch too small or not aligned");
    const DeviceScope scope(ctx->device);
    DRESSI_TRY_HIP(scope.error());
    const Forward a{x, y, mean, rstd, rows, aff, eps, activation};
    return for_vec(type, p.v, [&](auto w) {
        using T = std::remove_reference_t<decltype(w.v[0])>;
        return forward<T, sizeof(w) / sizeof(T)>(ctx->stream, p, a, scratch);
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
    const Rows rows = make_rows(n_items, n_px, n_ch, item_stride, px_stride);
    const Plan p = make_plan(type, rows.n, n_ch, true);
    const bool params = gw || gb, join = params && p.groups != 1;
    float* part = join ? (float*)((char*)scratch + row_bytes(p, rows.n)) : nullptr;
    const DeviceScope scope(ctx->device);
    if (rows.n > 0) {
        DRESSI_REQUIRE(gy && x && mean && rstd, "layer_norm_bwd: bad arguments");
        DRESSI_REQUIRE(((uintptr_t)gy | (uintptr_t)x | (uintptr_t)gx) % type_bytes(type) == 0,
                       "layer_norm_bwd: not aligned to its type");
        const size_t need = scratch_bytes_of(p, rows.n, n_ch, true);
        DRESSI_REQUIRE(
            need == 0 || (scratch && ((uintptr_t)scratch & 15) == 0 && scratch_bytes >= need),
            "layer_norm_bwd: scratch too small or not aligned");
        DRESSI_TRY_HIP(scope.error());
        const Backward a{gy, x, mean, rstd, gx, part, part_stride(n_ch),
                         join ? nullptr : gw, join ? nullptr : gb, rows, aff, activation};
        const int rc = for_vec(type, p.v, [&](auto w) {
            using T = std::remove_reference_t<decltype(w.v[0])>;
            return backward<T, sizeof(w) / sizeof(T)>(ctx->stream, p, a, (float2*)scratch);
        });
        if (rc) {
            return rc;
        }
    }
    if (join) {
        hipLaunchKernelGGL(k_ln_params, dim3(div_up(2 * n_ch, kParamCols)), dim3(kParamThreads), 0,
                           ctx->stream, part, part_stride(n_ch), p.groups, n_ch, affine_type, gw,
                           gb);
        DRESSI_CHECK_LAUNCH();
    }
    return DRESSI_OK;
}

}  // extern "C"
