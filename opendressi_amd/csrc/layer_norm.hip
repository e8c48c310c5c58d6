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
// Memory bounds it, with 20 operations a value forward and 28 backward (silu; a
// compute unit has 26 and 39 for each that the memory brings it, in 16 bits): gelu
// alone takes longer than that. So a row is read once and held in registers
// until its sums are known: by a few lanes of a wave, by a wave, or by a
// workgroup, as its length asks; only rows beyond a workgroup's registers are
// read twice. A lane holds vectors of 16 bytes wherever they begin (rows of an
// odd number of channels need no narrower ones), and a row's last vector, where
// it would end past the row, is moved back into it: its first values are the
// vector's before, count once in the sums, and are written twice with the same
// bits.
//
// The squares are those of x less the mean, from registers, so values far from
// zero lose no more than the mean's own rounding. Backward takes the mean and the
// deviation that forward left, and computes z as it did: relu masks what y says.
//
// The times beside the choices below are those of graphs of some calls, replayed,
// both sides in turn, statistics written; from 48 MB of x on over inputs that are
// others each time, 768 MB of x and as much of gy in all, for over the same ones
// again a cache may hold a part (16384 x 4096 bfloat16 forward 45 us in place of
// 54).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <initializer_list>

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
    uint32_t flat;  // rows are evenly spaced, and a workgroup's within 2^32 bytes
    float inv;      // 1 / n_ch
    __device__ __forceinline__ size_t at(uint64_t row) const {
        if (n_px == n) {
            return (size_t)(row * px_stride);
        }
        const uint64_t item = n <= 0xffffffffu ? (uint32_t)row / (uint32_t)n_px : row / n_px;
        return (size_t)(item * item_stride + (row - item * n_px) * px_stride);
    }
};
constexpr uint64_t kMaxPxStride = 1ull << 22;  // elements, of up to 256 rows

// The element at a distance in bytes.
template <typename T>
__device__ __forceinline__ T* at_byte(T* p, uint32_t bytes) {
    return (T*)((char*)p + bytes);
}
template <typename T>
__device__ __forceinline__ const T* at_byte(const T* p, uint32_t bytes) {
    return (const T*)((const char*)p + bytes);
}

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

template <typename T, int V>
__device__ __forceinline__ void load_floats(const void* p, uint32_t ch, float* w) {
    float x[V];
    unpack(load_loose<T, V>((const T*)p + ch), x);
#pragma unroll
    for (int j = 0; j < V; j++) {
        w[j] = x[j];
    }
}
// V of the weight's or bias's values.
template <int V>
__device__ __forceinline__ void load_params(const void* p, uint32_t type, uint32_t ch, float absent,
                                            float* w) {
    if (!p) {
#pragma unroll
        for (int j = 0; j < V; j++) {
            w[j] = absent;
        }
    } else if (type == DRESSI_F32) {
        load_floats<float, V>(p, ch, w);
    } else if (type == DRESSI_BF16) {
        load_floats<bf16, V>(p, ch, w);
    } else {
        load_floats<f16, V>(p, ch, w);
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

// The sum over `waves` waves of a workgroup from `first` on, in all threads,
// through part[]: one barrier, so that the next sum goes through another part.
__device__ __forceinline__ float wide_sum(float x, float* part, uint32_t waves) {
    x = lane_sum<64>(x);
    if ((threadIdx.x & 63u) == 0) {
        part[threadIdx.x >> 6] = x;
    }
    __syncthreads();
    x = part[0];
    for (uint32_t i = 1; i < waves; i++) {
        x += part[i];
    }
    return x;
}
__device__ __forceinline__ float2 wide_sum(float2 x, float2* part, uint32_t first, uint32_t waves) {
    x = make_float2(lane_sum<64>(x.x), lane_sum<64>(x.y));
    if ((threadIdx.x & 63u) == 0) {
        part[threadIdx.x >> 6] = x;
    }
    __syncthreads();
    x = part[first];
    for (uint32_t i = first + 1; i < first + waves; i++) {
        x.x += part[i].x;
        x.y += part[i].y;
    }
    return x;
}

// 1 / sqrt(v) to less than a step of a float: the hardware's, refined once.
__device__ __forceinline__ float inv_sqrt(float v) {
    if (!(v >= 0x1p-100f && v <= 0x1p100f)) {
        return 1.f / sqrtf(v);  // zero, an infinity, a NaN, and what the steps below lose
    }
    const float r = __builtin_amdgcn_rsqf(v);
    return fmaf(0.5f * r, fmaf(-v * r, r, 1.f), r);
}

// f(whether past the caches), in two branches that the compiler keeps apart: it
// would make one of them, through the caches, out of loads or stores that differ
// in that alone.
template <typename F>
__device__ __forceinline__ void by_stream(bool stream, F&& f) {
    if (stream) {
        asm volatile("");
        f(std::true_type());
        asm volatile("");
    } else {
        f(std::false_type());
    }
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
    bool stream, stream_in;
};

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------

// Whether a wave's load is one piece of memory, or long pieces, and may go past
// the caches: in short ones it would read lines again (3000000 x 130 bfloat16, three
// vectors each by eight lanes, 456 us, through the caches 433).
template <int L, int K>
constexpr bool kLongPieces = K == 1 || L >= 32;

// Rows that a lane has in flight, of E values each: 64 bytes (500000 x 400 float32,
// gelu, 8 values a lane: 287 us, 318 with 128 bytes).
template <typename T, int E>
constexpr int kInFlight = E * sizeof(T) >= 48 ? 1 : E * sizeof(T) >= 32 ? 2 : 4;

// L lanes hold a row, K vectors each. 8 x 1024 x 1024 x 64 bfloat16, silu, without
// statistics: 358 us, 6.0 TB/s; 64 of 96 channels of 512 x 512: 14.0, whose lines
// hold half as much again; 2000000 x 24 float32 65, 5.9 TB/s; one row 3. Gelu's
// arithmetic is what bounds it in 16 bits (4194304 x 64: 227 us, silu 175).
template <typename T, int V, int L, int K, bool WHOLE>
__global__ __launch_bounds__(kThreads) void k_ln_rows(const Forward a) {
    constexpr int E = K * V, R = kInFlight<T, E>;
    constexpr uint32_t kSlots = kThreads / L, kTake = kSlots * R;
    const uint32_t lane = threadIdx.x % L, slot = threadIdx.x / L;
    const Rows& rows = a.rows;
    const uint32_t px_bytes = (uint32_t)(rows.px_stride * sizeof(T));
    uint32_t first[K], skip[K];  // first: in bytes
    float w[E], b[E];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const Span<V> sp(k * L + lane, rows.n_ch);
        first[k] = sp.first * sizeof(T);
        skip[k] = sp.skip;
        load_params<V>(a.aff.weight, a.aff.type, sp.first, 1.f, w + k * V);
        load_params<V>(a.aff.bias, a.aff.type, sp.first, 0.f, b + k * V);
    }
    const uint32_t in = slot * px_bytes, out = slot * rows.n_ch * sizeof(T);
    const uint64_t step = (uint64_t)gridDim.x * kTake;
    for (uint64_t r0 = (uint64_t)blockIdx.x * kTake; r0 < rows.n; r0 += step) {
        const T* x = (const T*)a.x;
        Pack<T, V> v[R][K];
        if (rows.flat && r0 + kTake <= rows.n) {
            x += r0 * rows.px_stride;
            by_stream(kLongPieces<L, K> && a.stream_in, [&](auto past) {
#pragma unroll
                for (int i = 0; i < R; i++) {
#pragma unroll
                    for (int k = 0; k < K; k++) {
                        v[i][k] = load_loose<T, V, decltype(past)::value>(
                            at_byte(x + (size_t)(i * kSlots) * rows.px_stride, in + first[k]));
                    }
                }
            });
        } else {  // past the end the last row again
#pragma unroll
            for (int i = 0; i < R; i++) {
                const T* p = x + rows.at(std::min(r0 + i * kSlots + slot, rows.n - 1));
#pragma unroll
                for (int k = 0; k < K; k++) {
                    v[i][k] = load_loose<T, V>(at_byte(p, first[k]));
                }
            }
        }
        float z[R][E], m[R], q[R];
#pragma unroll
        for (int i = 0; i < R; i++) {
            m[i] = 0.f;
#pragma unroll
            for (int e = 0; e < E; e++) {
                z[i][e] = to_float(v[i][e / V].v[e % V]);
                m[i] += counted<WHOLE>(z[i][e], e % V, skip[e / V]);
            }
        }
#pragma unroll
        for (int i = 0; i < R; i++) {
            m[i] = lane_sum<L>(m[i]) * rows.inv;
            q[i] = 0.f;
#pragma unroll
            for (int e = 0; e < E; e++) {
                z[i][e] -= m[i];
                const float d = counted<WHOLE>(z[i][e], e % V, skip[e / V]);
                q[i] = fmaf(d, d, q[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < R; i++) {
            q[i] = inv_sqrt(fmaf(lane_sum<L>(q[i]), rows.inv, a.eps));
#pragma unroll
            for (int e = 0; e < E; e++) {
                z[i][e] = fmaf(z[i][e] * q[i], w[e], b[e]);
            }
        }
        act_values<T, R * E>(a.act, *(float (*)[R * E])&z[0][0]);
        T* y = (T*)a.y + r0 * rows.n_ch;
        by_stream(a.stream, [&](auto past) {
#pragma unroll
            for (int i = 0; i < R; i++) {
                if (r0 + i * kSlots + slot < rows.n) {
                    T* yi = y + (size_t)(i * kSlots) * rows.n_ch;
#pragma unroll
                    for (int k = 0; k < K; k++) {
                        if (WHOLE || skip[k] < V) {
                            store_loose<T, V, decltype(past)::value>(at_byte(yi, out + first[k]),
                                                                     z[i] + k * V);
                        }
                    }
                }
            }
        });
        if (lane == 0 && a.mean) {
#pragma unroll
            for (int i = 0; i < R; i++) {
                if (r0 + i * kSlots + slot < rows.n) {
                    (a.mean + r0 + i * kSlots)[slot] = m[i];
                    (a.rstd + r0 + i * kSlots)[slot] = q[i];
                }
            }
        }
    }
}

// A workgroup holds a row, K vectors a thread. HOLD: weight and bias stay in
// registers between rows. 16384 x 4096 bfloat16: 54 us, 4.9 TB/s; 4096 x 16384
// float32, which waits for its barriers with few workgroups: 105, 5.1 TB/s. 1024
// threads with 16 values are held to 64 registers, so that a compute unit has two
// workgroups of them (4000 x 15000 bfloat16 63 us, 71 without).
template <typename T, int V, int K, uint32_t THREADS, bool HOLD, bool WHOLE>
__global__ __launch_bounds__(THREADS, THREADS == 1024 && K * V == 16 ? 8 : 1) void k_ln_wide(
    const Forward a) {
    __shared__ float part[2][THREADS / 64];
    constexpr int E = K * V;
    const Rows& rows = a.rows;
    uint32_t first[K], skip[K];
    float w[E], b[E];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const Span<V> sp(k * blockDim.x + threadIdx.x, rows.n_ch);
        first[k] = sp.first;
        skip[k] = sp.skip;
        if (HOLD) {
            load_params<V>(a.aff.weight, a.aff.type, sp.first, 1.f, w + k * V);
            load_params<V>(a.aff.bias, a.aff.type, sp.first, 0.f, b + k * V);
        }
    }
    for (uint64_t row = blockIdx.x; row < rows.n; row += gridDim.x) {
        const T* p = (const T*)a.x + rows.at(row);
        Pack<T, V> v[K];
        by_stream(a.stream_in, [&](auto past) {
#pragma unroll
            for (int k = 0; k < K; k++) {
                v[k] = load_loose<T, V, decltype(past)::value>(p + first[k]);
            }
        });
        float m = 0.f, q = 0.f;
#pragma unroll
        for (int e = 0; e < E; e++) {
            m += counted<WHOLE>(to_float(v[e / V].v[e % V]), e % V, skip[e / V]);
        }
        m = wide_sum(m, part[0], blockDim.x >> 6) * rows.inv;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const float d = counted<WHOLE>(to_float(v[e / V].v[e % V]) - m, e % V, skip[e / V]);
            q = fmaf(d, d, q);
        }
        q = inv_sqrt(fmaf(wide_sum(q, part[1], blockDim.x >> 6), rows.inv, a.eps));
        T* y = (T*)a.y + row * rows.n_ch;
#pragma unroll
        for (int k = 0; k < K; k++) {
            if (!HOLD) {
                load_params<V>(a.aff.weight, a.aff.type, first[k], 1.f, w + k * V);
                load_params<V>(a.aff.bias, a.aff.type, first[k], 0.f, b + k * V);
            }
            float z[V];
            unpack(v[k], z);
#pragma unroll
            for (int j = 0; j < V; j++) {
                z[j] = fmaf((z[j] - m) * q, w[k * V + j], b[k * V + j]);
            }
            act_values<T, V>(a.act, z);
            if (WHOLE || skip[k] < V) {
                by_stream(a.stream, [&](auto past) {
                    store_loose<T, V, decltype(past)::value>(y + first[k], z);
                });
            }
        }
        if (threadIdx.x == 0 && a.mean) {
            a.mean[row] = m;
            a.rstd[row] = q;
        }
    }
}

// Rows beyond a workgroup's registers go in chunks of a workgroup's E values a
// thread, in two passes: one leaves every chunk's (mean, squares about it), the
// other joins those of its row, every wave for itself. A workgroup keeps to one
// chunk, whose weight and bias it holds, and takes every gridDim.x-th row. 1000 x
// 60001 bfloat16: 75 us, 4.8 TB/s over rows read twice; backward 169, 3.6.
constexpr int kChunkElems = 32, kChunkElemsBwd = 16;  // a thread's

// A thread's vectors of a chunk.
template <int V, int K>
struct ChunkSpan {
    uint32_t first[K], skip[K], count;  // count: of the chunk
    __device__ __forceinline__ ChunkSpan(uint32_t chunk, uint32_t n_ch) {
        constexpr uint32_t kVecs = K * kThreads;
#pragma unroll
        for (uint32_t k = 0; k < K; k++) {
            const Span<V> sp(chunk * kVecs + k * kThreads + threadIdx.x, n_ch);
            first[k] = sp.first;
            skip[k] = sp.skip;
        }
        count = std::min(n_ch - chunk * (kVecs * V), kVecs * V);
    }
};

template <typename T, int V>
__global__ __launch_bounds__(kThreads) void k_ln_chunk_stats(const Forward a, float2* row_part) {
    __shared__ float part[2][kThreads / 64];
    constexpr int K = kChunkElems / V;
    const ChunkSpan<V, K> sp(blockIdx.y, a.rows.n_ch);
    const float inv = 1.f / (float)sp.count;
    for (uint64_t row = blockIdx.x; row < a.rows.n; row += gridDim.x) {
        const T* p = (const T*)a.x + a.rows.at(row);
        Pack<T, V> v[K];
#pragma unroll
        for (int k = 0; k < K; k++) {
            v[k] = load_loose<T, V>(p + sp.first[k]);
        }
        float m = 0.f, q = 0.f;
#pragma unroll
        for (int e = 0; e < kChunkElems; e++) {
            m += counted<false>(to_float(v[e / V].v[e % V]), e % V, sp.skip[e / V]);
        }
        m = wide_sum(m, part[0], blockDim.x >> 6) * inv;
#pragma unroll
        for (int e = 0; e < kChunkElems; e++) {
            const float d = counted<false>(to_float(v[e / V].v[e % V]) - m, e % V, sp.skip[e / V]);
            q = fmaf(d, d, q);
        }
        q = wide_sum(q, part[1], blockDim.x >> 6);
        if (threadIdx.x == 0) {
            row_part[row * gridDim.y + blockIdx.y] = make_float2(m, q);
        }
    }
}

// A row's sums over its chunks' entries, in double, in all lanes.
template <typename F>
__device__ __forceinline__ double2 join_chunks(const float2* part, uint32_t chunks, F&& f) {
    double2 s = make_double2(0.0, 0.0);
    for (uint32_t i = threadIdx.x & 63u; i < chunks; i += 64) {
        f(i, part[i], s);
    }
    for (int o = 1; o < 64; o <<= 1) {
        s.x += __shfl_xor(s.x, o);
        s.y += __shfl_xor(s.y, o);
    }
    return s;
}

template <typename T, int V>
__global__ __launch_bounds__(kThreads) void k_ln_chunk_apply(const Forward a,
                                                             const float2* row_part) {
    constexpr int K = kChunkElems / V;
    const uint32_t n_ch = a.rows.n_ch, chunks = gridDim.y;
    const ChunkSpan<V, K> sp(blockIdx.y, n_ch);
    const double full = kChunkElems * kThreads, last = n_ch - (chunks - 1) * full;
    float w[kChunkElems], b[kChunkElems];
#pragma unroll
    for (int k = 0; k < K; k++) {
        load_params<V>(a.aff.weight, a.aff.type, sp.first[k], 1.f, w + k * V);
        load_params<V>(a.aff.bias, a.aff.type, sp.first[k], 0.f, b + k * V);
    }
    for (uint64_t row = blockIdx.x; row < a.rows.n; row += gridDim.x) {
        const T* p = (const T*)a.x + a.rows.at(row);
        Pack<T, V> v[K];
#pragma unroll
        for (int k = 0; k < K; k++) {
            v[k] = load_loose<T, V>(p + sp.first[k]);
        }
        // about the first chunk's mean: their difference loses nothing
        const float2* entries = row_part + row * chunks;
        const double pivot = (double)entries[0].x;
        const double2 s = join_chunks(entries, chunks, [&](uint32_t i, float2 e, double2& t) {
            const double n = i + 1 == chunks ? last : full, d = (double)e.x - pivot;
            t.x = fma(n, d, t.x);
            t.y += fma(n * d, d, (double)e.y);
        });
        const double d = s.x / n_ch, var = s.y / n_ch - d * d;
        const float mean = (float)(pivot + d);
        const float rstd = inv_sqrt((float)(var < 0.0 ? 0.0 : var) + a.eps);
        T* y = (T*)a.y + row * n_ch;
#pragma unroll
        for (int k = 0; k < K; k++) {
            float z[V];
            unpack(v[k], z);
#pragma unroll
            for (int j = 0; j < V; j++) {
                z[j] = fmaf((z[j] - mean) * rstd, w[k * V + j], b[k * V + j]);
            }
            act_values<T, V>(a.act, z);
            if (sp.skip[k] < V) {
                by_stream(a.stream, [&](auto past) {
                    store_loose<T, V, decltype(past)::value>(y + sp.first[k], z);
                });
            }
        }
        if (blockIdx.y == 0 && threadIdx.x == 0 && a.mean) {
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
    bool stream, stream_in;
};

// Of E values: xh in place of x and t = w gz in place of gy, gz added to the sums
// of its columns, and t to those of the row.
template <typename T, int V, int E, bool WHOLE>
__device__ __forceinline__ float2 slopes(float mean, float rstd, const float (&w)[E],
                                         const float (&b)[E], uint32_t act, const uint32_t* skip,
                                         float (&xh)[E], float (&t)[E], float (&gw)[E],
                                         float (&gb)[E]) {
    float z[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
        xh[e] = (xh[e] - mean) * rstd;
        z[e] = fmaf(xh[e], w[e], b[e]);
    }
    act_slopes<T, E>(act, z, t);
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int e = 0; e < E; e++) {
        gb[e] += t[e];
        gw[e] = fmaf(t[e], xh[e], gw[e]);
        t[e] *= w[e];
        const float c = counted<WHOLE>(t[e], e % V, skip[e / V]);
        s.x += c;
        s.y = fmaf(c, xh[e], s.y);  // an xh that is not finite is the whole row's
    }
    return s;
}

// gx of a vector, a and c the row's means of t and t xh.
template <typename T, int V>
__device__ __forceinline__ void write_gx(const float* xh, const float* t, float rstd, float a,
                                         float c, T* gx, bool stream) {
    float g[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        g[j] = rstd * fmaf(-xh[j], c, t[j] - a);
    }
    by_stream(stream, [&](auto past) { store_loose<T, V, decltype(past)::value>(gx, g); });
}

// A workgroup's sums of the columns `ch` on, of which the first `skip` are
// another's.
template <int V>
__device__ __forceinline__ void write_sums(const Backward& a, uint32_t ch, uint32_t skip,
                                           const float* gw, const float* gb) {
    float* p = a.part ? a.part + blockIdx.x * a.part_stride + ch : nullptr;
    if (p && skip == 0) {
        store_loose<float, V>(p, gw);
        store_loose<float, V>(p + a.rows.n_ch, gb);
        return;
    }
#pragma unroll
    for (uint32_t j = 0; j < V; j++) {
        if (j < skip) {
            continue;
        }
        if (p) {
            p[j] = gw[j];
            p[a.rows.n_ch + j] = gb[j];
            continue;
        }
        if (a.gw) {
            store_one(a.gw, a.aff.type, ch + j, gw[j]);
        }
        if (a.gb) {
            store_one(a.gb, a.aff.type, ch + j, gb[j]);
        }
    }
}

// Whether a lane reads its next row while it works on one, or else two at a time:
// the first where all lanes have values (4194304 x 64 bfloat16 297 us, 300 by two)
// and for long rows of 32 bits (100000 x 300 77 and 85, 500000 x 100 108 and 112),
// the second in 16 bits where some do not (500000 x 200 118, 129 ahead; 500000 x
// 248 140 and 150).
template <int V, int L, bool WHOLE>
constexpr bool kAhead = WHOLE || (V == 4 && L >= 32);

// L lanes hold a row, K vectors each, and keep the sums of their columns. 4 x 1024 x
// 1024 x 64 bfloat16, silu: 299 us, 5.4 TB/s (gelu 332); 500000 x 100 float32 108,
// 5.5 TB/s. Rows of just over a power of two of vectors leave half of the lanes
// idle: 800000 x 130 bfloat16 150 us, 4.2 TB/s.
template <typename T, int V, int L, int K, bool WHOLE>
__global__ __launch_bounds__(kThreads) void k_ln_bwd_rows(const Backward a) {
    constexpr int E = K * V, R = kAhead<V, L, WHOLE> ? 1 : 2;
    constexpr uint32_t kSlots = kThreads / L, kTake = kSlots * R, kWaves = kThreads / 64;
    __shared__ float red[kWaves][2][L * E];
    const uint32_t lane = threadIdx.x % L, slot = threadIdx.x / L;
    const Rows& rows = a.rows;
    const uint32_t px_bytes = (uint32_t)(rows.px_stride * sizeof(T));
    const uint32_t row_bytes = rows.n_ch * sizeof(T);
    uint32_t first[K], skip[K];  // first: in bytes
    float w[E], b[E], gw[E], gb[E];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const Span<V> sp(k * L + lane, rows.n_ch);
        first[k] = sp.first * sizeof(T);
        skip[k] = sp.skip;
        load_params<V>(a.aff.weight, a.aff.type, sp.first, 1.f, w + k * V);
        load_params<V>(a.aff.bias, a.aff.type, sp.first, 0.f, b + k * V);
    }
#pragma unroll
    for (int e = 0; e < E; e++) {
        gw[e] = gb[e] = 0.f;
    }
    struct Raw {
        Pack<T, V> x[R][K], g[R][K];
        float mean[R], rstd[R];
    };
    const uint32_t in = slot * px_bytes, out = slot * row_bytes;
    const auto load = [&](uint64_t r0, Raw& r) {
        const T* x = (const T*)a.x;
        const T* g = (const T*)a.gy;
        if (rows.flat && r0 + kTake <= rows.n) {
            x += r0 * rows.px_stride;
            g += r0 * rows.n_ch;
            by_stream(kLongPieces<L, K> && a.stream_in, [&](auto past) {
#pragma unroll
                for (int i = 0; i < R; i++) {
                    r.mean[i] = (a.mean + r0 + i * kSlots)[slot];
                    r.rstd[i] = (a.rstd + r0 + i * kSlots)[slot];
#pragma unroll
                    for (int k = 0; k < K; k++) {
                        r.x[i][k] = load_loose<T, V, decltype(past)::value>(
                            at_byte(x + (size_t)(i * kSlots) * rows.px_stride, in + first[k]));
                        r.g[i][k] = load_loose<T, V, decltype(past)::value>(
                            at_byte(g + (size_t)(i * kSlots) * rows.n_ch, out + first[k]));
                    }
                }
            });
        } else {  // past the end the last row again
#pragma unroll
            for (int i = 0; i < R; i++) {
                const uint64_t row = std::min(r0 + i * kSlots + slot, rows.n - 1);
                const T* p = x + rows.at(row);
                const T* q = g + row * rows.n_ch;
                r.mean[i] = a.mean[row];
                r.rstd[i] = a.rstd[row];
#pragma unroll
                for (int k = 0; k < K; k++) {
                    r.x[i][k] = load_loose<T, V>(at_byte(p, first[k]));
                    r.g[i][k] = load_loose<T, V>(at_byte(q, first[k]));
                }
            }
        }
    };
    const uint64_t step = (uint64_t)gridDim.x * kTake;
    uint64_t r0 = (uint64_t)blockIdx.x * kTake;  // there are no more workgroups than rows for them
    Raw raw;
    if (kAhead<V, L, WHOLE>) {
        load(r0, raw);
    }
    for (; r0 < rows.n; r0 += step) {
        Raw ahead;
        if (!kAhead<V, L, WHOLE>) {
            load(r0, raw);
        } else if (r0 + step < rows.n) {
            load(r0 + step, ahead);
        }
#pragma unroll
        for (int i = 0; i < R; i++) {
            const bool live = r0 + i * kSlots + slot < rows.n;
            float xh[E], t[E];
            float2 s = make_float2(0.f, 0.f);
            if (live) {
#pragma unroll
                for (int e = 0; e < E; e++) {
                    xh[e] = to_float(raw.x[i][e / V].v[e % V]);
                    t[e] = to_float(raw.g[i][e / V].v[e % V]);
                }
                s = slopes<T, V, E, WHOLE>(raw.mean[i], raw.rstd[i], w, b, a.act, skip, xh, t, gw,
                                           gb);
            }
            s.x = lane_sum<L>(s.x) * rows.inv;
            s.y = lane_sum<L>(s.y) * rows.inv;
            if (live && a.gx) {
                T* gx = (T*)a.gx + (r0 + i * kSlots) * rows.n_ch;
#pragma unroll
                for (int k = 0; k < K; k++) {
                    if (WHOLE || skip[k] < V) {
                        write_gx<T, V>(xh + k * V, t + k * V, raw.rstd[i], s.x, s.y,
                                       at_byte(gx, out + first[k]), a.stream);
                    }
                }
            }
        }
        if (kAhead<V, L, WHOLE>) {
            raw = ahead;
        }
    }
    if (!a.part && !a.gw && !a.gb) {
        return;
    }
    // a column's sums over the slots: of a wave, then of the waves
    const uint32_t wave = threadIdx.x >> 6;
#pragma unroll
    for (int e = 0; e < E; e++) {
#pragma unroll
        for (int o = L; o < 64; o <<= 1) {
            gw[e] += __shfl_xor(gw[e], o);
            gb[e] += __shfl_xor(gb[e], o);
        }
        if ((threadIdx.x & 63u) < L) {
            // a vector's values side by side
            const uint32_t at = ((e / V) * L + lane) * V + e % V;
            red[wave][0][at] = gw[e];
            red[wave][1][at] = gb[e];
        }
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < L * E; e += kThreads) {
        const Span<V> sp(e / V, rows.n_ch);
        if (e % V >= sp.skip) {
            float sw = red[0][0][e], sb = red[0][1][e];
#pragma unroll
            for (uint32_t i = 1; i < kWaves; i++) {
                sw += red[i][0][e];
                sb += red[i][1][e];
            }
            write_sums<1>(a, sp.first + e % V, 0, &sw, &sb);
        }
    }
}

// A workgroup holds a row, or two in a half each, K vectors a thread, and reads
// the next meanwhile, unless there are 1024 threads: those have too few registers
// each for that, and keep weight and bias in LDS (4096 x 16384 float32: 166 us, 4.9
// TB/s; 302 in chunks). 16384 x 4096 bfloat16: 75 us, 5.4 TB/s, 79 with a row a
// workgroup, of which there are then twice as many sums of gw and gb to add.
template <typename T, int V, int K, uint32_t THREADS, uint32_t HALVES, bool WHOLE>
__global__ __launch_bounds__(THREADS) void k_ln_bwd_wide(const Backward a) {
    __shared__ float2 part[2][THREADS / 64];
    constexpr int E = K * V;
    constexpr bool kFew = THREADS == 1024;
    __shared__ Pack<float, V> affine[kFew ? 2 : 1][kFew ? K * THREADS : 1];
    const Rows& rows = a.rows;
    const uint32_t lanes = blockDim.x / HALVES, half = threadIdx.x / lanes;
    const uint32_t lane = threadIdx.x - half * lanes;
    uint32_t first[K], skip[K];
    float w[E], b[E], gw[E], gb[E];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const Span<V> sp(k * lanes + lane, rows.n_ch);
        first[k] = sp.first;
        skip[k] = sp.skip;
        load_params<V>(a.aff.weight, a.aff.type, sp.first, 1.f, w + k * V);
        load_params<V>(a.aff.bias, a.aff.type, sp.first, 0.f, b + k * V);
        if (kFew) {  // each thread's own: no barrier
#pragma unroll
            for (int j = 0; j < V; j++) {
                affine[0][k * THREADS + threadIdx.x].v[j] = w[k * V + j];
                affine[1][k * THREADS + threadIdx.x].v[j] = b[k * V + j];
            }
        }
    }
#pragma unroll
    for (int e = 0; e < E; e++) {
        gw[e] = gb[e] = 0.f;
    }
    struct Raw {
        Pack<T, V> x[K], g[K];
        float mean, rstd;
    };
    const auto load = [&](uint64_t row, Raw& r) {
        const T* p = (const T*)a.x + rows.at(row);
        const T* q = (const T*)a.gy + row * rows.n_ch;
        r.mean = a.mean[row];
        r.rstd = a.rstd[row];
        by_stream(!kFew && a.stream_in, [&](auto past) {
#pragma unroll
            for (int k = 0; k < K; k++) {
                r.x[k] = load_loose<T, V, decltype(past)::value>(p + first[k]);
                r.g[k] = load_loose<T, V, decltype(past)::value>(q + first[k]);
            }
        });
    };
    uint32_t turn = 0;
    Raw raw;
    const uint64_t step = (uint64_t)gridDim.x * HALVES;
    const auto mine = [&](uint64_t row0) { return std::min(row0 + half, rows.n - 1); };
    uint64_t row0 = (uint64_t)blockIdx.x * HALVES;  // there are no more workgroups than rows
    if (!kFew) {
        load(mine(row0), raw);
    }
    for (; row0 < rows.n; row0 += step, turn ^= 1) {
        const uint64_t row = row0 + half;
        const bool live = HALVES == 1 || row < rows.n;
        Raw ahead;
        if (kFew) {
            load(row, raw);
        } else if (row0 + step < rows.n) {
            load(mine(row0 + step), ahead);
        }
        float xh[E], t[E];
#pragma unroll
        for (int e = 0; e < E; e++) {
            xh[e] = to_float(raw.x[e / V].v[e % V]);
            t[e] = to_float(raw.g[e / V].v[e % V]);
        }
        const float rstd = raw.rstd;
        float2 s = make_float2(0.f, 0.f);
        if constexpr (kFew) {
#pragma unroll
            for (int k = 0; k < K; k++) {
                float wk[V], bk[V];
                unpack(affine[0][k * THREADS + threadIdx.x], wk);
                unpack(affine[1][k * THREADS + threadIdx.x], bk);
                const auto part_of = [&](float* p) -> float (&)[V] {
                    return *(float (*)[V])(p + k * V);
                };
                const float2 sk = slopes<T, V, V, WHOLE>(
                    raw.mean, rstd, wk, bk, a.act, skip + k, part_of(xh), part_of(t), part_of(gw),
                    part_of(gb));
                s.x += sk.x;
                s.y += sk.y;
            }
        } else if (live) {
            s = slopes<T, V, E, WHOLE>(raw.mean, rstd, w, b, a.act, skip, xh, t, gw, gb);
        }
        s = wide_sum(s, part[turn], half * (lanes >> 6), lanes >> 6);
        if (live && a.gx) {
            T* gx = (T*)a.gx + row * rows.n_ch;
#pragma unroll
            for (int k = 0; k < K; k++) {
                if (WHOLE || skip[k] < V) {
                    write_gx<T, V>(xh + k * V, t + k * V, rstd, s.x * rows.inv, s.y * rows.inv,
                                   gx + first[k], a.stream);
                }
            }
        }
        if (!kFew) {
            raw = ahead;
        }
    }
    if (!a.part && !a.gw && !a.gb) {
        return;
    }
    if constexpr (HALVES == 2) {
        __shared__ float red[2][E][THREADS / 2];
        if (half == 1) {
#pragma unroll
            for (int e = 0; e < E; e++) {
                red[0][e][lane] = gw[e];
                red[1][e][lane] = gb[e];
            }
        }
        __syncthreads();
        if (half == 1) {
            return;
        }
#pragma unroll
        for (int e = 0; e < E; e++) {
            gw[e] += red[0][e][lane];
            gb[e] += red[1][e][lane];
        }
    }
#pragma unroll
    for (int k = 0; k < K; k++) {
        write_sums<V>(a, first[k], skip[k], gw + k * V, gb + k * V);
    }
}

// Longer rows, in chunks like the forward pass's. The first pass leaves a chunk's
// sums of t and t xh of each row, and the columns' over its rows.
template <typename T, int V, bool APPLY>
__global__ __launch_bounds__(kThreads) void k_ln_bwd_chunk(const Backward a, float2* row_part) {
    __shared__ float2 part[2][kThreads / 64];
    constexpr int E = kChunkElemsBwd, K = E / V;
    const Rows& rows = a.rows;
    const uint32_t chunk = blockIdx.y, chunks = gridDim.y;
    const ChunkSpan<V, K> sp(chunk, rows.n_ch);
    float w[E], b[E], gw[E], gb[E];
#pragma unroll
    for (int k = 0; k < K; k++) {
        load_params<V>(a.aff.weight, a.aff.type, sp.first[k], 1.f, w + k * V);
        load_params<V>(a.aff.bias, a.aff.type, sp.first[k], 0.f, b + k * V);
    }
#pragma unroll
    for (int e = 0; e < E; e++) {
        gw[e] = gb[e] = 0.f;
    }
    uint32_t turn = 0;
    for (uint64_t row = blockIdx.x; row < rows.n; row += gridDim.x, turn ^= 1) {
        const T* p = (const T*)a.x + rows.at(row);
        const T* q = (const T*)a.gy + row * rows.n_ch;
        const float mean = a.mean[row], rstd = a.rstd[row];
        Pack<T, V> xv[K], gv[K];
#pragma unroll
        for (int k = 0; k < K; k++) {
            xv[k] = load_loose<T, V>(p + sp.first[k]);
            gv[k] = load_loose<T, V>(q + sp.first[k]);
        }
        float xh[E], t[E];
#pragma unroll
        for (int e = 0; e < E; e++) {
            xh[e] = to_float(xv[e / V].v[e % V]);
            t[e] = to_float(gv[e / V].v[e % V]);
        }
        const float2 s = slopes<T, V, E, false>(mean, rstd, w, b, a.act, sp.skip, xh, t, gw, gb);
        if constexpr (APPLY) {
            const double2 sum = join_chunks(row_part + row * chunks, chunks,
                                            [](uint32_t, float2 e, double2& d) {
                                                d.x += (double)e.x;
                                                d.y += (double)e.y;
                                            });
            const float ma = (float)(sum.x / rows.n_ch), mc = (float)(sum.y / rows.n_ch);
            T* gx = (T*)a.gx + row * rows.n_ch;
#pragma unroll
            for (int k = 0; k < K; k++) {
                if (sp.skip[k] < V) {
                    write_gx<T, V>(xh + k * V, t + k * V, rstd, ma, mc, gx + sp.first[k], a.stream);
                }
            }
        } else {
            const float2 sum = wide_sum(s, part[turn], 0, kThreads / 64);
            if (threadIdx.x == 0) {
                row_part[row * chunks + chunk] = sum;
            }
        }
    }
    if (APPLY || (!a.part && !a.gw && !a.gb)) {
        return;
    }
#pragma unroll
    for (int k = 0; k < K; k++) {
        write_sums<V>(a, sp.first[k], sp.skip[k], gw + k * V, gb + k * V);
    }
}

// Adds the workgroups' sums of gw and gb, in their order: 16 columns of the
// 2 n_ch a workgroup, four a lane, over 256 lanes. n 0: sums of nothing. 1024 sums
// of 64 channels 5 us, 256 of 4096 channels 4.5: a launch and a few loads one
// after another.
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

// A type's vectors, and single values where a row is shorter.
constexpr uint32_t vec_of(uint32_t type, uint32_t n_ch) {
    const uint32_t v = type == DRESSI_F32 ? 4 : 8;
    return n_ch >= v ? v : 1;
}

// Values of a row up to which a wave, then a workgroup, holds it. Backward a wave
// with two vectors of 16 bits a lane holds so many registers that there are two a
// SIMD (65536 x 1024 bfloat16 87 us, 77 with 128 lanes a row; float32 143 and 149).
constexpr uint32_t kWaveElems = 64 * 32;
constexpr uint32_t wave_elems_bwd(uint32_t v) { return 64 * (v == 4 ? 16 : 8); }
constexpr uint32_t kHoldElems = 1024 * 32, kHoldElemsBwd = 1024 * 16;

// Bytes of results, and of inputs, from which they go past the caches. Results:
// 1000000 x 128 bfloat16 84 us so and 87 through them, 30000000 x 8 float16 167 and
// 214. Inputs: 30000000 x 8 float16 167 and 216; below, where a layer before may
// have left them in a cache, 100000 x 511 float32 takes 73 so and 71 through them.
constexpr uint64_t kStreamBytes = 32ull << 20, kStreamInBytes = 256ull << 20;

struct Plan {
    uint32_t v;
    bool wide, whole, stream, stream_in;
    uint32_t lanes;   // of a row; wide: the workgroup's threads
    uint32_t elems;   // of a lane
    uint32_t chunks;  // of a row, where there are some
    uint32_t groups;  // workgroups whose sums of gw and gb are added
};

// Lanes and values of each for a row that a wave holds. One vector a lane, where
// a wave's load or store is one piece of memory (2000000 x 24 float32 forward 65
// us, 88 with six vectors a lane); forward three, where fewer than 9 of 16 lanes
// had one (500000 x 264 float16 102 us, 114 with one; rows of 17 vectors gain by it
// where a cache holds x, and lose where none does: 800000 x 130 bfloat16 78 and 80,
// 102 and 91; backward the registers of three cost more than the lanes). Longer
// rows take a whole wave.
void cut_row(Plan& p, uint32_t n_ch, bool backward) {
    const uint32_t vecs = div_up(n_ch, p.v);
    p.lanes = p.elems = 1;
    if (p.v == 1) {  // a lane a row
        while (p.elems < n_ch) {
            p.elems *= 2;
        }
        return;
    }
    while (p.lanes < 64 && p.lanes < vecs) {
        p.lanes *= 2;
    }
    uint32_t iter = div_up(vecs, p.lanes);
    if (iter == 1 && !backward && 16 * vecs < 9 * p.lanes) {
        p.lanes /= 4;
        iter = 3;
    } else if (iter > 4 || (backward && iter > 2)) {
        iter = iter > 6 ? 8 : backward ? 4 : 6;
    }
    p.elems = iter * p.v;
}

// By the number of rows and not by where they lie: so is the scratch.
Plan make_plan(uint32_t type, uint64_t rows, uint32_t n_ch, bool backward) {
    Plan p{};
    p.v = vec_of(type, n_ch);
    const uint64_t bytes = rows * n_ch * type_bytes(type);
    p.stream = bytes >= kStreamBytes;
    p.stream_in = bytes * (backward ? 2 : 1) >= kStreamInBytes;
    if (n_ch > (backward ? kHoldElemsBwd : kHoldElems)) {
        p.elems = backward ? kChunkElemsBwd : kChunkElems;
        p.chunks = div_up(n_ch, p.elems * kThreads);
        p.groups = (uint32_t)std::min<uint64_t>(rows, std::max(1u, 1024 / p.chunks));
    } else if (n_ch > (backward ? wave_elems_bwd(p.v) : kWaveElems)) {
        p.wide = true;
        p.elems = p.v;
        while (p.elems < (backward ? 16 : 32) && n_ch > p.elems * 256) {
            p.elems *= 2;
        }
        if (!backward && n_ch > 8192 && n_ch <= 16 * 1024) {
            p.elems = 16;  // 4096 x 9216 bfloat16 38 us, 52 with 32 in half the threads
        }
        p.lanes = div_up(div_up(n_ch, p.elems), 64) * 64;
        // 512 threads for each of 256 compute units, or twice that where they hold 8 values; fewer
        // where their sums would be as much as the rows (1021 x 4096 bfloat16 16.3 us, 21.2 with
        // 512 workgroups; 1021 x 2048 11.1 and 13.8)
        const uint32_t most = (p.elems == 16 ? 256 : 512) * 256 / std::min(256u, p.lanes);
        const uint64_t pairs = p.lanes > 256 ? rows : (rows + 1) / 2;
        p.groups = (uint32_t)std::min<uint64_t>({pairs, most, std::max<uint64_t>(256, pairs / 8)});
    } else {
        cut_row(p, n_ch, backward);
        const bool ahead = n_ch == p.lanes * p.elems || (p.v == 4 && p.lanes >= 32);  // kAhead
        const uint64_t take = kThreads / p.lanes * (ahead ? 1 : 2);
        // four for each compute unit: 1280, where some have five, take 370 us for 4194304 x 64
        // bfloat16, 768 329 and these 299
        p.groups = (uint32_t)std::min<uint64_t>((rows + take - 1) / take, 1024);
    }
    p.whole = n_ch == p.lanes * p.elems;
    // a store that does not fill lines is slower past the caches, which would have
    // filled them (20000000 x 7 float16 backward, value by value: 667 and 392 us)
    p.stream = p.stream && (p.chunks > 0 || p.elems == p.v || p.lanes >= 8);
    return p;
}

size_t part_stride(uint32_t n_ch) { return (2 * (size_t)n_ch + 3) / 4 * 4; }

// Bytes of the chunks' sums, and of the workgroups' of gw and gb after them.
size_t row_bytes(const Plan& p, uint64_t rows) {
    return (rows * p.chunks * sizeof(float2) + 15) / 16 * 16;
}
size_t scratch_bytes_of(const Plan& p, uint64_t rows, uint32_t n_ch, bool backward) {
    const bool sums = backward && p.groups > 1;
    return row_bytes(p, rows) + (sums ? p.groups * part_stride(n_ch) * sizeof(float) : 0);
}

template <typename A>
int launch(void (*kernel)(A), uint64_t most, uint32_t limit, uint32_t threads, hipStream_t s,
           const A& a) {
    hipLaunchKernelGGL(kernel, dim3((uint32_t)std::min<uint64_t>(most, limit)), dim3(threads), 0, s,
                       a);
    DRESSI_CHECK_LAUNCH();
    return DRESSI_OK;
}

template <typename F>
auto for_bool(bool x, F&& f) {
    return x ? f(std::true_type()) : f(std::false_type());
}
// f(x as a constant) of the values in the list.
template <uint32_t FIRST, uint32_t... MORE, typename F>
int for_value(uint32_t x, F&& f) {
    if constexpr (sizeof...(MORE) > 0) {
        if (x != FIRST) {
            return for_value<MORE...>(x, f);
        }
    }
    return f(std::integral_constant<uint32_t, FIRST>());
}

// f(values) of a row that one lane holds value by value, its length rounded up to
// a power of two: up to 3 values of 32 bits, 7 of 16.
template <typename T, bool WHOLE, typename F>
int for_few(uint32_t elems, F&& f) {
    if constexpr (sizeof(T) == 4 && WHOLE) {
        return for_value<1, 2>(elems, f);
    } else if constexpr (sizeof(T) == 4) {
        return for_value<4>(elems, f);
    } else if constexpr (WHOLE) {
        return for_value<1, 2, 4>(elems, f);
    } else {
        return for_value<4, 8>(elems, f);
    }
}
// f(lanes) of a row with a vector for each: one is always whole.
template <bool WHOLE, typename F>
int for_lanes(uint32_t lanes, F&& f) {
    if constexpr (WHOLE) {
        return for_value<1, 2, 4, 8, 16, 32, 64>(lanes, f);
    } else {
        return for_value<2, 4, 8, 16, 32, 64>(lanes, f);
    }
}

template <typename T, int V>
int forward(hipStream_t s, const Plan& p, const Forward& a, void* scratch) {
    if (p.chunks) {
        const uint32_t most = std::max(1u, 2048 / p.chunks);
        const dim3 grid((uint32_t)std::min<uint64_t>(a.rows.n, most), p.chunks);
        if constexpr (V > 1) {
            hipLaunchKernelGGL((k_ln_chunk_stats<T, V>), grid, dim3(kThreads), 0, s, a,
                               (float2*)scratch);
            DRESSI_CHECK_LAUNCH();
            hipLaunchKernelGGL((k_ln_chunk_apply<T, V>), grid, dim3(kThreads), 0, s, a,
                               (const float2*)scratch);
            DRESSI_CHECK_LAUNCH();
        }
        return DRESSI_OK;
    }
    return for_bool(p.whole, [&](auto whole) {
        constexpr bool W = decltype(whole)::value;
        const auto rows = [&](auto lanes, auto elems) {
            constexpr int L = decltype(lanes)::value, K = decltype(elems)::value / V;
            constexpr uint32_t kTake = kThreads / L * kInFlight<T, K * V>;
            // 4194304 x 64 bfloat16: 175 us, 191 with 2048 workgroups
            return launch(k_ln_rows<T, V, L, K, W>, (a.rows.n + kTake - 1) / kTake, 16384, kThreads,
                          s, a);
        };
        if constexpr (V == 1) {
            return for_few<T, W>(p.elems, [&](auto elems) {
                return rows(std::integral_constant<int, 1>(), elems);
            });
        } else {
            if (p.wide) {
                return for_value<16, 32>(p.elems, [&](auto elems) {
                    constexpr int K = decltype(elems)::value / V;
                    const uint32_t limit = 256 * (2048 / p.lanes);
                    if (p.lanes > 256) {
                        return launch(k_ln_wide<T, V, K, 1024, false, W>, a.rows.n, limit, p.lanes,
                                      s, a);
                    }
                    return launch(k_ln_wide<T, V, K, 256, true, W>, a.rows.n, limit, p.lanes, s,
                                  a);
                });
            }
            if (p.lanes == 64 && p.elems > V) {
                const auto wave = [&](auto iter) {
                    return rows(std::integral_constant<int, 64>(),
                                std::integral_constant<int, decltype(iter)::value * V>());
                };
                if constexpr (V == 4) {
                    return for_value<2, 3, 4, 6, 8>(p.elems / V, wave);
                } else {
                    return for_value<2, 3, 4>(p.elems / V, wave);
                }
            }
            if constexpr (!W) {  // 17, or 33 to 35, vectors
                if (p.elems > V) {
                    return for_value<8, 16>(p.lanes, [&](auto lanes) {
                        return rows(lanes, std::integral_constant<int, 3 * V>());
                    });
                }
            }
            return for_lanes<W>(p.lanes, [&](auto lanes) {
                return rows(lanes, std::integral_constant<int, V>());
            });
        }
    });
}

template <typename T, int V>
int backward(hipStream_t s, const Plan& p, const Backward& a, float2* row_part) {
    if (p.chunks) {
        if constexpr (V > 1) {
            const dim3 grid(p.groups, p.chunks);
            hipLaunchKernelGGL((k_ln_bwd_chunk<T, V, false>), grid, dim3(kThreads), 0, s, a,
                               row_part);
            DRESSI_CHECK_LAUNCH();
            if (a.gx) {
                hipLaunchKernelGGL((k_ln_bwd_chunk<T, V, true>), grid, dim3(kThreads), 0, s, a,
                                   row_part);
                DRESSI_CHECK_LAUNCH();
            }
        }
        return DRESSI_OK;
    }
    return for_bool(p.whole, [&](auto whole) {
        constexpr bool W = decltype(whole)::value;
        const auto rows = [&](auto lanes, auto iter) {
            constexpr int L = decltype(lanes)::value, K = decltype(iter)::value;
            return launch(k_ln_bwd_rows<T, V, L, K, W>, p.groups, ~0u, kThreads, s, a);
        };
        if constexpr (V == 1) {
            return for_few<T, W>(p.elems, [&](auto elems) {
                return rows(std::integral_constant<int, 1>(), elems);
            });
        } else {
            if (p.wide) {
                return for_value<8, 16>(p.elems, [&](auto elems) {
                    constexpr int K = decltype(elems)::value / V;
                    if constexpr (K * V == 16) {
                        if (p.lanes > 512) {
                            return launch(k_ln_bwd_wide<T, V, K, 1024, 1, W>, p.groups, ~0u,
                                          p.lanes, s, a);
                        }
                        if (p.lanes > 256) {
                            return launch(k_ln_bwd_wide<T, V, K, 512, 1, W>, p.groups, ~0u,
                                          p.lanes, s, a);
                        }
                    }
                    return launch(k_ln_bwd_wide<T, V, K, 512, 2, W>, p.groups, ~0u, 2 * p.lanes, s,
                                  a);
                });
            }
            if constexpr (V == 4) {
                if (p.elems > V) {
                    return for_value<2, 4>(p.elems / V, [&](auto iter) {
                        return rows(std::integral_constant<int, 64>(), iter);
                    });
                }
            }
            return for_lanes<W>(p.lanes, [&](auto lanes) {
                return rows(lanes, std::integral_constant<int, 1>());
            });
        }
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
    Rows r{n_items * n_px, n_px, item_stride, px_stride, n_ch, 0, 1.f / (float)n_ch};
    if (n_px == 1) {
        r.px_stride = item_stride;
    }
    if (n_items == 1 || n_px == 1 || item_stride == n_px * px_stride) {
        r.n_px = r.n;
    }
    r.flat = r.n_px == r.n && r.px_stride <= kMaxPxStride;
    return r;
}

// Whether the pointers lie as their types ask.
int check_aligned(const char* what, uint32_t type, std::initializer_list<const void*> rows,
                  uint32_t affine_type, std::initializer_list<const void*> params,
                  std::initializer_list<const void*> stats) {
    const auto off = [](std::initializer_list<const void*> list, size_t bytes) {
        uintptr_t all = 0;
        for (const void* p : list) {
            all |= (uintptr_t)p;
        }
        return all % bytes != 0;
    };
    DRESSI_REQUIRE(!off(rows, type_bytes(type)), "%s: not aligned to its type", what);
    DRESSI_REQUIRE(!off(params, type_bytes(affine_type)),
                   "%s: the weight, the bias or a gradient of theirs is not aligned to its type",
                   what);
    DRESSI_REQUIRE(!off(stats, sizeof(float)), "%s: mean or rstd is not aligned", what);
    return DRESSI_OK;
}

// Whether results, packed, may be written while rows at `in` are read: not over
// them, unless over each row's own values, where they are packed too and are read
// by the lanes that write there or before a barrier: in chunks a moved-back vector
// is not.
int check_apart(const char* what, const void* out, const void* in, uint32_t type, const Rows& r,
                bool packed, const Plan& p) {
    const uintptr_t at = (uintptr_t)out, from = (uintptr_t)in;
    const uintptr_t bytes = (uintptr_t)(r.n * r.n_ch * type_bytes(type));
    const bool same = packed && (p.chunks == 0 || r.n_ch % p.v == 0);
    const bool clear = !packed || at + bytes <= from || from + bytes <= at;
    DRESSI_REQUIRE(!out || (at == from ? same : clear), "%s: results overlap what is read", what);
    return DRESSI_OK;
}
bool is_packed(const Rows& r) {
    return r.n_px == r.n && (r.n <= 1 || r.px_stride == r.n_ch);
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
    if (int rc = check_aligned("layer_norm", type, {x, y}, affine_type, {weight, bias},
                               {mean, rstd})) {
        return rc;
    }
    const Rows rows = make_rows(n_items, n_px, n_ch, item_stride, px_stride);
    const Plan p = make_plan(type, rows.n, n_ch, false);
    const size_t need = scratch_bytes_of(p, rows.n, n_ch, false);
    DRESSI_REQUIRE(
        need == 0 || (scratch && ((uintptr_t)scratch & 15) == 0 && scratch_bytes >= need),
        "layer_norm: scratch too small or not aligned");
    if (int rc = check_apart("layer_norm", y, x, type, rows, is_packed(rows), p)) {
        return rc;
    }
    const DeviceScope scope(ctx->device);
    DRESSI_TRY_HIP(scope.error());
    const Forward a{x, y, mean, rstd, rows, aff, eps, activation, p.stream, p.stream_in};
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
    if (int rc = check_aligned("layer_norm_bwd", type, {gy, x, gx}, affine_type,
                               {weight, bias, gw, gb}, {mean, rstd})) {
        return rc;
    }
    const Rows rows = make_rows(n_items, n_px, n_ch, item_stride, px_stride);
    const Plan p = make_plan(type, rows.n, n_ch, true);
    const bool params = gw || gb, join = params && p.groups != 1;
    float* part = join ? (float*)((char*)scratch + row_bytes(p, rows.n)) : nullptr;
    if (rows.n > 0) {
        DRESSI_REQUIRE(gy && x && mean && rstd, "layer_norm_bwd: bad arguments");
        const size_t need = scratch_bytes_of(p, rows.n, n_ch, true);
        DRESSI_REQUIRE(
            need == 0 || (scratch && ((uintptr_t)scratch & 15) == 0 && scratch_bytes >= need),
            "layer_norm_bwd: scratch too small or not aligned");
        int rc = check_apart("layer_norm_bwd", gx, gy, type, rows, true, p);
        if (rc || (rc = check_apart("layer_norm_bwd", gx, x, type, rows, is_packed(rows), p))) {
            return rc;
        }
    } else if (!join) {
        return DRESSI_OK;
    }
    const DeviceScope scope(ctx->device);
    DRESSI_TRY_HIP(scope.error());
    if (rows.n > 0) {
        const Backward a{gy, x, mean, rstd, gx, part, part_stride(n_ch),
                         join ? nullptr : gw, join ? nullptr : gb, rows, aff, activation,
                         p.stream, p.stream_in};
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
