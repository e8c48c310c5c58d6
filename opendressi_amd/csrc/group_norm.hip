// group_norm.hip -- group normalisation of channels-last images with an
// activation, forward and backward (dressi_group_norm, dressi_group_norm_bwd).
//
// Item n, group g of D = C / G channels, M = n_px D values:
//
//   mu = mean x, s = 1 / sqrt(mean (x - mu)^2 + eps), xh = (x - mu) s
//   z = xh w + b, y = act(z)
//   gz = gy act'(z), gb = sum gz, gw = sum gz xh (over items and pixels)
//   gx = s (w gz - mean_g(w gz) - xh mean_g(w gz xh))
//
// Memory bounds it. A group's channels lie side by side in a pixel, so a
// workgroup takes whole pixels of a run (a "chunk") of one item: a thread
// keeps one vector of V channels and walks the pixels. Two passes: one leaves
// each chunk's sums, the other begins by joining the chunks' sums of its item
// (every workgroup for itself: a launch in between costs more) and then reads
// the image again.
//
// Statistics: a batch of a thread's values gives its mean and the squares
// about that mean, both from registers, and (count, mean, squares) of two sets
// are joined exactly; so values far from zero lose nothing to cancellation.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "internal.h"
#include "typed.h"

namespace dressi {
namespace {

constexpr uint32_t kMaxThreads = 512;
constexpr uint32_t kMaxVecs = 256;  // of a workgroup
constexpr uint32_t kBatch = 4;      // pixels of a thread in flight
constexpr uint32_t kTargetGroups = 1024;  // workgroups that a launch should have

// How an image is cut. A block is a set of whole groups or, where a group has
// more than kMaxVecs vectors, one part of a group.
struct Cut {
    uint64_t n_px;
    uint64_t item_stride, px_stride;  // of x, in elements
    uint32_t n_items, n_ch, n_groups;
    uint32_t vpg;        // vectors of a group
    uint32_t gpb;        // groups of a block (1 where parts > 1)
    uint32_t parts;      // blocks of a group
    uint32_t n_blocks;
    uint32_t rows;       // pixels that a workgroup takes side by side
    uint32_t threads;
    uint32_t chunks;     // of an item
    uint32_t chunk_px;

    // vectors of a block, and its first
    __host__ __device__ uint32_t first_vec(uint32_t b) const {
        return parts == 1 ? b * gpb * vpg : (b / parts) * vpg + (b % parts) * kMaxVecs;
    }
    __host__ __device__ uint32_t vecs(uint32_t b) const {
        if (parts == 1) {
            const uint32_t left = n_groups - b * gpb;
            return (left < gpb ? left : gpb) * vpg;
        }
        const uint32_t left = vpg - (b % parts) * kMaxVecs;
        return left < kMaxVecs ? left : kMaxVecs;
    }
    __device__ uint32_t px_of(uint32_t chunk) const {
        const uint64_t left = n_px - (uint64_t)chunk * chunk_px;
        return left < chunk_px ? (uint32_t)left : chunk_px;
    }
};

Cut make_cut(uint32_t n_items, uint64_t n_px, uint32_t n_ch, uint32_t n_groups, uint32_t v) {
    Cut c{};
    c.n_px = n_px;
    c.n_items = n_items;
    c.n_ch = n_ch;
    c.n_groups = n_groups;
    c.vpg = n_ch / n_groups / v;
    c.parts = div_up(c.vpg, kMaxVecs);
    c.gpb = c.parts > 1 ? 1 : std::min(n_groups, kMaxVecs / c.vpg);
    c.n_blocks = c.parts > 1 ? n_groups * c.parts : div_up(n_groups, c.gpb);
    const uint32_t most = c.vecs(0);
    c.rows = std::max(1u, kMaxThreads / most);
    c.threads = div_up(c.rows * most, 64) * 64;
    const uint64_t others = (uint64_t)n_items * c.n_blocks;
    // chunks of 2^30 pixels at most
    const uint64_t want = std::max((kTargetGroups + others - 1) / others, (n_px >> 30) + 1);
    const uint64_t batch = (uint64_t)c.rows * kBatch;
    const uint64_t chunks = std::max<uint64_t>(1, std::min(want, (n_px + batch - 1) / batch));
    c.chunk_px = (uint32_t)((n_px + chunks - 1) / chunks + c.rows - 1) / c.rows * c.rows;
    c.chunks = (uint32_t)((n_px + c.chunk_px - 1) / c.chunk_px);
    return c;
}

// A thread's place: its vector of the block and the row of pixels it walks.
struct Place {
    uint32_t vec, row, nv;
    bool live;
    __device__ Place(const Cut& c) {
        nv = c.vecs(blockIdx.y);
        row = threadIdx.x / nv;
        vec = threadIdx.x - row * nv;
        live = row < c.rows;
    }
};

// (n, mean, squares about it) of two sets joined.
__device__ __forceinline__ void join(float& n, float& mean, float& m2, float nb, float meanb,
                                     float m2b) {
    const float sum = n + nb;
    if (nb > 0.f) {
        const float d = meanb - mean, share = nb / sum;
        mean = fmaf(d, share, mean);
        m2 += m2b + d * d * (n * share);
        n = sum;
    }
}

__device__ __forceinline__ uint32_t half_up(uint32_t n) {  // the power of two in [n / 2, n)
    return n <= 1 ? 0u : 1u << (31 - __builtin_clz(n - 1));
}

// ---------------------------------------------------------------------------
// activations
// ---------------------------------------------------------------------------

__device__ __forceinline__ float sigmoid(float z) {
    return 1.f / (1.f + __expf(-z));
}
__device__ __forceinline__ float gauss_cdf(float z) {
    return 0.5f * (1.f + erff(z * 0.70710678118654752f));
}

template <int V>
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
                z[j] *= gauss_cdf(z[j]);
            }
            break;
        default:
            break;
    }
}

// g times the activation's slope at z
template <int V>
__device__ __forceinline__ void act_slopes(uint32_t act, const float (&z)[V], float (&g)[V]) {
    switch (act) {
        case DRESSI_ACT_RELU:
#pragma unroll
            for (int j = 0; j < V; j++) {
                g[j] = z[j] > 0.f ? g[j] : 0.f * g[j];
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
                const float pdf = 0.39894228040143268f * __expf(-0.5f * z[j] * z[j]);
                g[j] *= fmaf(z[j], pdf, gauss_cdf(z[j]));
            }
            break;
        default:
            break;
    }
}

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------

template <typename T, int V>
__global__ __launch_bounds__(kMaxThreads) void k_gn_stats(const T* x, const Cut c, float2* part) {
    __shared__ float sn[kMaxThreads], smean[kMaxThreads], sm2[kMaxThreads];
    const Place at(c);
    const uint32_t item = blockIdx.x / c.chunks, chunk = blockIdx.x - item * c.chunks;
    float n = 0.f, mean = 0.f, m2 = 0.f;
    if (at.live) {
        const T* p = x + (size_t)item * c.item_stride +
                     ((size_t)chunk * c.chunk_px) * c.px_stride +
                     (size_t)(c.first_vec(blockIdx.y) + at.vec) * V;
        const uint32_t len = c.px_of(chunk);
        uint32_t i = at.row;
        for (; i + (kBatch - 1) * c.rows < len; i += kBatch * c.rows) {
            float v[kBatch][V];
#pragma unroll
            for (uint32_t k = 0; k < kBatch; k++) {
                load_vec<T, V>(p + (size_t)(i + k * c.rows) * c.px_stride, v[k]);
            }
            float s = 0.f, q = 0.f;
#pragma unroll
            for (uint32_t k = 0; k < kBatch; k++) {
#pragma unroll
                for (int j = 0; j < V; j++) {
                    s += v[k][j];
                }
            }
            s *= 1.f / (kBatch * V);
#pragma unroll
            for (uint32_t k = 0; k < kBatch; k++) {
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float d = v[k][j] - s;
                    q = fmaf(d, d, q);
                }
            }
            join(n, mean, m2, (float)(kBatch * V), s, q);
        }
        for (; i < len; i += c.rows) {
            float v[V], s = 0.f, q = 0.f;
            load_vec<T, V>(p + (size_t)i * c.px_stride, v);
#pragma unroll
            for (int j = 0; j < V; j++) {
                s += v[j];
            }
            s *= 1.f / V;
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float d = v[j] - s;
                q = fmaf(d, d, q);
            }
            join(n, mean, m2, (float)V, s, q);
        }
    }
    sn[threadIdx.x] = n;
    smean[threadIdx.x] = mean;
    sm2[threadIdx.x] = m2;
    __syncthreads();
    // over the rows, then over a group's vectors
    const uint32_t per = c.parts == 1 ? c.vpg : at.nv;
    const uint32_t j = at.vec % per;
    const auto take = [&](uint32_t from) {
        join(n, mean, m2, sn[from], smean[from], sm2[from]);
        sn[threadIdx.x] = n;
        smean[threadIdx.x] = mean;
        sm2[threadIdx.x] = m2;
    };
    for (uint32_t left = c.rows, s = half_up(left); s > 0; left = s, s = half_up(left)) {
        if (at.row < s && at.row + s < left) {
            take(threadIdx.x + s * at.nv);
        }
        __syncthreads();
    }
    for (uint32_t left = per, s = half_up(left); s > 0; left = s, s = half_up(left)) {
        if (at.row == 0 && j < s && j + s < left) {
            take(threadIdx.x + s);
        }
        __syncthreads();
    }
    if (at.row == 0 && j == 0) {
        const uint32_t slot = c.parts == 1 ? blockIdx.y * c.gpb + at.vec / per : blockIdx.y;
        part[((size_t)item * c.n_groups * c.parts + slot) * c.chunks + chunk] =
            make_float2(mean, m2);
    }
}

// Lanes that share the joining of one group's chunks: a power of two, so that
// the workgroup takes all of its groups at once.
__device__ __forceinline__ uint32_t lanes_of_group(uint32_t threads, uint32_t groups) {
    uint32_t l = 64;
    while (l > 1 && l * groups > threads) {
        l >>= 1;
    }
    return l;
}

// (mean, 1 / sqrt(var + eps)) of the block's groups into `stat`.
__device__ __forceinline__ void join_chunks(const Cut& c, uint32_t item, const float2* part,
                                            int v, float eps, float2* stat) {
    const uint32_t groups = c.parts == 1 ? c.vecs(blockIdx.y) / c.vpg : 1;
    const uint32_t first = c.parts == 1 ? blockIdx.y * c.gpb : blockIdx.y / c.parts;
    const uint32_t lanes = lanes_of_group(blockDim.x, groups);
    const uint32_t g = threadIdx.x / lanes, lane = threadIdx.x & (lanes - 1);
    float n = 0.f, mean = 0.f, m2 = 0.f;
    if (g < groups) {
        const uint32_t entries = c.parts * c.chunks;
        const float2* p =
            part + ((size_t)item * c.n_groups + first + g) * c.parts * c.chunks;
        const uint32_t b0 = (first + g) * c.parts;
        for (uint32_t e = lane; e < entries; e += lanes) {
            const uint32_t chunk = c.parts == 1 ? e : e % c.chunks;
            const uint32_t vecs = c.parts == 1 ? c.vpg : c.vecs(b0 + e / c.chunks);
            const float2 q = p[e];
            join(n, mean, m2, (float)c.px_of(chunk) * (float)(vecs * v), q.x, q.y);
        }
    }
    for (uint32_t o = 1; o < lanes; o <<= 1) {
        const float nb = __shfl_xor(n, o), meanb = __shfl_xor(mean, o), m2b = __shfl_xor(m2, o);
        // both lanes of a pair join in the same order
        if (threadIdx.x & o) {
            float na = nb, ma = meanb, qa = m2b;
            join(na, ma, qa, n, mean, m2);
            n = na, mean = ma, m2 = qa;
        } else {
            join(n, mean, m2, nb, meanb, m2b);
        }
    }
    if (g < groups && lane == 0) {
        stat[g] = make_float2(mean, 1.f / sqrtf(m2 / n + eps));
    }
    __syncthreads();
}

__device__ __forceinline__ float load_as_float(const void* p, uint32_t type, size_t i) {
    return type == DRESSI_F32    ? ((const float*)p)[i]
           : type == DRESSI_BF16 ? to_float(((const bf16*)p)[i])
                                 : to_float(((const f16*)p)[i]);
}
__device__ __forceinline__ void store_as(void* p, uint32_t type, size_t i, float x) {
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

template <int V>
__device__ __forceinline__ void load_affine(const Affine& a, uint32_t ch, float (&w)[V],
                                            float (&b)[V]) {
#pragma unroll
    for (int j = 0; j < V; j++) {
        w[j] = a.weight ? load_as_float(a.weight, a.type, ch + j) : 1.f;
        b[j] = a.bias ? load_as_float(a.bias, a.type, ch + j) : 0.f;
    }
}

template <typename T, int V>
__global__ __launch_bounds__(kMaxThreads) void k_gn_apply(const T* x, const Cut c,
                                                          const float2* part, const Affine aff,
                                                          float eps, uint32_t act, T* y,
                                                          float* mean_out, float* rstd_out) {
    __shared__ float2 stat[kMaxVecs];
    const Place at(c);
    const uint32_t item = blockIdx.x / c.chunks, chunk = blockIdx.x - item * c.chunks;
    join_chunks(c, item, part, V, eps, stat);
    if (!at.live) {
        return;
    }
    const uint32_t vec = c.first_vec(blockIdx.y) + at.vec;
    const float2 ms = stat[c.parts == 1 ? at.vec / c.vpg : 0];
    if (chunk == 0 && at.row == 0 && vec % c.vpg == 0) {
        mean_out[(size_t)item * c.n_groups + vec / c.vpg] = ms.x;
        rstd_out[(size_t)item * c.n_groups + vec / c.vpg] = ms.y;
    }
    float w[V], b[V];
    load_affine<V>(aff, vec * V, w, b);
#pragma unroll
    for (int j = 0; j < V; j++) {
        w[j] *= ms.y;
    }
    const size_t px0 = (size_t)chunk * c.chunk_px;
    const T* p = x + (size_t)item * c.item_stride + px0 * c.px_stride + (size_t)vec * V;
    T* o = y + ((size_t)item * c.n_px + px0) * c.n_ch + (size_t)vec * V;
    const uint32_t len = c.px_of(chunk);
    uint32_t i = at.row;
    for (; i + (kBatch - 1) * c.rows < len; i += kBatch * c.rows) {
        float v[kBatch][V];
#pragma unroll
        for (uint32_t k = 0; k < kBatch; k++) {
            load_vec<T, V>(p + (size_t)(i + k * c.rows) * c.px_stride, v[k]);
        }
#pragma unroll
        for (uint32_t k = 0; k < kBatch; k++) {
#pragma unroll
            for (int j = 0; j < V; j++) {
                v[k][j] = fmaf(v[k][j] - ms.x, w[j], b[j]);
            }
            act_values<V>(act, v[k]);
            store_vec<T, V>(o + (size_t)(i + k * c.rows) * c.n_ch, v[k]);
        }
    }
    for (; i < len; i += c.rows) {
        float v[V];
        load_vec<T, V>(p + (size_t)i * c.px_stride, v);
#pragma unroll
        for (int j = 0; j < V; j++) {
            v[j] = fmaf(v[j] - ms.x, w[j], b[j]);
        }
        act_values<V>(act, v);
        store_vec<T, V>(o + (size_t)i * c.n_ch, v);
    }
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------

// Per chunk the channels' (sum gz, sum gz xh), and the groups' sums of both
// weighted.
template <typename T, int V>
__global__ __launch_bounds__(kMaxThreads) void k_gn_bwd_sums(const T* gy, const T* x, const Cut c,
                                                             const Affine aff, uint32_t act,
                                                             const float* mean, const float* rstd,
                                                             float2* group_part,
                                                             float2* ch_part) {
    __shared__ float2 red[V][kMaxThreads];
    const Place at(c);
    const uint32_t item = blockIdx.x / c.chunks, chunk = blockIdx.x - item * c.chunks;
    const uint32_t vec = c.first_vec(blockIdx.y) + at.vec;
    float sa[V], sb[V], w[V], b[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        sa[j] = sb[j] = 0.f;
    }
    if (at.live) {
        load_affine<V>(aff, vec * V, w, b);
        const float mu = mean[(size_t)item * c.n_groups + vec / c.vpg];
        const float s = rstd[(size_t)item * c.n_groups + vec / c.vpg];
        const size_t px0 = (size_t)chunk * c.chunk_px;
        const T* p = x + (size_t)item * c.item_stride + px0 * c.px_stride + (size_t)vec * V;
        const T* q = gy + ((size_t)item * c.n_px + px0) * c.n_ch + (size_t)vec * V;
        const uint32_t len = c.px_of(chunk);
        const auto add = [&](float (&xv)[V], float (&gv)[V]) {
            float z[V];
#pragma unroll
            for (int j = 0; j < V; j++) {
                xv[j] = (xv[j] - mu) * s;
                z[j] = fmaf(xv[j], w[j], b[j]);
            }
            act_slopes<V>(act, z, gv);
#pragma unroll
            for (int j = 0; j < V; j++) {
                sa[j] += gv[j];
                sb[j] = fmaf(gv[j], xv[j], sb[j]);
            }
        };
        uint32_t i = at.row;
        for (; i + (kBatch - 1) * c.rows < len; i += kBatch * c.rows) {
            float xv[kBatch][V], gv[kBatch][V];
#pragma unroll
            for (uint32_t k = 0; k < kBatch; k++) {
                load_vec<T, V>(p + (size_t)(i + k * c.rows) * c.px_stride, xv[k]);
                load_vec<T, V>(q + (size_t)(i + k * c.rows) * c.n_ch, gv[k]);
            }
#pragma unroll
            for (uint32_t k = 0; k < kBatch; k++) {
                add(xv[k], gv[k]);
            }
        }
        for (; i < len; i += c.rows) {
            float xv[V], gv[V];
            load_vec<T, V>(p + (size_t)i * c.px_stride, xv);
            load_vec<T, V>(q + (size_t)i * c.n_ch, gv);
            add(xv, gv);
        }
    }
#pragma unroll
    for (int j = 0; j < V; j++) {
        red[j][threadIdx.x] = make_float2(sa[j], sb[j]);
    }
    __syncthreads();
    for (uint32_t left = c.rows, s = half_up(left); s > 0; left = s, s = half_up(left)) {
        if (at.row < s && at.row + s < left) {
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float2 o = red[j][threadIdx.x + s * at.nv];
                sa[j] += o.x;
                sb[j] += o.y;
                red[j][threadIdx.x] = make_float2(sa[j], sb[j]);
            }
        }
        __syncthreads();
    }
    const uint32_t per = c.parts == 1 ? c.vpg : at.nv;
    const uint32_t j0 = at.vec % per;
    float ga = 0.f, gb = 0.f;
    if (at.row == 0) {
        float2* o = ch_part + (size_t)blockIdx.x * c.n_ch + (size_t)vec * V;
#pragma unroll
        for (int j = 0; j < V; j++) {
            o[j] = make_float2(sa[j], sb[j]);
            ga = fmaf(w[j], sa[j], ga);
            gb = fmaf(w[j], sb[j], gb);
        }
        red[0][threadIdx.x] = make_float2(ga, gb);
    }
    __syncthreads();
    for (uint32_t left = per, s = half_up(left); s > 0; left = s, s = half_up(left)) {
        if (at.row == 0 && j0 < s && j0 + s < left) {
            const float2 o = red[0][threadIdx.x + s];
            ga += o.x;
            gb += o.y;
            red[0][threadIdx.x] = make_float2(ga, gb);
        }
        __syncthreads();
    }
    if (at.row == 0 && j0 == 0) {
        const uint32_t slot = c.parts == 1 ? blockIdx.y * c.gpb + at.vec / per : blockIdx.y;
        group_part[((size_t)item * c.n_groups * c.parts + slot) * c.chunks + chunk] =
            make_float2(ga, gb);
    }
}

template <typename T, int V>
__global__ __launch_bounds__(kMaxThreads) void k_gn_bwd_apply(const T* gy, const T* x, const Cut c,
                                                              const Affine aff, uint32_t act,
                                                              const float* mean, const float* rstd,
                                                              const float2* group_part, T* gx) {
    __shared__ float2 mean_of[kMaxVecs];
    const Place at(c);
    const uint32_t item = blockIdx.x / c.chunks, chunk = blockIdx.x - item * c.chunks;
    {
        const uint32_t groups = c.parts == 1 ? c.vecs(blockIdx.y) / c.vpg : 1;
        const uint32_t first = c.parts == 1 ? blockIdx.y * c.gpb : blockIdx.y / c.parts;
        const uint32_t lanes = lanes_of_group(blockDim.x, groups);
        const uint32_t g = threadIdx.x / lanes, lane = threadIdx.x & (lanes - 1);
        const uint32_t entries = c.parts * c.chunks;
        float a = 0.f, b = 0.f;
        if (g < groups) {
            const float2* p = group_part + ((size_t)item * c.n_groups + first + g) * entries;
            for (uint32_t e = lane; e < entries; e += lanes) {
                a += p[e].x;
                b += p[e].y;
            }
        }
        for (uint32_t o = 1; o < lanes; o <<= 1) {
            a += __shfl_xor(a, o);
            b += __shfl_xor(b, o);
        }
        if (g < groups && lane == 0) {
            const float m = 1.f / ((float)c.n_px * (float)(c.n_ch / c.n_groups));
            mean_of[g] = make_float2(a * m, b * m);
        }
        __syncthreads();
    }
    if (!at.live) {
        return;
    }
    const uint32_t vec = c.first_vec(blockIdx.y) + at.vec;
    const float2 ab = mean_of[c.parts == 1 ? at.vec / c.vpg : 0];
    const float mu = mean[(size_t)item * c.n_groups + vec / c.vpg];
    const float s = rstd[(size_t)item * c.n_groups + vec / c.vpg];
    float w[V], b[V];
    load_affine<V>(aff, vec * V, w, b);
    const size_t px0 = (size_t)chunk * c.chunk_px;
    const T* p = x + (size_t)item * c.item_stride + px0 * c.px_stride + (size_t)vec * V;
    const size_t at_out = ((size_t)item * c.n_px + px0) * c.n_ch + (size_t)vec * V;
    const T* q = gy + at_out;
    T* o = gx + at_out;
    const uint32_t len = c.px_of(chunk);
    const auto grad = [&](float (&xv)[V], float (&gv)[V]) {
        float z[V];
#pragma unroll
        for (int j = 0; j < V; j++) {
            xv[j] = (xv[j] - mu) * s;
            z[j] = fmaf(xv[j], w[j], b[j]);
        }
        act_slopes<V>(act, z, gv);
#pragma unroll
        for (int j = 0; j < V; j++) {
            gv[j] = s * (fmaf(gv[j], w[j], -ab.x) - xv[j] * ab.y);
        }
    };
    uint32_t i = at.row;
    for (; i + (kBatch - 1) * c.rows < len; i += kBatch * c.rows) {
        float xv[kBatch][V], gv[kBatch][V];
#pragma unroll
        for (uint32_t k = 0; k < kBatch; k++) {
            load_vec<T, V>(p + (size_t)(i + k * c.rows) * c.px_stride, xv[k]);
            load_vec<T, V>(q + (size_t)(i + k * c.rows) * c.n_ch, gv[k]);
        }
#pragma unroll
        for (uint32_t k = 0; k < kBatch; k++) {
            grad(xv[k], gv[k]);
            store_vec<T, V>(o + (size_t)(i + k * c.rows) * c.n_ch, gv[k]);
        }
    }
    for (; i < len; i += c.rows) {
        float xv[V], gv[V];
        load_vec<T, V>(p + (size_t)i * c.px_stride, xv);
        load_vec<T, V>(q + (size_t)i * c.n_ch, gv);
        grad(xv, gv);
        store_vec<T, V>(o + (size_t)i * c.n_ch, gv);
    }
}

// gw, gb: the chunks' channel sums over all items, in a fixed order; 32
// channels and 32 shares of the chunks a workgroup.
__global__ __launch_bounds__(1024) void k_gn_param_grad(const float2* ch_part, size_t n_rows,
                                                        uint32_t n_ch, uint32_t type, void* gw,
                                                        void* gb) {
    __shared__ double sa[32][33], sb[32][33];
    const uint32_t lane = threadIdx.x & 31u, row = threadIdx.x >> 5;
    const uint32_t ch = blockIdx.x * 32 + lane;
    double a = 0.0, b = 0.0;
    if (ch < n_ch) {
#pragma unroll 4
        for (size_t r = row; r < n_rows; r += 32) {
            const float2 q = ch_part[r * n_ch + ch];
            a += (double)q.x;
            b += (double)q.y;
        }
    }
    sa[row][lane] = a;
    sb[row][lane] = b;
    __syncthreads();
    for (uint32_t s = 16; s > 0; s >>= 1) {
        if (row < s) {
            sa[row][lane] += sa[row + s][lane];
            sb[row][lane] += sb[row + s][lane];
        }
        __syncthreads();
    }
    if (row == 0 && ch < n_ch) {
        if (gb) {
            store_as(gb, type, ch, (float)sa[0][lane]);
        }
        if (gw) {
            store_as(gw, type, ch, (float)sb[0][lane]);
        }
    }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

// The widest vector that a group's channels, the strides and the pointers
// allow, 16 bytes at most. A vector never straddles groups.
uint32_t vec_width(uint32_t type, uint32_t n_ch, uint32_t n_groups, uint64_t item_stride,
                   uint64_t px_stride, std::initializer_list<const void*> ptrs) {
    const uint32_t size = (uint32_t)type_bytes(type);
    uint64_t bits = (uint64_t)(n_ch / n_groups) | item_stride | px_stride | (16u / size);
    uint32_t v = (uint32_t)(bits & (~bits + 1));
    for (const void* p : ptrs) {
        while (v > 1 && (uintptr_t)p % ((size_t)v * size) != 0) {
            v >>= 1;
        }
    }
    return v;
}

struct Scratch {
    size_t group_part, ch_part, bytes;
};
Scratch scratch_of(const Cut& c, bool backward) {
    Scratch s;
    s.group_part = sizeof(float2) * (size_t)c.n_items * c.n_groups * c.parts * c.chunks;
    s.ch_part = backward ? sizeof(float2) * (size_t)c.n_items * c.chunks * c.n_ch : 0;
    s.bytes = s.group_part + s.ch_part;
    return s;
}

int check_shape(const char* what, uint32_t type, uint32_t n_items, uint64_t n_px, uint32_t n_ch,
                uint32_t n_groups, uint32_t act, const Affine& aff) {
    DRESSI_REQUIRE(type <= DRESSI_F16, "%s: unknown type %u", what, type);
    DRESSI_REQUIRE(aff.type <= DRESSI_F16, "%s: unknown type %u of the weight", what, aff.type);
    DRESSI_REQUIRE(act <= DRESSI_ACT_GELU, "%s: unknown activation %u", what, act);
    DRESSI_REQUIRE(n_ch <= (1u << 20), "%s: too many channels", what);
    DRESSI_REQUIRE(n_groups > 0 && n_ch % n_groups == 0 && n_ch > 0,
                   "%s: %u channels are not %u whole groups", what, n_ch, n_groups);
    DRESSI_REQUIRE(n_px <= (1ull << 40), "%s: too many pixels", what);
    DRESSI_REQUIRE(n_items <= (1u << 20), "%s: too many items", what);
    return DRESSI_OK;
}

template <typename F>
int for_width(uint32_t type, uint32_t v, F&& f) {
    switch (type) {
        case DRESSI_F32:
            return v == 4 ? f(Pack<float, 4>()) : v == 2 ? f(Pack<float, 2>()) : f(Pack<float, 1>());
        case DRESSI_BF16:
            return v == 8   ? f(Pack<bf16, 8>())
                   : v == 4 ? f(Pack<bf16, 4>())
                   : v == 2 ? f(Pack<bf16, 2>())
                            : f(Pack<bf16, 1>());
        default:
            return v == 8   ? f(Pack<f16, 8>())
                   : v == 4 ? f(Pack<f16, 4>())
                   : v == 2 ? f(Pack<f16, 2>())
                            : f(Pack<f16, 1>());
    }
}

template <typename T, int V>
int launch_forward(hipStream_t s, const Cut& c, const void* x, const Affine& aff, float eps,
                   uint32_t act, void* scratch, void* y, float* mean, float* rstd) {
    const dim3 grid(c.n_items * c.chunks, c.n_blocks), block(c.threads);
    hipLaunchKernelGGL((k_gn_stats<T, V>), grid, block, 0, s, (const T*)x, c, (float2*)scratch);
    DRESSI_CHECK_LAUNCH();
    hipLaunchKernelGGL((k_gn_apply<T, V>), grid, block, 0, s, (const T*)x, c,
                       (const float2*)scratch, aff, eps, act, (T*)y, mean, rstd);
    DRESSI_CHECK_LAUNCH();
    return DRESSI_OK;
}

template <typename T, int V>
int launch_backward(hipStream_t s, const Cut& c, const void* gy, const void* x, const Affine& aff,
                    uint32_t act, const float* mean, const float* rstd, void* scratch, void* gx,
                    void* gw, void* gb) {
    const dim3 grid(c.n_items * c.chunks, c.n_blocks), block(c.threads);
    float2* group_part = (float2*)scratch;
    float2* ch_part = (float2*)((char*)scratch + scratch_of(c, true).group_part);
    hipLaunchKernelGGL((k_gn_bwd_sums<T, V>), grid, block, 0, s, (const T*)gy, (const T*)x, c, aff,
                       act, mean, rstd, group_part, ch_part);
    DRESSI_CHECK_LAUNCH();
    if (gx) {
        hipLaunchKernelGGL((k_gn_bwd_apply<T, V>), grid, block, 0, s, (const T*)gy, (const T*)x, c,
                           aff, act, mean, rstd, group_part, (T*)gx);
        DRESSI_CHECK_LAUNCH();
    }
    if (gw || gb) {
        hipLaunchKernelGGL(k_gn_param_grad, dim3(div_up(c.n_ch, 32)), dim3(1024), 0, s, ch_part,
                           (size_t)c.n_items * c.chunks, c.n_ch, aff.type, gw, gb);
        DRESSI_CHECK_LAUNCH();
    }
    return DRESSI_OK;
}

}  // namespace
}  // namespace dressi

using namespace dressi;

extern "C" {

size_t dressi_group_norm_scratch(uint32_t type, uint32_t n_items, uint64_t n_px, uint32_t n_ch,
                                 uint32_t n_groups, int backward) {
    if (type > DRESSI_F16 || n_items == 0 || n_px == 0 || n_ch == 0 || n_groups == 0 ||
        n_ch % n_groups != 0) {
        return 0;
    }
    size_t most = 0;
    for (uint32_t v = 1; v <= 16u / type_bytes(type) && n_ch / n_groups % v == 0; v *= 2) {
        most = std::max(most,
                        scratch_of(make_cut(n_items, n_px, n_ch, n_groups, v), backward != 0).bytes);
    }
    return most;
}

int dressi_group_norm(dressi_ctx* ctx, const void* x, uint32_t type, uint32_t n_items,
                      uint64_t n_px, uint32_t n_ch, uint64_t item_stride, uint64_t px_stride,
                      uint32_t n_groups, const void* weight, const void* bias,
                      uint32_t affine_type, float eps, uint32_t activation, void* scratch,
                      size_t scratch_bytes, void* y, float* mean, float* rstd) {
    DRESSI_REQUIRE(ctx, "NULL context");
    const Affine aff{weight, bias, affine_type};
    if (int rc = check_shape("group_norm", type, n_items, n_px, n_ch, n_groups, activation, aff)) {
        return rc;
    }
    if (n_items == 0 || n_px == 0) {
        return DRESSI_OK;
    }
    DRESSI_REQUIRE(x && y && mean && rstd && scratch, "group_norm: bad arguments");
    DRESSI_REQUIRE(px_stride >= n_ch || n_px == 1, "group_norm: pixels overlap");
    const uint32_t v = vec_width(type, n_ch, n_groups, n_items > 1 ? item_stride : 0,
                                 n_px > 1 ? px_stride : 0, {x, y});
    Cut c = make_cut(n_items, n_px, n_ch, n_groups, v);
    c.item_stride = item_stride;
    c.px_stride = px_stride;
    DRESSI_REQUIRE(scratch_bytes >= scratch_of(c, false).bytes, "group_norm: scratch too small");
    return for_width(type, v, [&](auto w) {
        using T = std::remove_reference_t<decltype(w.v[0])>;
        return launch_forward<T, sizeof(w) / sizeof(T)>(ctx->stream, c, x, aff, eps, activation,
                                                        scratch, y, mean, rstd);
    });
}

int dressi_group_norm_bwd(dressi_ctx* ctx, const void* gy, const void* x, uint32_t type,
                          uint32_t n_items, uint64_t n_px, uint32_t n_ch, uint64_t item_stride,
                          uint64_t px_stride, uint32_t n_groups, const void* weight,
                          const void* bias, uint32_t affine_type, uint32_t activation,
                          const float* mean, const float* rstd, void* scratch,
                          size_t scratch_bytes, void* gx, void* gw, void* gb) {
    DRESSI_REQUIRE(ctx, "NULL context");
    const Affine aff{weight, bias, affine_type};
    if (int rc = check_shape("group_norm_bwd", type, n_items, n_px, n_ch, n_groups, activation,
                             aff)) {
        return rc;
    }
    if (n_items == 0 || n_px == 0) {
        // sums of nothing
        for (void* p : {gw, gb}) {
            if (p) {
                hipLaunchKernelGGL(k_gn_param_grad, dim3(div_up(n_ch, 32)), dim3(1024), 0,
                                   ctx->stream, nullptr, (size_t)0, n_ch, affine_type, p, nullptr);
                DRESSI_CHECK_LAUNCH();
            }
        }
        return DRESSI_OK;
    }
    DRESSI_REQUIRE(gy && x && mean && rstd && scratch, "group_norm_bwd: bad arguments");
    DRESSI_REQUIRE(px_stride >= n_ch || n_px == 1, "group_norm_bwd: pixels overlap");
    const uint32_t v = vec_width(type, n_ch, n_groups, n_items > 1 ? item_stride : 0,
                                 n_px > 1 ? px_stride : 0, {gy, x, gx});
    Cut c = make_cut(n_items, n_px, n_ch, n_groups, v);
    c.item_stride = item_stride;
    c.px_stride = px_stride;
    DRESSI_REQUIRE(scratch_bytes >= scratch_of(c, true).bytes, "group_norm_bwd: scratch too small");
    return for_width(type, v, [&](auto w) {
        using T = std::remove_reference_t<decltype(w.v[0])>;
        return launch_backward<T, sizeof(w) / sizeof(T)>(ctx->stream, c, gy, x, aff, activation,
                                                         mean, rstd, scratch, gx, gw, gb);
    });
}

}  // extern "C"
