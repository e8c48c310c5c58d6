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
// Memory bounds it: about 12 operations a value forward and 20 backward, 5 (with
// gelu 20) of them an exponential's. A group's channels lie side by side in a
// pixel, so a workgroup takes whole pixels of a run (a "chunk") of one item: a
// thread keeps one vector of V channels and walks the pixels. Two passes: one
// leaves each chunk's sums, the other begins by joining the chunks' sums of its
// item (every workgroup for itself) and then reads the image again. Reading it
// once would take a wait between the workgroups of one launch, which two such
// launches side by side could spend for ever; a small image, or a group of few
// pixels, is held by one workgroup and read once. What crosses the memory is
// each pass's images and nothing else (counters: 4 x 1024 x 1024 x 64 bfloat16,
// forward 537 MB read twice and written once).
//
// Statistics are those of x less a pivot, in two passes a thread's first value: a
// batch of its values gives its mean and the squares about that mean, both from
// registers, and (count, mean, squares) of two sets are joined; sets of several
// threads and chunks are added in double. So values far from zero lose nothing to cancellation. What
// passes between workgroups, and what one pass adds up, is less a pivot of the whole
// group. One far
// from the rest would round it to the distance (one pixel of 1024 x 1024 off by
// 10^4 deviations, as the pivot: the mean off by 4e-5 deviations), so that pivot is
// the middle one of three values.
//
// The times beside the choices below are those of graphs of 30 calls, replayed, both
// sides in turn; a kernel's own under the profiler are up to a microsecond longer.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "internal.h"
#include "norm_core.h"
#include "typed.h"

namespace dressi {
namespace {

constexpr uint32_t kMaxThreads = 512;
constexpr uint32_t kMaxVecs = 256;  // of a workgroup
constexpr uint32_t kMinPixels = 2;  // that a thread should have of a chunk
// Workgroups that a launch should have: two a compute unit. Each joins the sums of
// its item's chunks, so more of them cost one large item (512 x 512 x 64 bfloat16
// forward: 23 us with 512, 31 with 1024 of half the threads) and fewer leave loads
// unissued (2 x 512 x 512 x 66: forward 49 and backward 77 us with 512, 53 and 94
// with 256; 512 x 512 x 64 is level).
constexpr uint32_t kTargetGroups = 512;
// Pixels that a thread keeps in registers (one pass). A workgroup's reads are a
// block's few channels of each pixel, a cache line each: past 4096 pixels
// (backward, with three images: 2048) two passes over whole pixels take less,
// 9.3 us against 11.2 for 64 x 64 x 32 float32 backward, 10.8 against 16.5 for
// 64 x 64 x 64 bfloat16; forward they take 8.4 and 9.2 there, one pass 8.1 and 9.1.
constexpr uint32_t kHold = 8, kHoldBwd = 4;
constexpr uint32_t kItemThreads = 512;  // of a workgroup that holds its pixels

// How an image is cut. A vector of V channels lies in one group, or (split)
// over several, each channel then counting for itself: a thread has S = 1 or
// S = V sums. A unit is the fewest groups that whole vectors make up: one, or
// V over the powers of two in D. A block is a set of whole units or, where a
// unit of one group has more than kMaxVecs vectors, a part of it.
struct Cut {
    uint64_t n_px;
    uint64_t item_stride, px_stride;  // of x, in elements
    uint32_t n_items, n_ch, n_groups;
    uint32_t group_ch;   // channels of a group
    uint32_t unit_vecs;  // vectors of a unit
    uint32_t upb;        // units of a block (1 where parts > 1)
    uint32_t gpb;        // groups of a block (1 where parts > 1)
    uint32_t parts;      // blocks of a group
    uint32_t n_blocks;
    uint32_t rows;       // pixels that a workgroup takes side by side
    uint32_t lanes;      // one pass: of a row, a power of two
    uint32_t threads;
    uint32_t chunks;     // of an item
    uint32_t chunk_px;
    uint32_t stream;     // results go past the caches
    uint32_t keep_px;    // of a chunk, its last: what the first pass leaves in a cache

    // vectors of a block, and its first
    __host__ __device__ uint32_t first_vec(uint32_t b) const {
        return parts == 1 ? b * upb * unit_vecs : (b / parts) * unit_vecs + (b % parts) * kMaxVecs;
    }
    __host__ __device__ uint32_t vecs(uint32_t b) const {
        if (parts == 1) {
            const uint32_t left = n_groups - b * gpb;
            return left < gpb ? left * unit_vecs / (gpb / upb) : upb * unit_vecs;
        }
        const uint32_t left = unit_vecs - (b % parts) * kMaxVecs;
        return left < kMaxVecs ? left : kMaxVecs;
    }
    // groups of a block (or one, of which it is a part), and its first
    __device__ uint32_t groups(uint32_t b) const {
        const uint32_t left = n_groups - (parts == 1 ? b * gpb : b / parts);
        return left < gpb ? left : gpb;
    }
    __device__ uint32_t first_group(uint32_t b) const { return parts == 1 ? b * gpb : b / parts; }
    __device__ uint32_t px_of(uint32_t chunk) const {
        const uint64_t left = n_px - (uint64_t)chunk * chunk_px;
        return left < chunk_px ? (uint32_t)left : chunk_px;
    }
};

// The fields that follow from the channels, with `upb_most` units of a block at
// most; vectors of v channels.
Cut make_blocks(uint32_t n_items, uint64_t n_px, uint32_t n_ch, uint32_t n_groups, uint32_t v,
                uint32_t upb_most) {
    Cut c{};
    c.n_px = n_px;
    c.n_items = n_items;
    c.n_ch = n_ch;
    c.n_groups = n_groups;
    c.group_ch = n_ch / n_groups;
    uint32_t unit = 1;  // groups
    while (c.group_ch * unit % v != 0) {
        unit *= 2;
    }
    c.unit_vecs = c.group_ch * unit / v;
    c.parts = unit == 1 ? div_up(c.unit_vecs, kMaxVecs) : 1;
    c.upb = c.parts > 1 ? 1
                        : std::max(1u, std::min({n_groups / unit, kMaxVecs / c.unit_vecs, upb_most}));
    c.gpb = c.upb * unit;
    c.n_blocks = c.parts > 1 ? n_groups * c.parts : div_up(n_groups, c.gpb);
    return c;
}

// For two passes over the image.
Cut make_cut(uint32_t n_items, uint64_t n_px, uint32_t n_ch, uint32_t n_groups, uint32_t v) {
    Cut c = make_blocks(n_items, n_px, n_ch, n_groups, v, n_groups);
    const uint32_t most = c.vecs(0);
    c.rows = std::max(1u, kMaxThreads / most);
    c.threads = div_up(c.rows * most, 64) * 64;
    const uint64_t others = (uint64_t)n_items * c.n_blocks;
    // chunks of 2^30 pixels at most
    const uint64_t want = std::max((kTargetGroups + others - 1) / others, (n_px >> 30) + 1);
    const uint64_t batch = (uint64_t)c.rows * kMinPixels;
    const uint64_t chunks = std::max<uint64_t>(1, std::min(want, (n_px + batch - 1) / batch));
    c.chunk_px = (uint32_t)((n_px + chunks - 1) / chunks + c.rows - 1) / c.rows * c.rows;
    c.chunks = (uint32_t)((n_px + c.chunk_px - 1) / c.chunk_px);
    return c;
}

// For one pass: a workgroup holds all pixels of a block, at most `hold` vectors a
// thread; a row's vectors lie in one wave. chunks is 0 where they are too many.
// Blocks take as many groups as leave 256 workgroups: their reads are longer then.
// They are the launch's y, which ends at kMaxBatchItems; two passes, whose blocks
// hold 129 vectors at least or all groups, stay far below it.
Cut make_item_cut(uint32_t n_items, uint64_t n_px, uint32_t n_ch, uint32_t n_groups,
                  uint32_t v, uint32_t hold) {
    const uint64_t most = std::max<uint64_t>(1, (uint64_t)n_items * n_groups / 256);
    for (uint32_t gpb = (uint32_t)std::min<uint64_t>(most, n_groups); gpb > 0; gpb /= 2) {
        Cut c = make_blocks(n_items, n_px, n_ch, n_groups, v, gpb);
        if (c.vecs(0) > 64) {
            continue;
        }
        uint32_t lanes = 1;
        while (lanes < c.vecs(0)) {
            lanes *= 2;
        }
        c.rows = kItemThreads / lanes;
        if (n_px <= (uint64_t)c.rows * hold && c.n_blocks <= kMaxBatchItems) {
            // no more rows than pixels, in whole waves
            const uint64_t need = (n_px * lanes + 63) / 64 * 64;
            c.threads = (uint32_t)std::min<uint64_t>(kItemThreads, need);
            c.rows = c.threads / lanes;
            c.lanes = lanes;
            c.chunks = 1;
            c.chunk_px = (uint32_t)n_px;
            return c;
        }
    }
    return Cut{};
}

// Pixels of a thread in flight. Forward 4 of 16 bytes in one group (1024 x 1024 x
// 64 bfloat16 in 8 groups: 71 us, 78 with 8), else 8 (2 x 512 x 512 x 66 in 6: 50
// us, 51 with 4). Backward 4, of the widest vectors 2, whose registers leave too
// few waves else (1024 x 1024 x 64 bfloat16: 122 us, 126 with 4; eight of them in
// 16 groups: 903 and 918).
template <typename T, int V, int S>
constexpr uint32_t kBatchOf = S == 1 && sizeof(T) * V >= 16 ? 4 : 8;
template <int V>
constexpr uint32_t kBatchBwdOf = V == 8 ? 2 : 4;

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
    // pixels of a chunk that the thread takes: its row, then each c.rows on
    __device__ uint32_t pixels(const Cut& c, uint32_t chunk) const {
        const uint32_t len = c.px_of(chunk);
        return live && row < len ? (len - row + c.rows - 1) / c.rows : 0;
    }
};

__device__ __forceinline__ float2 shfl_xor(float2 x, uint32_t o) {
    return make_float2(__shfl_xor(x.x, o), __shfl_xor(x.y, o));
}
__device__ __forceinline__ double2 shfl_xor(double2 x, uint32_t o) {
    return make_double2(__shfl_xor(x.x, o), __shfl_xor(x.y, o));
}
__device__ __forceinline__ float shfl_xor(float x, uint32_t o) { return __shfl_xor(x, o); }

__device__ __forceinline__ void accumulate(float& a, float b) { a += b; }
template <typename N>
__device__ __forceinline__ void accumulate(N& a, N b) {
    a.x += b.x;
    a.y += b.y;
}

// (n, mean, squares about it) of two sets joined.
__device__ __forceinline__ void join(float& n, float& mean, float& m2, float nb, float meanb,
                                     float m2b, float share) {
    const float d = meanb - mean;
    mean = fmaf(d, share, mean);
    m2 += m2b + d * d * (n * share);
}

// Lanes that share one of n sums or groups, as a power of two: so many that the
// workgroup takes all of them at once if it can.
__device__ __forceinline__ uint32_t lanes_of(uint32_t n) {
    uint32_t shift = 6;
    while (shift > 0 && (n << shift) > blockDim.x) {
        shift--;
    }
    return shift;
}

// Sums over a workgroup. Each thread has left S entries, of its vector's channels
// or groups; sum k is that of terms(k)(s, thread, row), entry s of a thread, over
// the rows and the `per` entries k per .. of a row, counted through its vectors.
// use(k, sum) is called by the first of the lanes that take a sum; all threads
// call this.
template <int S, typename N, typename Terms, typename Use>
__device__ __forceinline__ void add_terms(uint32_t rows, uint32_t nv, uint32_t per, uint32_t n,
                                          Terms&& terms, Use&& use) {
    const uint32_t shift = lanes_of(n), lanes = 1u << shift, k0 = threadIdx.x >> shift;
    uint32_t side = shift;  // of the lanes, side by side over the rows
    while (side > 0 && (1u << side) >= 2 * rows) {
        side--;
    }
    const uint32_t lane = threadIdx.x & (lanes - 1), lr = 1u << side;
    for (uint32_t k = k0; k - k0 < n; k += blockDim.x >> shift) {
        N s{};
        if (k < n) {
            const auto term = terms(k);
            for (uint32_t q = lane >> side; q < per; q += lanes >> side) {
                const uint32_t entry = k * per + q, at = entry / S;
                for (uint32_t r = lane & (lr - 1); r < rows; r += lr) {
                    accumulate(s, term(entry - at * S, r * nv + at, r));
                }
            }
        }
        for (uint32_t o = 1; o < lanes; o <<= 1) {
            accumulate(s, shfl_xor(s, o));
        }
        if (k < n && lane == 0) {
            use(k, s);
        }
    }
}
// Of pairs in red[s][thread].
template <int S, uint32_t THREADS, typename Use>
__device__ __forceinline__ void add_all(const float2 (*red)[THREADS], uint32_t rows, uint32_t nv,
                                        uint32_t per, uint32_t n, Use&& use) {
    const auto term = [&](uint32_t s, uint32_t i, uint32_t) { return red[s][i]; };
    add_terms<S, float2>(rows, nv, per, n, [&](uint32_t) { return term; }, use);
}

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------

// A thread's first `count` of B vectors, less the pivots, joined to each of
// its S sets (n, mean, m2): their mean, then the squares about it.
template <typename T, int V, int S, int B>
__device__ __forceinline__ void add_batch(const Pack<T, V> (&v)[B], uint32_t count,
                                          const float (&pivot)[S], float& n, float (&mean)[S],
                                          float (&m2)[S]) {
    constexpr int W = V / S;
    const float values = (float)(count * W), inv = count == B ? 1.f / (B * W) : 1.f / values;
    float s[S], q[S];
#pragma unroll
    for (int g = 0; g < S; g++) {
        s[g] = q[g] = 0.f;
    }
#pragma unroll
    for (uint32_t k = 0; k < B; k++) {
        float x[V];
        unpack(v[k], x);
#pragma unroll
        for (int g = 0; g < S; g++) {
            float t = 0.f;
#pragma unroll
            for (int j = 0; j < W; j++) {
                t += x[g * W + j] - pivot[g];
            }
            s[g] += k < count ? t : 0.f;
        }
    }
#pragma unroll
    for (int g = 0; g < S; g++) {
        s[g] *= inv;
    }
#pragma unroll
    for (uint32_t k = 0; k < B; k++) {
        float x[V];
        unpack(v[k], x);
#pragma unroll
        for (int g = 0; g < S; g++) {
            float t = 0.f;
#pragma unroll
            for (int j = 0; j < W; j++) {
                const float d = (x[g * W + j] - pivot[g]) - s[g];
                t = fmaf(d, d, t);
            }
            q[g] += k < count ? t : 0.f;
        }
    }
    const float share = values * __builtin_amdgcn_rcpf(n + values);
#pragma unroll
    for (int g = 0; g < S; g++) {
        join(n, mean[g], m2[g], values, s[g], q[g], share);
    }
    n += values;
}

// B of a thread's pixels, `stride` elements apart; past `count` the last again.
template <typename T, int V, int B>
__device__ __forceinline__ void load_batch(const T* p, size_t stride, uint32_t count, bool stream,
                                           Pack<T, V> (&v)[B]) {
    if (stream) {
#pragma unroll
        for (uint32_t k = 0; k < B; k++) {
            v[k] = load_pack<T, V, true>(p + (k < count ? k : count - 1) * stride);
        }
    } else {
#pragma unroll
        for (uint32_t k = 0; k < B; k++) {
            v[k] = load_pack<T, V>(p + (k < count ? k : count - 1) * stride);
        }
    }
}

// What a group's values are taken less: the middle one of its first channel's
// values at three of the item's pixels, about a quarter of it apart and in no
// common column. What is far from the rest (a few pixels, a patch of them, a
// border) does not have two of the three. Loaded early and looked at late.
template <typename T>
struct Pivot {
    T v[3];
    __device__ __forceinline__ void load(const T* x, const Cut& c, uint32_t item, uint32_t group) {
        const T* p = x + (size_t)item * c.item_stride + (size_t)group * c.group_ch;
        v[0] = p[((c.n_px * 15467) >> 16) * c.px_stride];
        v[1] = p[((c.n_px * 33461) >> 16) * c.px_stride];
        v[2] = p[((c.n_px * 50159) >> 16) * c.px_stride];
    }
    __device__ __forceinline__ float value() const {
        return __builtin_amdgcn_fmed3f(to_float(v[0]), to_float(v[1]), to_float(v[2]));
    }
};

// Group (of the image) of set g of vector `vec`.
template <int V, int S>
__device__ __forceinline__ uint32_t group_of(const Cut& c, uint32_t vec, int g) {
    return (vec * V + g * (V / S)) / c.group_ch;
}

// The first pass: each chunk's (mean less the pivot, squares) for each group.
// 4 x 1024 x 1024 x 64 bfloat16: 84 us, 6.4 TB/s. A small image's time is that
// of a launch and of a few loads one after another: 512 x 512 x 64 10 us.
template <typename T, int V, int S>
__global__ __launch_bounds__(kMaxThreads) void k_gn_stats(const T* x, const Cut c, float2* part) {
    constexpr uint32_t kBatch = kBatchOf<T, V, S>;
    __shared__ float2 red[S][kMaxThreads];
    __shared__ float about[S][kMaxThreads];
    const Place at(c);
    const uint32_t item = blockIdx.x / c.chunks, chunk = blockIdx.x - item * c.chunks;
    const uint32_t vec = c.first_vec(blockIdx.y) + at.vec, group0 = c.first_group(blockIdx.y);
    float n = 0.f, mean[S], m2[S], pivot[S];
#pragma unroll
    for (int g = 0; g < S; g++) {
        mean[g] = m2[g] = pivot[g] = 0.f;
    }
    const uint32_t groups = c.groups(blockIdx.y), mine = threadIdx.x >> lanes_of(groups);
    Pivot<T> base;
    base.load(x, c, item, group0 + std::min(mine, groups - 1));
    uint32_t left = at.pixels(c, chunk);
    if (left > 0) {
        const T* p = x + (size_t)item * c.item_stride +
                     ((size_t)chunk * c.chunk_px + at.row) * c.px_stride + (size_t)vec * V;
        const size_t step = (size_t)c.rows * c.px_stride;
        const uint32_t keep = c.keep_px / c.rows;
        uint32_t count = left % kBatch ? left % kBatch : kBatch;
        while (left > 0) {
            Pack<T, V> v[kBatch];
            load_batch<T, V, kBatch>(p, step, count, left > keep, v);
#pragma unroll
            for (int g = 0; g < S; g++) {
                pivot[g] = n > 0.f ? pivot[g] : to_float(v[0].v[g * (V / S)]);
            }
            add_batch<T, V, S, kBatch>(v, count, pivot, n, mean, m2);
            left -= count;
            p += count * step;
            count = kBatch;
        }
    }
    const uint32_t len = c.px_of(chunk), entries = at.nv * S / groups;
    if (at.live) {
#pragma unroll
        for (int g = 0; g < S; g++) {
            red[g][threadIdx.x] = make_float2(mean[g], m2[g]);
            about[g][threadIdx.x] = pivot[g];
        }
    }
    __syncthreads();
    // the chunk's sums and squares about one of its pivots in double, where their
    // difference loses nothing to a thread's values far from the others'
    const auto pivot_of_group = [&](uint32_t k) {
        return (double)about[k * entries % S][k * entries / S];
    };
    const double values = (double)len * (double)(entries * (V / S));
    // of a thread: of the first len % rows rows, and of the others
    const uint32_t over = len % c.rows;
    const double most = (double)((len / c.rows + 1) * (V / S)), least = most - (double)(V / S);
    add_terms<S, double2>(
        c.rows, at.nv, entries, groups,
        [&](uint32_t k) {
            return [&, p = pivot_of_group(k)](uint32_t set, uint32_t i, uint32_t row) {
                const float2 x = red[set][i];
                const double m = ((double)about[set][i] - p) + (double)x.x;
                const double n = row < over ? most : least, s = n * m;
                return make_double2(s, fma(s, m, (double)x.y));
            };
        },
        [&](uint32_t k, double2 s) {
            const double d = s.x / values;
            if (k != mine) {
                base.load(x, c, item, group0 + k);
            }
            const uint32_t slot = c.parts == 1 ? group0 + k : blockIdx.y;
            part[((size_t)item * c.n_groups * c.parts + slot) * c.chunks + chunk] = make_float2(
                (float)(pivot_of_group(k) - (double)base.value() + d), (float)fma(-s.x, d, s.y));
        });
}

// (mean, 1 / sqrt(var + eps)) of the block's groups into `stat`: sums and
// squares about the pivot in double, where their difference loses nothing.
template <typename T, int V>
__device__ __forceinline__ void join_chunks(const T* x, const Cut& c, uint32_t item,
                                            const float2* part, float eps, float2* stat) {
    const uint32_t groups = c.groups(blockIdx.y), group0 = c.first_group(blockIdx.y);
    const uint32_t shift = lanes_of(groups), lanes = 1u << shift, g0 = threadIdx.x >> shift;
    const uint32_t lane = threadIdx.x & (lanes - 1);
    const double last = (double)c.px_of(c.chunks - 1);
    for (uint32_t g = g0; g - g0 < groups; g += blockDim.x >> shift) {
        double s = 0.0, q = 0.0;
        Pivot<T> pivot;
        if (g < groups) {
            pivot.load(x, c, item, group0 + g);
            const float2* p =
                part + ((size_t)item * c.n_groups + group0 + g) * c.parts * c.chunks;
            for (uint32_t k = 0; k < c.parts; k++, p += c.chunks) {
                const uint32_t ch = c.parts == 1 ? c.group_ch
                                                 : c.vecs((group0 + g) * c.parts + k) * V;
                const double full = (double)c.chunk_px * ch, less = last * ch;
#pragma unroll 8
                for (uint32_t e = lane; e < c.chunks; e += lanes) {
                    const double n = e == c.chunks - 1 ? less : full;
                    const double m = (double)p[e].x, nm = n * m;
                    s += nm;
                    q += fma(nm, m, (double)p[e].y);
                }
            }
        }
        for (uint32_t o = 1; o < lanes; o <<= 1) {
            s += __shfl_xor(s, o);
            q += __shfl_xor(q, o);
        }
        if (g < groups && lane == 0) {
            const double n = (double)c.n_px * c.group_ch, mean = s / n;
            const double m2 = q - s * mean;
            const float var = m2 < 0.0 ? 0.f : (float)(m2 / n);  // a NaN stays one
            stat[g] = make_float2((float)((double)pivot.value() + mean), 1.f / sqrtf(var + eps));
        }
    }
    __syncthreads();
}

// V results, past the caches where they are many (they would drive out what
// the next pass or item still reads).
template <typename T, int V>
__device__ __forceinline__ void put(T* p, const float (&x)[V], uint32_t stream) {
    if (stream) {
        store_vec<T, V, true>(p, x);
    } else {
        store_vec<T, V>(p, x);
    }
}

// act((x - mean) ws + b), ws = rstd w
template <typename T, int V, int S>
__device__ __forceinline__ void normalise(const Pack<T, V>& x, const float (&mean)[S],
                                          const float (&ws)[V], const float (&b)[V], uint32_t act,
                                          T* y, uint32_t stream) {
    float v[V];
    unpack(x, v);
#pragma unroll
    for (int j = 0; j < V; j++) {
        v[j] = fmaf(v[j] - mean[j / (V / S)], ws[j], b[j]);
    }
    act_values<T, V>(act, v);
    put<T, V>(y, v, stream);
}

// Workgroups of consecutive numbers run on the 8 dies in turn, each with an L2
// of its own: the k-th from the end of those on the same die.
__device__ __forceinline__ uint32_t backwards(uint32_t k, uint32_t n) {
    const uint32_t rounds = n / 8;
    return k < rounds * 8 ? (rounds - 1 - k / 8) * 8 + k % 8 : k;
}

// The second pass; 4 x 1024 x 1024 x 64 bfloat16: 192 us, 5.6 TB/s; 512 x 512 x
// 64: 14.9 us. It walks the image backwards, each part on the die that
// read it in the first pass: what was read last may still be in a cache (4 x 256
// x 256 x 64 float32, both passes: 34.2 us, 37.3 with the dies mixed).
template <typename T, int V, int S>
__global__ __launch_bounds__(kMaxThreads) void k_gn_apply(const T* x, const Cut c,
                                                          const float2* part, const Affine aff,
                                                          float eps, uint32_t act, T* y,
                                                          float* mean_out, float* rstd_out) {
    constexpr uint32_t kBatch = kBatchOf<T, V, S>;
    __shared__ float2 stat[S * kMaxVecs];
    const Place at(c);
    const uint32_t unit = backwards(blockIdx.x, gridDim.x);
    const uint32_t item = unit / c.chunks, chunk = unit - item * c.chunks;
    uint32_t left = at.pixels(c, chunk);
    const uint32_t vec = c.first_vec(blockIdx.y) + at.vec, group0 = c.first_group(blockIdx.y);
    const size_t px0 = (size_t)chunk * c.chunk_px + at.row;
    const T* p = x + (size_t)item * c.item_stride + px0 * c.px_stride + (size_t)vec * V;
    T* o = y + ((size_t)item * c.n_px + px0) * c.n_ch + (size_t)vec * V;
    const size_t step = (size_t)c.rows * c.px_stride, ostep = (size_t)c.rows * c.n_ch;
    // the first batch and the weights are on their way while the chunks are joined
    Pack<T, V> v[kBatch];
    uint32_t count = left < kBatch ? left : kBatch;
    const uint32_t all = left, keep = c.keep_px / c.rows;
    float w[V], b[V], mean[S];
    if (left > 0) {
        load_batch<T, V, kBatch>(p + (left - count) * step, step, count, keep == 0, v);
        load_affine<V>(aff, vec * V, w, b);
    }
    join_chunks<T, V>(x, c, item, part, eps, stat);
    if (chunk == 0 && (c.parts == 1 || blockIdx.y % c.parts == 0)) {
        for (uint32_t g = threadIdx.x; g < c.groups(blockIdx.y); g += blockDim.x) {
            mean_out[(size_t)item * c.n_groups + group0 + g] = stat[g].x;
            rstd_out[(size_t)item * c.n_groups + group0 + g] = stat[g].y;
        }
    }
    if (left == 0) {
        return;
    }
#pragma unroll
    for (int g = 0; g < S; g++) {
        const float2 ms = stat[group_of<V, S>(c, vec, g) - group0];
        mean[g] = ms.x;
#pragma unroll
        for (int j = 0; j < V / S; j++) {
            w[g * (V / S) + j] *= ms.y;
        }
    }
    while (true) {
        left -= count;
#pragma unroll
        for (uint32_t k = 0; k < kBatch; k++) {
            if (k < count) {
                normalise<T, V, S>(v[k], mean, w, b, act, o + (left + k) * ostep, c.stream);
            }
        }
        if (left == 0) {
            break;
        }
        count = left < kBatch ? left : kBatch;
        load_batch<T, V, kBatch>(p + (left - count) * step, step, count, all - left >= keep, v);
    }
}

// A thread's place in one pass: `lanes` lanes of a wave take a row, so that a
// sum over rows is one over lanes and then over waves.
struct ItemPlace {
    uint32_t vec, row, mine;
    __device__ ItemPlace(const Cut& c) {
        vec = threadIdx.x & (c.lanes - 1);
        row = threadIdx.x / c.lanes;
        const uint32_t len = (uint32_t)c.n_px;
        mine = vec < c.vecs(blockIdx.y) && row < len ? (len - row + c.rows - 1) / c.rows : 0;
    }
};

// The sum of `s` over the thread's group; every thread calls it, those without
// pixels with 0. `part` is not reused before the next barrier but one.
template <typename N>
__device__ __forceinline__ N add_item(const Cut& c, const ItemPlace& at, N s, N (*part)[64]) {
    const uint32_t waves = blockDim.x / 64, wave = threadIdx.x / 64, per = c.unit_vecs;
    const bool even = (per & (per - 1)) == 0;
    for (uint32_t o = c.lanes; o < 64; o *= 2) {
        accumulate(s, shfl_xor(s, o));
    }
    if (even) {
        for (uint32_t o = 1; o < per; o *= 2) {
            accumulate(s, shfl_xor(s, o));
        }
    }
    if ((threadIdx.x & 63u) < c.lanes) {
        part[wave][at.vec] = s;
    }
    __syncthreads();
    if (even) {
        N sum = part[0][at.vec];
        for (uint32_t i = 1; i < waves; i++) {
            accumulate(sum, part[i][at.vec]);
        }
        return sum;
    }
    if (threadIdx.x < c.lanes) {
        N sum = part[0][at.vec];
        for (uint32_t i = 1; i < waves; i++) {
            accumulate(sum, part[i][at.vec]);
        }
        part[0][at.vec] = sum;
    }
    __syncthreads();
    const uint32_t first = at.vec / per * per;
    N sum = part[0][first];
    for (uint32_t i = 1; i < per; i++) {
        // a lane past the block's vectors reads on within the row
        accumulate(sum, part[0][(first + i) & 63u]);
    }
    return sum;
}

// Both passes where a block's pixels fit its workgroup's registers: x is read
// once, in one launch. 8 x 32 x 32 x 256 bfloat16: 7.6 us, 10.1 in two passes;
// 16 x 16 x 32 float32: 4.3 and 7.9.
template <typename T, int V>
__global__ __launch_bounds__(kItemThreads) void k_gn_item(const T* x, const Cut c,
                                                          const Affine aff, float eps,
                                                          uint32_t act, T* y, float* mean_out,
                                                          float* rstd_out) {
    __shared__ float part[2][kItemThreads / 64][64];
    const ItemPlace at(c);
    const uint32_t vec = c.first_vec(blockIdx.y) + at.vec, group = vec / c.unit_vecs;
    const uint32_t item = blockIdx.x;
    const T* p = x + (size_t)item * c.item_stride + (size_t)at.row * c.px_stride + (size_t)vec * V;
    T* o = y + ((size_t)item * c.n_px + at.row) * c.n_ch + (size_t)vec * V;
    const size_t step = (size_t)c.rows * c.px_stride, ostep = (size_t)c.rows * c.n_ch;
    Pack<T, V> v[kHold];
#pragma unroll
    for (uint32_t k = 0; k < kHold; k++) {
        if (k < at.mine) {
            v[k] = load_pack<T, V>(p + k * step);
        }
    }
    float w[V], b[V], pivot = 0.f;
    if (at.mine > 0) {
        Pivot<T> p3;
        p3.load(x, c, item, group);
        load_affine<V>(aff, vec * V, w, b);
        pivot = p3.value();
    }
    const float values = (float)c.n_px * (float)c.group_ch;
    float s = 0.f, q = 0.f;
#pragma unroll
    for (uint32_t k = 0; k < kHold; k++) {
        if (k < at.mine) {
            float f[V];
            unpack(v[k], f);
#pragma unroll
            for (int j = 0; j < V; j++) {
                s += f[j] - pivot;
            }
        }
    }
    const float d_mean = add_item(c, at, s, part[0]) / values;
#pragma unroll
    for (uint32_t k = 0; k < kHold; k++) {
        if (k < at.mine) {
            float f[V];
            unpack(v[k], f);
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float d = (f[j] - pivot) - d_mean;
                q = fmaf(d, d, q);
            }
        }
    }
    const float rstd = 1.f / sqrtf(add_item(c, at, q, part[1]) / values + eps);
    if (at.mine == 0) {
        return;
    }
    const float mean[1] = {pivot + d_mean};
    if (at.row == 0 && at.vec % c.unit_vecs == 0) {
        mean_out[(size_t)item * c.n_groups + group] = mean[0];
        rstd_out[(size_t)item * c.n_groups + group] = rstd;
    }
#pragma unroll
    for (int j = 0; j < V; j++) {
        w[j] *= rstd;
    }
#pragma unroll
    for (uint32_t k = 0; k < kHold; k++) {
        if (k < at.mine) {
            normalise<T, V, 1>(v[k], mean, w, b, act, o + k * ostep, c.stream);
        }
    }
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------

// What a thread of the backward pass knows of its channels; ws = rstd w. With it
// z is rounded as in the forward pass, so that relu's mask is that of its y, and
// gx = ws gz - mean_g(ws gz) - xh mean_g(ws gz xh) takes two operations.
template <int V, int S>
struct Channels {
    float mu[S], rstd[S], ws[V], b[V];

    __device__ __forceinline__ void load(const Cut& c, const Affine& aff, uint32_t item,
                                         uint32_t vec, const float* mean, const float* rs) {
        load_affine<V>(aff, vec * V, ws, b);
#pragma unroll
        for (int g = 0; g < S; g++) {
            const size_t at = (size_t)item * c.n_groups + group_of<V, S>(c, vec, g);
            mu[g] = mean[at];
            rstd[g] = rs[at];
        }
#pragma unroll
        for (int j = 0; j < V; j++) {
            ws[j] *= rstd[j / (V / S)];
        }
    }
    // xh and gz of a vector
    template <typename T>
    __device__ __forceinline__ void gradients(const Pack<T, V>& x, const Pack<T, V>& gy,
                                              uint32_t act, float (&xh)[V], float (&gz)[V]) const {
        float z[V];
        unpack(x, xh);
        unpack(gy, gz);
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float d = xh[j] - mu[j / (V / S)];
            xh[j] = d * rstd[j / (V / S)];
            z[j] = fmaf(d, ws[j], b[j]);
        }
        act_slopes<T, V>(act, z, gz);
    }
    template <typename T>
    __device__ __forceinline__ void add(const Pack<T, V>& x, const Pack<T, V>& gy, uint32_t act,
                                        float (&sa)[V], float (&sb)[V]) const {
        float xh[V], gz[V];
        gradients(x, gy, act, xh, gz);
#pragma unroll
        for (int j = 0; j < V; j++) {
            sa[j] += gz[j];
            sb[j] = fmaf(gz[j], xh[j], sb[j]);
        }
    }
    // gx from the groups' means of ws gz and ws gz xh
    template <typename T>
    __device__ __forceinline__ void finish(const Pack<T, V>& x, const Pack<T, V>& gy, uint32_t act,
                                           const float2 (&m)[S], T* gx, uint32_t stream) const {
        float xh[V], gz[V];
        gradients(x, gy, act, xh, gz);
#pragma unroll
        for (int j = 0; j < V; j++) {
            const int g = j / (V / S);
            gz[j] = fmaf(-xh[j], m[g].y, fmaf(gz[j], ws[j], -m[g].x));
        }
        put<T, V>(gx, gz, stream);
    }
};

// The first pass: per chunk the groups' sums of ws gz and ws gz xh, and for all
// chunks of a workgroup the channels' sums of gz and gz xh. 4 x 1024 x 1024 x 64
// bfloat16: 170 us, 6.3 TB/s. MANY: it takes every gridDim.x-th chunk of all
// items'; else it has one, and a set of sums less in its registers.
template <typename T, int V, int S, bool MANY>
__global__ __launch_bounds__(kMaxThreads) void k_gn_bwd_sums(const T* gy, const T* x, const Cut c,
                                                             const Affine aff, uint32_t act,
                                                             const float* mean, const float* rstd,
                                                             float2* group_part,
                                                             float2* ch_part) {
    constexpr uint32_t kBatchBwd = kBatchBwdOf<V>;
    __shared__ float2 red[V][kMaxThreads];
    const Place at(c);
    const uint32_t vec = c.first_vec(blockIdx.y) + at.vec;
    const uint32_t groups = c.groups(blockIdx.y), group0 = c.first_group(blockIdx.y);
    const size_t step = (size_t)c.rows * c.px_stride, qstep = (size_t)c.rows * c.n_ch;
    float a[V], b[V], sa[V], sb[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        sa[j] = sb[j] = 0.f;
    }
    for (uint32_t unit = blockIdx.x; unit < c.n_items * c.chunks; unit += gridDim.x) {
        const uint32_t item = unit / c.chunks, chunk = unit - item * c.chunks;
#pragma unroll
        for (int j = 0; j < V; j++) {
            a[j] = b[j] = 0.f;
        }
        Channels<V, S> ch;
        uint32_t left = at.pixels(c, chunk);
        if (left > 0) {
            ch.load(c, aff, item, vec, mean, rstd);
            const size_t px0 = (size_t)chunk * c.chunk_px + at.row;
            const T* p = x + (size_t)item * c.item_stride + px0 * c.px_stride + (size_t)vec * V;
            const T* q = gy + ((size_t)item * c.n_px + px0) * c.n_ch + (size_t)vec * V;
            const uint32_t keep = c.keep_px / c.rows;
            uint32_t count = left % kBatchBwd ? left % kBatchBwd : kBatchBwd;
            while (left > 0) {
                Pack<T, V> xv[kBatchBwd], gv[kBatchBwd];
                load_batch<T, V, kBatchBwd>(p, step, count, left > keep, xv);
                load_batch<T, V, kBatchBwd>(q, qstep, count, left > keep, gv);
#pragma unroll
                for (uint32_t k = 0; k < kBatchBwd; k++) {
                    if (k < count) {
                        ch.add(xv[k], gv[k], act, a, b);
                    }
                }
                left -= count;
                p += count * step;
                q += count * qstep;
                count = kBatchBwd;
            }
        }
        if (at.live) {
#pragma unroll
            for (int g = 0; g < S; g++) {
                float2 s = make_float2(0.f, 0.f);
                if (at.pixels(c, chunk) > 0) {
#pragma unroll
                    for (int j = g * (V / S); j < (g + 1) * (V / S); j++) {
                        s.x = fmaf(ch.ws[j], a[j], s.x);
                        s.y = fmaf(ch.ws[j], b[j], s.y);
                    }
                }
                red[g][threadIdx.x] = s;
            }
        }
#pragma unroll
        for (int j = 0; MANY && j < V; j++) {
            sa[j] += a[j];
            sb[j] += b[j];
        }
        __syncthreads();
        add_all<S, kMaxThreads>(red, c.rows, at.nv, at.nv * S / groups, groups,
                                [&](uint32_t k, float2 s) {
            const uint32_t slot = c.parts == 1 ? group0 + k : blockIdx.y;
            group_part[((size_t)item * c.n_groups * c.parts + slot) * c.chunks + chunk] = s;
        });
        __syncthreads();
        if (!MANY) {
            break;
        }
    }
#pragma unroll
    for (int j = 0; j < V; j++) {
        red[j][threadIdx.x] = MANY ? make_float2(sa[j], sb[j]) : make_float2(a[j], b[j]);
    }
    __syncthreads();
    float2* o = ch_part + (size_t)blockIdx.x * c.n_ch + (size_t)c.first_vec(blockIdx.y) * V;
    add_all<V, kMaxThreads>(red, c.rows, at.nv, 1, at.nv * V,
                            [&](uint32_t k, float2 s) { o[k] = s; });
}

// gw and gb of kParamCh channels: the chunks' sums over all items in a fixed
// order, the workgroup's threads taking shares of the chunks.
constexpr uint32_t kParamCh = 8;
struct ParamGrad {
    const float2* ch_part;
    size_t n_rows;
    uint32_t n_ch, type;
    void* gw;
    void* gb;
};

__device__ __forceinline__ void param_grad(const ParamGrad& a, uint32_t block) {
    __shared__ double2 sum[kMaxThreads / 64][kParamCh];
    const uint32_t lane = threadIdx.x % kParamCh, row = threadIdx.x / kParamCh;
    const uint32_t ch = block * kParamCh + lane;
    double2 s = make_double2(0.0, 0.0);
    if (ch < a.n_ch) {
#pragma unroll 8
        for (size_t r = row; r < a.n_rows; r += blockDim.x / kParamCh) {
            const float2 q = a.ch_part[r * a.n_ch + ch];
            s.x += (double)q.x;
            s.y += (double)q.y;
        }
    }
    for (uint32_t o = kParamCh; o < 64; o *= 2) {
        s.x += __shfl_xor(s.x, o);
        s.y += __shfl_xor(s.y, o);
    }
    if ((threadIdx.x & 63u) < kParamCh) {
        sum[threadIdx.x / 64][lane] = s;
    }
    __syncthreads();
    if (row == 0 && ch < a.n_ch) {
        for (uint32_t r = 1; r < blockDim.x / 64; r++) {
            s.x += sum[r][lane].x;
            s.y += sum[r][lane].y;
        }
        if (a.gb) {
            store_one(a.gb, a.type, ch, (float)s.x);
        }
        if (a.gw) {
            store_one(a.gw, a.type, ch, (float)s.y);
        }
    }
}

__global__ __launch_bounds__(kMaxThreads) void k_gn_param_grad(const ParamGrad a) {
    param_grad(a, blockIdx.x);
}

// The second pass, backwards like the forward one; 4 x 1024 x 1024 x 64 bfloat16:
// 287 us, 5.6 TB/s. The last `extra` columns of workgroups take gw and gb.
template <typename T, int V, int S>
__global__ __launch_bounds__(kMaxThreads) void k_gn_bwd_apply(const T* gy, const T* x, const Cut c,
                                                              const Affine aff, uint32_t act,
                                                              const float* mean, const float* rstd,
                                                              const float2* group_part, T* gx,
                                                              const ParamGrad params,
                                                              uint32_t extra) {
    constexpr uint32_t kBatchBwd = kBatchBwdOf<V>;
    __shared__ float2 mean_of[S * kMaxVecs];
    const uint32_t units = gridDim.x - extra;
    if (blockIdx.x >= units) {
        param_grad(params, (blockIdx.x - units) * gridDim.y + blockIdx.y);
        return;
    }
    const Place at(c);
    const uint32_t unit = backwards(blockIdx.x, units);
    const uint32_t item = unit / c.chunks, chunk = unit - item * c.chunks;
    uint32_t left = at.pixels(c, chunk);
    const uint32_t vec = c.first_vec(blockIdx.y) + at.vec, group0 = c.first_group(blockIdx.y);
    const size_t px0 = (size_t)chunk * c.chunk_px + at.row;
    const T* p = x + (size_t)item * c.item_stride + px0 * c.px_stride + (size_t)vec * V;
    const size_t at_out = ((size_t)item * c.n_px + px0) * c.n_ch + (size_t)vec * V;
    const T* q = gy + at_out;
    T* o = gx + at_out;
    const size_t step = (size_t)c.rows * c.px_stride, qstep = (size_t)c.rows * c.n_ch;
    Pack<T, V> xv[kBatchBwd], gv[kBatchBwd];
    uint32_t count = left < kBatchBwd ? left : kBatchBwd;
    const uint32_t all = left, keep = c.keep_px / c.rows;
    Channels<V, S> ch;
    if (left > 0) {
        load_batch<T, V, kBatchBwd>(p + (left - count) * step, step, count, keep == 0, xv);
        load_batch<T, V, kBatchBwd>(q + (left - count) * qstep, qstep, count, keep == 0, gv);
        ch.load(c, aff, item, vec, mean, rstd);
    }
    {
        const uint32_t groups = c.groups(blockIdx.y), entries = c.parts * c.chunks;
        const uint32_t shift = lanes_of(groups), lanes = 1u << shift, g0 = threadIdx.x >> shift;
        const uint32_t lane = threadIdx.x & (lanes - 1);
        const float inv = 1.f / ((float)c.n_px * (float)c.group_ch);
        for (uint32_t g = g0; g - g0 < groups; g += blockDim.x >> shift) {
            float2 s = make_float2(0.f, 0.f);
            if (g < groups) {
                const float2* e0 = group_part + ((size_t)item * c.n_groups + group0 + g) * entries;
#pragma unroll 8
                for (uint32_t e = lane; e < entries; e += lanes) {
                    accumulate(s, e0[e]);
                }
            }
            for (uint32_t d = 1; d < lanes; d <<= 1) {
                accumulate(s, shfl_xor(s, d));
            }
            if (g < groups && lane == 0) {
                mean_of[g] = make_float2(s.x * inv, s.y * inv);
            }
        }
        __syncthreads();
    }
    if (left == 0) {
        return;
    }
    float2 m[S];
#pragma unroll
    for (int g = 0; g < S; g++) {
        m[g] = mean_of[group_of<V, S>(c, vec, g) - group0];
    }
    while (true) {
        left -= count;
#pragma unroll
        for (uint32_t k = 0; k < kBatchBwd; k++) {
            if (k < count) {
                ch.finish(xv[k], gv[k], act, m, o + (left + k) * qstep, c.stream);
            }
        }
        if (left == 0) {
            break;
        }
        count = left < kBatchBwd ? left : kBatchBwd;
        const bool past = all - left >= keep;
        load_batch<T, V, kBatchBwd>(p + (left - count) * step, step, count, past, xv);
        load_batch<T, V, kBatchBwd>(q + (left - count) * qstep, qstep, count, past, gv);
    }
}

// Both passes where a block's pixels fit its workgroup's registers. A workgroup
// takes every gridDim.x-th item; ch_part (null for one workgroup a block: gw
// and gb are whole then) gets its items' channel sums. 8 x 32 x 32 x 256
// bfloat16: 11.8 us with the launch that adds them, 12.6 in two passes.
template <typename T, int V>
__global__ __launch_bounds__(kItemThreads) void k_gn_bwd_item(
        const T* gy, const T* x, const Cut c, const Affine aff, uint32_t act, const float* mean,
        const float* rstd, float2* ch_part, T* gx, void* gw, void* gb) {
    __shared__ float2 part[2][kItemThreads / 64][64];
    __shared__ float2 red[V][kItemThreads];
    const ItemPlace at(c);
    const uint32_t vec = c.first_vec(blockIdx.y) + at.vec;
    const size_t step = (size_t)c.rows * c.px_stride, qstep = (size_t)c.rows * c.n_ch;
    const float inv = 1.f / ((float)c.n_px * (float)c.group_ch);
    float sa[V], sb[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        sa[j] = sb[j] = 0.f;
    }
    Channels<V, 1> ch;
    uint32_t turn = 0;
    for (uint32_t item = blockIdx.x; item < c.n_items; item += gridDim.x, turn ^= 1) {
        const T* p = x + (size_t)item * c.item_stride + (size_t)at.row * c.px_stride +
                     (size_t)vec * V;
        const size_t at_out = ((size_t)item * c.n_px + at.row) * c.n_ch + (size_t)vec * V;
        const T* q = gy + at_out;
        Pack<T, V> xv[kHoldBwd], gv[kHoldBwd];
#pragma unroll
        for (uint32_t k = 0; k < kHoldBwd; k++) {
            if (k < at.mine) {
                xv[k] = load_pack<T, V>(p + k * step);
                gv[k] = load_pack<T, V>(q + k * qstep);
            }
        }
        float2 g = make_float2(0.f, 0.f);
        if (at.mine > 0) {
            float a[V], b[V];
#pragma unroll
            for (int j = 0; j < V; j++) {
                a[j] = b[j] = 0.f;
            }
            ch.load(c, aff, item, vec, mean, rstd);
#pragma unroll
            for (uint32_t k = 0; k < kHoldBwd; k++) {
                if (k < at.mine) {
                    ch.add(xv[k], gv[k], act, a, b);
                }
            }
#pragma unroll
            for (int j = 0; j < V; j++) {
                g.x = fmaf(ch.ws[j], a[j], g.x);
                g.y = fmaf(ch.ws[j], b[j], g.y);
                sa[j] += a[j];
                sb[j] += b[j];
            }
        }
        g = add_item(c, at, g, part[turn]);
        if (at.mine > 0 && gx) {
            const float2 m[1] = {make_float2(g.x * inv, g.y * inv)};
#pragma unroll
            for (uint32_t k = 0; k < kHoldBwd; k++) {
                if (k < at.mine) {
                    ch.finish(xv[k], gv[k], act, m, gx + at_out + k * qstep, c.stream);
                }
            }
        }
    }
    if (!ch_part && !gw && !gb) {
        return;
    }
#pragma unroll
    for (int j = 0; j < V; j++) {
        red[j][threadIdx.x] = make_float2(sa[j], sb[j]);
    }
    __syncthreads();
    const uint32_t ch0 = c.first_vec(blockIdx.y) * V;
    add_all<V, kItemThreads>(red, c.rows, c.lanes, 1, c.vecs(blockIdx.y) * V,
                             [&](uint32_t k, float2 s) {
        if (ch_part) {
            ch_part[(size_t)blockIdx.x * c.n_ch + ch0 + k] = s;
            return;
        }
        if (gb) {
            store_one(gb, aff.type, ch0 + k, s.x);
        }
        if (gw) {
            store_one(gw, aff.type, ch0 + k, s.y);
        }
    });
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

// How wide a thread's vectors are: 16 bytes at most, as the channels, the strides
// and the images' addresses (or-ed) allow. `whole`: that no group's edge cuts. One
// pass takes whole ones, two passes wider ones where there are (their channels
// count apart then: 2 x 512 x 512 x 66 bfloat16 in 6 groups, forward: 50 us with
// vectors of 2 cut by edges, 73 with single channels).
struct Width {
    uint32_t any, whole;
};
Width vec_width(uint32_t type, uint32_t n_ch, uint32_t n_groups, uint64_t item_stride,
                uint64_t px_stride, uint64_t addresses) {
    const uint32_t size = (uint32_t)type_bytes(type);
    const auto low_bit = [](uint64_t x) { return (uint32_t)(x & (~x + 1)); };
    const uint32_t v =
        low_bit((uint64_t)n_ch | item_stride | px_stride | addresses / size | (16u / size));
    const uint32_t group_ch = n_ch / n_groups, whole = std::min(v, low_bit(group_ch));
    // a unit of several groups has to fit a workgroup
    const uint32_t unit = v / whole;
    return {unit > 1 && group_ch * unit / v > kMaxVecs ? whole : v, whole};
}

// Workgroups of a block whose channel sums are added afterwards: few, where
// the units (chunks, or items in one pass) are many.
uint32_t sum_rows(uint64_t units, const Cut& c) {
    const uint64_t most = std::max(1u, 2048 / c.n_blocks);
    const uint64_t each = (units + most - 1) / most;
    return (uint32_t)((units + each - 1) / each);
}

// Bytes of the chunks' and of the channels' sums.
struct Scratch {
    size_t group_part, ch_part, bytes;
};
Scratch scratch_of(const Cut& c, bool whole, bool backward) {
    Scratch s;
    s.group_part =
        whole ? 0 : sizeof(float2) * (size_t)c.n_items * c.n_groups * c.parts * c.chunks;
    s.ch_part = backward ? sizeof(float2) * sum_rows((uint64_t)c.n_items * c.chunks, c) * c.n_ch : 0;
    s.bytes = s.group_part + s.ch_part;
    return s;
}

// Bytes of an image from which results go past the caches. Forward with them and
// without takes 70 and 88 us for 1024 x 1024 x 64 bfloat16, 23.3 and 24.8 for
// 512 x 512 x 64; with a pass after it that reads the result 125 and 127, 37 and 37.
constexpr uint64_t kStreamBytes = 32ull << 20;

// Bytes of the first pass's reads that the second may find in the last-level cache
// (256 MB): the ends of the chunks. The rest goes past it both times: 8 x 1024 x
// 1024 x 64 bfloat16 560 us forward and 904 backward, 573 and 1063 with all of it
// through the caches; all past them 1024 x 1024 x 64 takes 80 us forward, not 72.
// 96 and 224 MB kept measure the same.
constexpr uint64_t kKeepBytes = 160ull << 20;

// How a call is cut: in one pass if it can be.
struct Plan {
    Cut c;
    uint32_t v;
    bool whole, split;
};
Plan make_plan(uint32_t type, uint32_t n_items, uint64_t n_px, uint32_t n_ch, uint64_t item_stride,
               uint64_t px_stride, uint32_t n_groups, uint64_t addresses, uint32_t hold,
               uint32_t images) {
    const Width w = vec_width(type, n_ch, n_groups, n_items > 1 ? item_stride : 0,
                              n_px > 1 ? px_stride : 0, addresses);
    Plan p;
    p.v = w.whole;
    p.split = false;
    p.c = make_item_cut(n_items, n_px, n_ch, n_groups, w.whole, hold);
    p.whole = p.c.chunks != 0;
    if (!p.whole) {
        p.v = w.any;
        p.split = w.any != w.whole;
        p.c = make_cut(n_items, n_px, n_ch, n_groups, w.any);
    }
    p.c.item_stride = item_stride;
    p.c.px_stride = px_stride;
    const uint64_t bytes = (uint64_t)n_items * n_px * n_ch * type_bytes(type);
    p.c.stream = bytes >= kStreamBytes;
    const uint64_t again = bytes * images;  // of the second pass's reads
    p.c.keep_px = again <= kKeepBytes ? p.c.chunk_px
                                      : (uint32_t)(p.c.chunk_px * ((double)kKeepBytes / again));
    return p;
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
    DRESSI_REQUIRE(n_items <= (1u << 31), "%s: too many items", what);
    return DRESSI_OK;
}

// f(a vector's type, whether a group's edge may cut it)
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
int launch_item(hipStream_t s, const Cut& c, const void* x, const Affine& aff, float eps,
                uint32_t act, void* y, float* mean, float* rstd) {
    const uint32_t most = (uint32_t)(kLaunchThreads / kItemThreads);  // items of a launch
    for (uint32_t i = 0; i < c.n_items; i += most) {
        hipLaunchKernelGGL((k_gn_item<T, V>), dim3(std::min(most, c.n_items - i), c.n_blocks),
                           dim3(c.threads), 0, s, (const T*)x + (size_t)i * c.item_stride, c, aff,
                           eps, act, (T*)y + (size_t)i * c.n_px * c.n_ch,
                           mean + (size_t)i * c.n_groups, rstd + (size_t)i * c.n_groups);
        DRESSI_CHECK_LAUNCH();
    }
    return DRESSI_OK;
}

// Items of a launch whose workgroups each take a chunk of one.
uint32_t items_at_once(const Cut& c) {
    return (uint32_t)std::max<uint64_t>(1, kLaunchThreads / kMaxThreads / c.chunks);
}

template <typename T, int V, int S>
int launch_forward(hipStream_t s, const Cut& c, const void* x, const Affine& aff, float eps,
                   uint32_t act, void* scratch, void* y, float* mean, float* rstd) {
    const uint32_t most = items_at_once(c);
    for (uint32_t i = 0; i < c.n_items; i += most) {
        const dim3 grid(std::min(most, c.n_items - i) * c.chunks, c.n_blocks), block(c.threads);
        const T* xi = (const T*)x + (size_t)i * c.item_stride;
        hipLaunchKernelGGL((k_gn_stats<T, V, S>), grid, block, 0, s, xi, c, (float2*)scratch);
        DRESSI_CHECK_LAUNCH();
        hipLaunchKernelGGL((k_gn_apply<T, V, S>), grid, block, 0, s, xi, c, (const float2*)scratch,
                           aff, eps, act, (T*)y + (size_t)i * c.n_px * c.n_ch,
                           mean + (size_t)i * c.n_groups, rstd + (size_t)i * c.n_groups);
        DRESSI_CHECK_LAUNCH();
    }
    return DRESSI_OK;
}

int launch_param_grad(hipStream_t s, const ParamGrad& a) {
    hipLaunchKernelGGL(k_gn_param_grad, dim3(div_up(a.n_ch, kParamCh)), dim3(kMaxThreads), 0, s, a);
    DRESSI_CHECK_LAUNCH();
    return DRESSI_OK;
}

template <typename T, int V>
int launch_bwd_item(hipStream_t s, const Cut& c, const void* gy, const void* x, const Affine& aff,
                    uint32_t act, const float* mean, const float* rstd, void* scratch, void* gx,
                    void* gw, void* gb) {
    const uint32_t rows = sum_rows(c.n_items, c);
    const bool sums = rows > 1 && (gw || gb);  // the workgroups' are added afterwards
    hipLaunchKernelGGL((k_gn_bwd_item<T, V>), dim3(rows, c.n_blocks), dim3(c.threads), 0, s,
                       (const T*)gy, (const T*)x, c, aff, act, mean, rstd,
                       sums ? (float2*)scratch : nullptr, (T*)gx, gw, gb);
    DRESSI_CHECK_LAUNCH();
    return sums ? launch_param_grad(s, ParamGrad{(const float2*)scratch, rows, c.n_ch, aff.type,
                                                 gw, gb})
                : DRESSI_OK;
}

template <typename T, int V, int S>
int launch_backward(hipStream_t s, const Cut& c, const void* gy, const void* x, const Affine& aff,
                    uint32_t act, const float* mean, const float* rstd, void* scratch, void* gx,
                    void* gw, void* gb) {
    const uint32_t rows = sum_rows((uint64_t)c.n_items * c.chunks, c);
    const dim3 block(c.threads);
    float2* group_part = (float2*)scratch;
    float2* ch_part = (float2*)((char*)scratch + scratch_of(c, false, true).group_part);
    const ParamGrad params{ch_part, rows, c.n_ch, aff.type, gw, gb};
    const auto sums = rows < (uint64_t)c.n_items * c.chunks ? k_gn_bwd_sums<T, V, S, true>
                                                            : k_gn_bwd_sums<T, V, S, false>;
    hipLaunchKernelGGL(sums, dim3(rows, c.n_blocks), block, 0, s, (const T*)gy, (const T*)x, c,
                       aff, act, mean, rstd, group_part, ch_part);
    DRESSI_CHECK_LAUNCH();
    if (!gx) {
        return gw || gb ? launch_param_grad(s, params) : DRESSI_OK;
    }
    const uint32_t most = items_at_once(c);
    for (uint32_t i = 0; i < c.n_items; i += most) {
        const uint32_t items = std::min(most, c.n_items - i);
        const uint32_t extra = i + items == c.n_items && (gw || gb) ? div_up(div_up(c.n_ch, kParamCh), c.n_blocks) : 0;
        const size_t at = (size_t)i * c.n_px * c.n_ch, g = (size_t)i * c.n_groups;
        hipLaunchKernelGGL((k_gn_bwd_apply<T, V, S>), dim3(items * c.chunks + extra, c.n_blocks),
                           block, 0, s, (const T*)gy + at,
                           (const T*)x + (size_t)i * c.item_stride, c, aff, act, mean + g,
                           rstd + g, group_part + g * c.parts * c.chunks, (T*)gx + at, params,
                           extra);
        DRESSI_CHECK_LAUNCH();
    }
    return DRESSI_OK;
}

}  // namespace
}  // namespace dressi

using namespace dressi;

extern "C" {

size_t dressi_group_norm_scratch(uint32_t type, uint32_t n_items, uint64_t n_px, uint32_t n_ch,
                                 uint64_t item_stride, uint64_t px_stride, uint32_t n_groups,
                                 uint64_t addresses, int backward) {
    if (type > DRESSI_F16 || n_items == 0 || n_px == 0 || n_ch == 0 || n_groups == 0 ||
        n_ch % n_groups != 0) {
        return 0;
    }
    const Plan p = make_plan(type, n_items, n_px, n_ch, item_stride, px_stride, n_groups,
                             addresses, backward ? kHoldBwd : kHold, backward ? 2 : 1);
    return scratch_of(p.c, p.whole, backward != 0).bytes;
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
    DRESSI_REQUIRE(eps >= 0.f && std::isfinite(eps), "group_norm: eps %g", (double)eps);
    if (n_items == 0 || n_px == 0) {
        return DRESSI_OK;
    }
    DRESSI_REQUIRE(x && y && mean && rstd, "group_norm: bad arguments");
    DRESSI_REQUIRE(px_stride >= n_ch || n_px == 1, "group_norm: pixels overlap");
    const uint64_t addresses = (uintptr_t)x | (uintptr_t)y;
    DRESSI_REQUIRE(addresses % type_bytes(type) == 0, "group_norm: not aligned to its type");
    const Plan p = make_plan(type, n_items, n_px, n_ch, item_stride, px_stride, n_groups,
                             addresses, kHold, 1);
    const size_t need = scratch_of(p.c, p.whole, false).bytes;
    DRESSI_REQUIRE(need == 0 || (scratch && scratch_bytes >= need), "group_norm: scratch too small");
    return for_width(type, p.v, [&](auto w) {
        using T = std::remove_reference_t<decltype(w.v[0])>;
        constexpr int V = sizeof(w) / sizeof(T);
        hipStream_t s = ctx->stream;
        return p.whole ? launch_item<T, V>(s, p.c, x, aff, eps, activation, y, mean, rstd)
               : p.split
                   ? launch_forward<T, V, V>(s, p.c, x, aff, eps, activation, scratch, y, mean, rstd)
                   : launch_forward<T, V, 1>(s, p.c, x, aff, eps, activation, scratch, y, mean,
                                             rstd);
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
    if (!gx && !gw && !gb) {
        return DRESSI_OK;
    }
    if (n_items == 0 || n_px == 0) {
        // sums of nothing
        return gw || gb ? launch_param_grad(ctx->stream,
                                            ParamGrad{nullptr, 0, n_ch, affine_type, gw, gb})
                        : DRESSI_OK;
    }
    DRESSI_REQUIRE(gy && x && mean && rstd, "group_norm_bwd: bad arguments");
    DRESSI_REQUIRE(px_stride >= n_ch || n_px == 1, "group_norm_bwd: pixels overlap");
    const uint64_t addresses = (uintptr_t)gy | (uintptr_t)x | (uintptr_t)gx;
    DRESSI_REQUIRE(addresses % type_bytes(type) == 0, "group_norm_bwd: not aligned to its type");
    const Plan p = make_plan(type, n_items, n_px, n_ch, item_stride, px_stride, n_groups,
                             addresses, kHoldBwd, 2);
    DRESSI_REQUIRE(scratch && scratch_bytes >= scratch_of(p.c, p.whole, true).bytes,
                   "group_norm_bwd: scratch too small");
    return for_width(type, p.v, [&](auto w) {
        using T = std::remove_reference_t<decltype(w.v[0])>;
        constexpr int V = sizeof(w) / sizeof(T);
        hipStream_t s = ctx->stream;
        return p.whole ? launch_bwd_item<T, V>(s, p.c, gy, x, aff, activation, mean, rstd, scratch,
                                               gx, gw, gb)
               : p.split ? launch_backward<T, V, V>(s, p.c, gy, x, aff, activation, mean, rstd,
                                                    scratch, gx, gw, gb)
                         : launch_backward<T, V, 1>(s, p.c, gy, x, aff, activation, mean, rstd,
                                                    scratch, gx, gw, gb);
    });
}

}  // extern "C"
