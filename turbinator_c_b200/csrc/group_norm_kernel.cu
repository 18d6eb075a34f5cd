/*
 * Group norm with an activation, channels last: forward and backward
 * (include/turbinator/training/cuda_learner.h).
 *
 * Bound: HBM, given that x (and dy) are read once.  A tile is some positions of
 * some whole groups of one sample; a CTA keeps a tile in shared memory, filled
 * by asynchronous copies, so that mean, variance about that mean, and result
 * come from one read.  Threads form rows of `lanes` packs, each thread keeping
 * its channels over all its positions.
 *
 *   - A sample's groups that fit one tile, or the tiles of one cluster (8 CTAs),
 *     take one kernel: the tiles' statistics meet in distributed shared memory.
 *   - Larger maps take three: each tile's statistics, their merge, and the
 *     result from a second read, last tiles first, while they are in L2.
 *   - A group of more channels than a CTA has threads times its pack takes a
 *     CTA of its own and reads three times, value by value: 1 x 20,000 x 272 bf16
 *     on odd rows 6.6 ms, of which a split over the positions would leave little.
 *
 * 4,096 maps of 256 x 64 bf16, silu: forward 61 us (4.4 TB/s), backward 143 us
 * (2.8 TB/s: neither DRAM, at a third, nor issue, at half, is full; a tile's
 * loads, sums and stores follow each other, and registers and shared memory
 * leave two CTAs an SM); 8 maps of 65,536 x 128: 87 us.
 *
 * Statistics of tiles merge by counts, means and squares about the own mean, so
 * that a mean far from zero costs no digits.  Per-channel sums are the common
 * step of both directions: a pack may cross groups.
 */
#include <cooperative_groups.h>

#include "tb_learner.cuh"

namespace cg = cooperative_groups;
using namespace tb_learn;

namespace {

constexpr int kThreads = 128;         /* of a CTA */
constexpr int kBackwardThreads = 256;
constexpr int kCluster = 8; /* CTAs of a cluster at most */

struct NormShape {
    size_t samples, positions;
    int channels, groups, per_group;
    size_t xs, xp, ys, yp, gs, gp; /* strides of samples and positions: x; y and dy; dx */
    int act;
    float epsilon;
};

/* Tiles of a sample: `parts` of the positions by `blocks` of whole groups. */
struct Tiling {
    int pack;                /* elements of a load */
    int block_groups, lanes; /* groups and packs of a tile's row */
    int blocks, threads, rows_at_once;
    int rows, parts;         /* positions of a part */
    int turns;               /* packs of a thread that the tile has room for */
    int share;               /* threads that add up a channel's total: a power of two */
    bool folds;              /* rows of a warp fold by shuffles: lanes divides 32 */
    int sum_rows;            /* rows of partial sums that meet in shared memory */
    unsigned magic_parts, magic_blocks, magic_lanes, magic_rows, magic_group; /* floor((2^32 - 1) / ..), rows: rows_at_once */
    bool fits;               /* the parts fit one cluster */
    size_t tiles;            /* of all samples */
};

template <class V, int N> __device__ __forceinline__ void activate(V (&u)[N], int act) {
    if (act == TB_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = vmul(u[i], vsigmoid(u[i]));
    } else if (act == TB_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = veach(u[i], [](float v) { return v > 0.0f || v != v ? v : 0.0f; });
    } else if (act == TB_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = veach(u[i], [](float v) { return 0.5f * v * (1.0f + erff(v * 0.70710678f)); });
    }
}

/* u becomes the activation's slope there. */
template <class V, int N> __device__ __forceinline__ void slopes(V (&u)[N], int act) {
    if (act == TB_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < N; ++i) { /* s (1 + u (1 - s)) */
            const V s = vsigmoid(u[i]);
            const V t = vfma(s, vall<V>(-1.0f), vall<V>(1.0f));
            u[i] = vmul(s, vfma(u[i], t, vall<V>(1.0f)));
        }
    } else if (act == TB_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = veach(u[i], [](float v) { return v > 0.0f ? 1.0f : 0.0f; });
    } else if (act == TB_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            u[i] = veach(u[i], [](float v) {
                return 0.5f * (1.0f + erff(v * 0.70710678f)) + v * expf(-0.5f * v * v) * 0.39894228f;
            });
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = vall<V>(1.0f);
    }
}

/* ---- a tile ---- */

/* Where a CTA and its thread are. */
struct Seat {
    unsigned n;
    int part, block, lane, row, c0; /* c0: the tile's first channel */
    int first, rows;                /* the tile's first position, its positions */
    int mine;                       /* positions of the thread */
    int groups, channels;           /* of the tile: fewer in a sample's last block */
    bool in;                        /* the thread has a place in the rows */
};

__device__ __forceinline__ Seat seat_of(const NormShape &d, const Tiling &g, unsigned tile) {
    Seat s;
    const unsigned whole = divided(tile, g.parts, g.magic_parts);
    s.part = static_cast<int>(tile - whole * g.parts); /* the parts of a cluster are neighbours */
    s.n = divided(whole, g.blocks, g.magic_blocks);
    s.block = static_cast<int>(whole - s.n * g.blocks);
    s.c0 = s.block * g.block_groups * d.per_group;
    s.row = static_cast<int>(divided(threadIdx.x, g.lanes, g.magic_lanes));
    s.lane = static_cast<int>(threadIdx.x) - s.row * g.lanes;
    s.first = s.part * g.rows;
    s.rows = min(static_cast<int>(d.positions) - s.first, g.rows);
    s.groups = min(g.block_groups, d.groups - s.block * g.block_groups);
    s.channels = s.groups * d.per_group;
    s.in = s.row < g.rows_at_once && s.lane * g.pack < s.channels;
    s.mine = s.in && s.row < s.rows
                 ? static_cast<int>(divided(s.rows - s.row + g.rows_at_once - 1, g.rows_at_once, g.magic_rows)) : 0;
    return s;
}

template <class T, int PACK> __device__ __forceinline__ void copy_pack(Held<T, PACK> *to, const T *from) {
    const uint32_t t = static_cast<uint32_t>(__cvta_generic_to_shared(to));
    if constexpr (PACK * sizeof(T) == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(t), "l"(from) : "memory");
    else if constexpr (PACK * sizeof(T) == 4)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(t), "l"(from) : "memory");
    else
        *to = *reinterpret_cast<const Held<T, PACK> *>(from);
}

/* Starts copying the thread's packs into its places of the tile (to[i * STEP]
 * is its i-th; STEP: of the widest CTA, so that places are known offsets); it
 * reads no others, so that its own wait will do. */
template <int STEP, class T, int PACK>
__device__ __forceinline__ void load_tile(Held<T, PACK> *to, const T *p, size_t stride, const Seat &s, const Tiling &g) {
    p += (s.first + s.row) * stride + s.c0 + s.lane * PACK;
    const size_t jump = g.rows_at_once * stride;
#pragma unroll 4
    for (int i = 0; i < s.mine; ++i) {
        copy_pack<T, PACK>(to, p);
        to += STEP;
        p += jump;
    }
}
__device__ __forceinline__ void tile_loaded() { asm volatile("cp.async.wait_all;" ::: "memory"); }

/* Per-channel values of a thread. */
template <int PACK> struct Channels {
    Array<PACK> v;
};
/* f(channel of the tile) for each of the thread's; of its first where it has none. */
template <int PACK, class F> __device__ __forceinline__ Channels<PACK> channels_of(const Seat &s, F &&f) {
    float t[PACK];
#pragma unroll
    for (int k = 0; k < PACK; ++k) t[k] = f(s.in ? s.lane * PACK + k : 0);
    Channels<PACK> r;
#pragma unroll
    for (int k = 0; k < Values<PACK>::kCount; ++k) r.v[k] = vload<typename Values<PACK>::V>(t + 2 * k);
    return r;
}
__device__ __forceinline__ int group_of(int channel, const NormShape &d, const Tiling &g) {
    return static_cast<int>(divided(channel, d.per_group, g.magic_group));
}

/* The same for f(group of the tile): once where packs do not cross groups. */
template <int PACK, class F>
__device__ __forceinline__ Channels<PACK> by_group(const Seat &s, const NormShape &d, const Tiling &g, F &&f) {
    using V = typename Values<PACK>::V;
    if (d.per_group % PACK) return channels_of<PACK>(s, [&](int c) { return f(group_of(c, d, g)); });
    const V v = vall<V>(f(s.in ? group_of(s.lane * PACK, d, g) : 0));
    Channels<PACK> r;
#pragma unroll
    for (int k = 0; k < Values<PACK>::kCount; ++k) r.v[k] = v;
    return r;
}
template <int PACK> __device__ __forceinline__ Channels<PACK> times(const Channels<PACK> &a, const Channels<PACK> &b) {
    Channels<PACK> r;
#pragma unroll
    for (int k = 0; k < Values<PACK>::kCount; ++k) r.v[k] = vmul(a.v[k], b.v[k]);
    return r;
}
/* Parameters of the thread's channels, or `other` where there are none. */
template <int PACK> __device__ __forceinline__ Channels<PACK> parameters_of(const Seat &s, const float *p, float other) {
    return channels_of<PACK>(s, [&](int c) { return p ? p[s.c0 + c] : other; });
}

template <class T, int PACK>
__device__ __forceinline__ void taken(const Held<T, PACK> &h, Array<PACK> &v) {
    float e[PACK];
    unpack(h, e);
#pragma unroll
    for (int k = 0; k < Values<PACK>::kCount; ++k) v[k] = vload<typename Values<PACK>::V>(e + 2 * k);
}
template <class T, int PACK> __device__ __forceinline__ void put(T *to, const Array<PACK> &v) {
    float e[PACK];
#pragma unroll
    for (int k = 0; k < Values<PACK>::kCount; ++k) vstore(e + 2 * k, v[k]);
    *reinterpret_cast<Held<T, PACK> *>(to) = packed<T, PACK>(e);
}

/* ---- sums over a tile ---- */

/* Shared memory of a tile: rows of per-channel partial sums, of N values a
 * channel, their totals, backward the channels' scale, per group four values,
 * and the tile (x, then du). */
struct Sums {
    float *rows, *channel, *scale, *group;
    unsigned char *tile;
    int channels, pitch; /* channels of a row, to whole 16 bytes; of N rows of them and a shift of banks */
};
template <int N> __device__ __forceinline__ Sums sums_of(float *shared, const Tiling &g) {
    Sums s;
    s.channels = (g.lanes * g.pack + 3) & ~3;
    s.pitch = N * s.channels + 4;
    s.rows = shared;
    s.channel = shared + g.sum_rows * s.pitch;
    s.scale = s.channel + N * s.channels;
    s.group = s.scale + (N > 1 ? s.channels : 0);
    s.tile = reinterpret_cast<unsigned char *>(s.group + 4 * g.block_groups);
    return s;
}
/* n: values a channel, 1 forward and 2 backward, where du is kept too, in f32. */
size_t shared_bytes(const Tiling &g, size_t size, int n, bool du) {
    const size_t channels = (static_cast<size_t>(g.lanes) * g.pack + 3) & ~size_t(3);
    const size_t places = static_cast<size_t>(g.turns) * (n > 1 ? kBackwardThreads : kThreads) * g.pack;
    return (g.sum_rows * (n * channels + 4) + (n > 1 ? n + 1 : n) * channels + 4 * g.block_groups) * sizeof(float) +
           places * (size + (du ? sizeof(float) : 0));
}

/* channel[i * s.channels + c] = the sum over the CTA's rows of each thread's
 * own[i]; ends with the totals visible to all. */
template <int PACK, int N>
__device__ __forceinline__ void channel_totals(const Array<PACK> (&own)[N], const Sums &s, const Seat &at, const Tiling &g) {
    float e[N][PACK];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int k = 0; k < Values<PACK>::kCount; ++k) vstore(e[i] + 2 * k, own[i][k]);
    bool leaves = at.in;
    int row = at.row;
    if (g.folds) {
        for (int o = g.lanes; o < 32; o *= 2)
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int v = 0; v < PACK; ++v) e[i][v] += __shfl_xor_sync(0xffffffffu, e[i][v], o);
        leaves = at.in && threadIdx.x % 32 < g.lanes;
        row = threadIdx.x / 32;
    }
    if (leaves) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float *to = s.rows + row * s.pitch + i * s.channels + at.lane * PACK;
            if constexpr (PACK % 4 == 0) {
#pragma unroll
                for (int v = 0; v < PACK; v += 4)
                    *reinterpret_cast<float4 *>(to + v) = make_float4(e[i][v], e[i][v + 1], e[i][v + 2], e[i][v + 3]);
            } else {
#pragma unroll
                for (int v = 0; v < PACK; ++v) to[v] = e[i][v];
            }
        }
    }
    __syncthreads();
    /* g.share neighbouring threads for each total */
    const int mine = threadIdx.x & (g.share - 1), each = blockDim.x / g.share;
    for (int base = 0; base < N * s.channels; base += each) {
        const int c = base + threadIdx.x / g.share;
        float t = 0.0f;
        if (c < N * s.channels)
#pragma unroll 4
            for (int r = mine; r < g.sum_rows; r += g.share) t += s.rows[r * s.pitch + c];
        for (int o = 1; o < g.share; o *= 2) t += __shfl_xor_sync(0xffffffffu, t, o);
        if (mine == 0 && c < N * s.channels) s.channel[c] = t;
    }
    __syncthreads();
}

/* f(group, sum over its channels of value(channel)) for each of the tile's groups, by one thread each. */
template <class Value, class F>
__device__ __forceinline__ void group_totals(const NormShape &d, const Seat &at, Value &&value, F &&f) {
    if (d.per_group <= 32) {
        for (int i = threadIdx.x; i < at.groups; i += blockDim.x) {
            float t = 0.0f;
            for (int c = i * d.per_group; c < (i + 1) * d.per_group; ++c) t += value(c);
            f(i, t);
        }
    } else {
        for (int i = threadIdx.x / 32; i < at.groups; i += blockDim.x / 32) {
            float t = 0.0f;
            for (int c = threadIdx.x % 32; c < d.per_group; c += 32) t += value(i * d.per_group + c);
            t = warp_sum(t);
            if (threadIdx.x % 32 == 0) f(i, t);
        }
    }
}

/* ---- forward ---- */

/* Leaves the tile's own mean and squares about it of each group in
 * s.group[2 * group], [2 * group + 1]; visible to all. */
template <class T, int PACK>
__device__ __forceinline__ void tile_statistics(const Held<T, PACK> *tile, const Sums &s, const Seat &at,
                                                const NormShape &d, const Tiling &g) {
    using V = typename Values<PACK>::V;
    constexpr int N = Values<PACK>::kCount;
    Array<PACK> own[1], e;
#pragma unroll
    for (int k = 0; k < N; ++k) own[0][k] = vall<V>(0.0f);
#pragma unroll 4
    for (int i = 0; i < at.mine; ++i) {
        taken<T, PACK>(tile[i * kThreads], e);
#pragma unroll
        for (int k = 0; k < N; ++k) own[0][k] = vadd(own[0][k], e[k]);
    }
    channel_totals<PACK, 1>(own, s, at, g);
    const float count = static_cast<float>(at.rows) * static_cast<float>(d.per_group);
    group_totals(d, at, [&](int c) { return s.channel[c]; }, [&](int i, float t) { s.group[2 * i] = t / count; });
    __syncthreads();
    const Channels<PACK> less = by_group<PACK>(at, d, g, [&](int i) { return -s.group[2 * i]; });
#pragma unroll
    for (int k = 0; k < N; ++k) own[0][k] = vall<V>(0.0f);
#pragma unroll 4
    for (int i = 0; i < at.mine; ++i) {
        taken<T, PACK>(tile[i * kThreads], e);
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const V off = vadd(e[k], less.v[k]);
            own[0][k] = vfma(off, off, own[0][k]);
        }
    }
    channel_totals<PACK, 1>(own, s, at, g);
    group_totals(d, at, [&](int c) { return s.channel[c]; }, [&](int i, float t) { s.group[2 * i + 1] = t; });
    __syncthreads();
}

/* A thread's channels: u = (x - mean) scale + shift. */
template <int PACK> struct Affine {
    Channels<PACK> less, scale, shift; /* less = -mean */
};
template <int PACK>
__device__ __forceinline__ void result(Array<PACK> &e, const Affine<PACK> &f, int act) {
#pragma unroll
    for (int k = 0; k < Values<PACK>::kCount; ++k) e[k] = vfma(vadd(e[k], f.less.v[k]), f.scale.v[k], f.shift.v[k]);
    activate(e, act);
}

/* The tile's statistics and, where the whole sample's groups are in the
 * cluster, its result; else the statistics go to partial [samples, blocks,
 * parts, 2 block_groups]. */
template <class T, int PACK, bool WHOLE>
__global__ void __launch_bounds__(kThreads, 6)
norm_forward_tiles(NormShape d, Tiling g, const T *x, const float *gamma, const float *beta, T *y, float *mean_out,
                   float *rstd_out, float *partial) {
    extern __shared__ __align__(16) float shared[];
    const Seat at = seat_of(d, g, blockIdx.x);
    const Sums s = sums_of<1>(shared, g);
    Held<T, PACK> *const tile = reinterpret_cast<Held<T, PACK> *>(s.tile) + threadIdx.x;
    load_tile<kThreads, T, PACK>(tile, x + at.n * d.xs, d.xp, at, g);
    tile_loaded();
    tile_statistics<T, PACK>(tile, s, at, d, g);
    if constexpr (!WHOLE) {
        for (int i = threadIdx.x; i < 2 * g.block_groups; i += blockDim.x)
            partial[static_cast<size_t>(blockIdx.x) * 2 * g.block_groups + i] = s.group[i];
    } else {
        float *merged = s.group + 2 * g.block_groups;
        cg::cluster_group cluster = cg::this_cluster();
        if (g.parts > 1) cluster.sync();
        for (int i = threadIdx.x; i < at.groups; i += blockDim.x) {
            float mean = s.group[2 * i], squares = s.group[2 * i + 1];
            const float total = static_cast<float>(d.positions) * static_cast<float>(d.per_group);
            if (g.parts > 1) { /* in the parts' order */
                const auto rows = [&](int r) {
                    return static_cast<float>(r + 1 < g.parts ? g.rows : static_cast<int>(d.positions) - r * g.rows);
                };
                float sum = 0.0f;
                for (int r = 0; r < g.parts; ++r) sum += rows(r) * cluster.map_shared_rank(s.group, r)[2 * i];
                mean = sum / static_cast<float>(d.positions);
                squares = 0.0f;
                for (int r = 0; r < g.parts; ++r) {
                    const float *other = cluster.map_shared_rank(s.group, r) + 2 * i;
                    const float off = other[0] - mean;
                    squares += fmaf(rows(r) * static_cast<float>(d.per_group) * off, off, other[1]);
                }
            }
            const float rstd = 1.0f / sqrtf(squares / total + d.epsilon);
            merged[2 * i] = mean;
            merged[2 * i + 1] = rstd;
            if (mean_out && at.part == 0) {
                const size_t to = static_cast<size_t>(at.n) * d.groups + at.block * g.block_groups + i;
                mean_out[to] = mean;
                rstd_out[to] = rstd;
            }
        }
        if (g.parts > 1) cluster.barrier_arrive(); /* no CTA leaves before the others have read */
        __syncthreads();
        Affine<PACK> f;
        f.less = by_group<PACK>(at, d, g, [&](int i) { return -merged[2 * i]; });
        f.scale = times<PACK>(by_group<PACK>(at, d, g, [&](int i) { return merged[2 * i + 1]; }),
                              parameters_of<PACK>(at, gamma, 1.0f));
        f.shift = parameters_of<PACK>(at, beta, 0.0f);
        T *p = y + at.n * d.ys + (at.first + at.row) * d.yp + at.c0 + at.lane * PACK;
        const size_t jump = g.rows_at_once * d.yp;
#pragma unroll 4
        for (int i = 0; i < at.mine; ++i) {
            Array<PACK> e;
            taken<T, PACK>(tile[i * kThreads], e);
            result<PACK>(e, f, d.act);
            put<T, PACK>(p, e);
            p += jump;
        }
        if (g.parts > 1) cluster.barrier_wait();
    }
}

/* One warp per (sample, group): merges the tiles' statistics. */
__global__ void __launch_bounds__(kThreads)
norm_merge(NormShape d, Tiling g, const float *partial, float *mean_out, float *rstd_out) {
    const size_t at = static_cast<size_t>(blockIdx.x) * (kThreads / 32) + threadIdx.x / 32;
    if (at >= d.samples * d.groups) return;
    const int lane = threadIdx.x % 32, group = static_cast<int>(at % d.groups);
    const size_t n = at / d.groups, block = group / g.block_groups;
    const float *p = partial + (n * g.blocks + block) * g.parts * 2 * g.block_groups + 2 * (group % g.block_groups);
    const size_t pitch = 2 * g.block_groups;
    const auto rows = [&](int r) {
        return static_cast<float>(r + 1 < g.parts ? g.rows : static_cast<int>(d.positions) - r * g.rows);
    };
    float sum = 0.0f;
#pragma unroll 8
    for (int r = lane; r < g.parts; r += 32) sum += rows(r) * p[r * pitch];
    const float mean = warp_sum(sum) / static_cast<float>(d.positions);
    float squares = 0.0f;
#pragma unroll 8
    for (int r = lane; r < g.parts; r += 32) {
        const float off = p[r * pitch] - mean;
        squares += fmaf(rows(r) * static_cast<float>(d.per_group) * off, off, p[r * pitch + 1]);
    }
    squares = warp_sum(squares);
    if (lane == 0) {
        mean_out[at] = mean;
        rstd_out[at] = 1.0f / sqrtf(squares / (static_cast<float>(d.positions) * static_cast<float>(d.per_group)) + d.epsilon);
    }
}

/* Packs that a thread of the second read has under way. */
constexpr int kAhead = 4;

/* The result from given statistics. */
template <class T, int PACK>
__global__ void __launch_bounds__(kThreads, 6)
norm_forward_apply(NormShape d, Tiling g, const T *x, const float *gamma, const float *beta, const float *mean,
                   const float *rstd, T *y) {
    const Seat at = seat_of(d, g, gridDim.x - 1 - blockIdx.x);
    const T *from = x + at.n * d.xs + (at.first + at.row) * d.xp + at.c0 + at.lane * PACK;
    T *to = y + at.n * d.ys + (at.first + at.row) * d.yp + at.c0 + at.lane * PACK;
    const size_t from_jump = g.rows_at_once * d.xp, to_jump = g.rows_at_once * d.yp;
    const size_t first = static_cast<size_t>(at.n) * d.groups + at.block * g.block_groups;
    Affine<PACK> f;
    f.less = by_group<PACK>(at, d, g, [&](int i) { return -mean[first + i]; });
    f.scale = times<PACK>(by_group<PACK>(at, d, g, [&](int i) { return rstd[first + i]; }),
                          parameters_of<PACK>(at, gamma, 1.0f));
    f.shift = parameters_of<PACK>(at, beta, 0.0f);
    Held<T, PACK> next[kAhead];
    const auto load = [&](int i) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (i + j < at.mine) next[j] = *reinterpret_cast<const Held<T, PACK> *>(from + j * from_jump);
        from += kAhead * from_jump;
    };
    load(0);
    for (int i = 0; i < at.mine; i += kAhead) {
        Held<T, PACK> v[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) v[j] = next[j];
        load(i + kAhead);
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (i + j < at.mine) {
                Array<PACK> e;
                taken<T, PACK>(v[j], e);
                result<PACK>(e, f, d.act);
                put<T, PACK>(to + j * to_jump, e);
            }
        to += kAhead * to_jump;
    }
}

/* ---- backward ---- */

/* z = x - mean, u = z scale + beta with scale = rstd gamma. */
template <int PACK> struct Given {
    Channels<PACK> less, scale, beta; /* less = -mean */
};
template <int PACK>
__device__ __forceinline__ Given<PACK> given_of(const NormShape &d, const Tiling &g, const Seat &at, const float *gamma,
                                                const float *beta, const float *mean, const float *rstd) {
    const size_t first = static_cast<size_t>(at.n) * d.groups + at.block * g.block_groups;
    Given<PACK> f;
    f.less = by_group<PACK>(at, d, g, [&](int i) { return -mean[first + i]; });
    f.scale = times<PACK>(by_group<PACK>(at, d, g, [&](int i) { return rstd[first + i]; }),
                          parameters_of<PACK>(at, gamma, 1.0f));
    f.beta = parameters_of<PACK>(at, beta, 0.0f);
    return f;
}
/* x becomes z, dy becomes du = dy act'(u). */
template <int PACK>
__device__ __forceinline__ void gradients(Array<PACK> &x, Array<PACK> &dy, const Given<PACK> &f, int act) {
    Array<PACK> u;
#pragma unroll
    for (int k = 0; k < Values<PACK>::kCount; ++k) {
        x[k] = vadd(x[k], f.less.v[k]);
        u[k] = vfma(x[k], f.scale.v[k], f.beta.v[k]);
    }
    slopes(u, act);
#pragma unroll
    for (int k = 0; k < Values<PACK>::kCount; ++k) dy[k] = vmul(dy[k], u[k]);
}
/* With hat = z rstd and m1, m2 the group's means of du gamma and du gamma hat:
 * dx = rstd (du gamma - m1 - hat m2) = du scale + n1 + z n2.  The tiles sum du
 * scale and du scale z, so with their means M1 = rstd m1 and M2 = m2. */
template <int PACK> struct Less {
    Channels<PACK> n1, n2; /* -M1, -rstd^2 M2 */
};
template <int PACK>
__device__ __forceinline__ Less<PACK> less_of(const NormShape &d, const Tiling &g, const Seat &at, const float *rstd,
                                              const float *means) {
    const size_t first = static_cast<size_t>(at.n) * d.groups + at.block * g.block_groups;
    Less<PACK> f;
    f.n1 = by_group<PACK>(at, d, g, [&](int i) { return -means[2 * i]; });
    f.n2 = by_group<PACK>(at, d, g, [&](int i) { return -rstd[first + i] * rstd[first + i] * means[2 * i + 1]; });
    return f;
}
template <int PACK>
__device__ __forceinline__ void input_gradient(Array<PACK> &z, const Array<PACK> &du, const Given<PACK> &f,
                                               const Less<PACK> &l) {
#pragma unroll
    for (int k = 0; k < Values<PACK>::kCount; ++k)
        z[k] = vfma(du[k], f.scale.v[k], vfma(z[k], l.n2.v[k], l.n1.v[k]));
}

/* The tile's sums and, where the whole sample's groups are in the cluster, dx:
 * du, found once, waits for the sums in shared memory in f32 (twice the bytes
 * of a 16-bit dy, but the activation's slope costs more than that again).
 * Per-channel sums go to partial [samples, parts, 2, channels], and where the
 * sample is larger the groups' to sums [samples, parts, 2, groups]. */
template <class T, int PACK, bool WHOLE>
__global__ void __launch_bounds__(kBackwardThreads, 2)
norm_backward_tiles(NormShape d, Tiling g, const T *x, const float *gamma, const float *beta, const float *mean,
                    const float *rstd, const T *dy, T *dx, float *partial, float *sums) {
    using V = typename Values<PACK>::V;
    constexpr int N = Values<PACK>::kCount;
    extern __shared__ __align__(16) float shared[];
    const Seat at = seat_of(d, g, blockIdx.x);
    const Sums s = sums_of<2>(shared, g);
    constexpr int STEP = kBackwardThreads;
    Held<T, PACK> *const tile = reinterpret_cast<Held<T, PACK> *>(s.tile) + threadIdx.x;
    V *const kept = reinterpret_cast<V *>(s.tile + static_cast<size_t>(g.turns) * STEP * sizeof(Held<T, PACK>)) +
                    threadIdx.x; /* [turns][N][STEP] */
    load_tile<STEP, T, PACK>(tile, x + at.n * d.xs, d.xp, at, g);
    const T *from = dy + at.n * d.ys + (at.first + at.row) * d.yp + at.c0 + at.lane * PACK;
    const size_t from_jump = g.rows_at_once * d.yp;
    Held<T, PACK> next[kAhead];
    const auto load = [&](int i) {
        if (i + kAhead <= at.mine) {
#pragma unroll
            for (int j = 0; j < kAhead; ++j) next[j] = *reinterpret_cast<const Held<T, PACK> *>(from + j * from_jump);
        } else {
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
                if (i + j < at.mine) next[j] = *reinterpret_cast<const Held<T, PACK> *>(from + j * from_jump);
        }
        from += kAhead * from_jump;
    };
    load(0);
    const Given<PACK> f = given_of<PACK>(d, g, at, gamma, beta, mean, rstd);
    if (at.in && at.row == 0) /* for the groups' sums */
#pragma unroll
        for (int k = 0; k < N; ++k) vstore(s.scale + at.lane * PACK + 2 * k, f.scale.v[k]);
    tile_loaded();
    {
        Array<PACK> own[2]; /* sums of du and of du z */
#pragma unroll
        for (int k = 0; k < N; ++k) own[0][k] = own[1][k] = vall<V>(0.0f);
        const auto take = [&](const Held<T, PACK> &w, int i) {
            Array<PACK> z, du;
            taken<T, PACK>(tile[i * STEP], z);
            taken<T, PACK>(w, du);
            gradients<PACK>(z, du, f, d.act);
#pragma unroll
            for (int k = 0; k < N; ++k) {
                own[0][k] = vadd(own[0][k], du[k]);
                own[1][k] = vfma(du[k], z[k], own[1][k]);
                if (WHOLE) kept[(i * N + k) * STEP] = du[k];
            }
        };
        for (int i = 0; i < at.mine; i += kAhead) {
            Held<T, PACK> w[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) w[j] = next[j];
            load(i + kAhead);
            if (i + kAhead <= at.mine) {
#pragma unroll
                for (int j = 0; j < kAhead; ++j) take(w[j], i + j);
            } else {
#pragma unroll
                for (int j = 0; j < kAhead - 1; ++j)
                    if (i + j < at.mine) take(w[j], i + j);
            }
        }
        channel_totals<PACK, 2>(own, s, at, g);
        /* scale = rstd gamma: these are rstd times the sums of du gamma and du gamma z */
        const float *second = s.channel + s.channels;
        group_totals(d, at, [&](int c) { return s.channel[c] * s.scale[c]; }, [&](int i, float t) { s.group[2 * i] = t; });
        group_totals(d, at, [&](int c) { return second[c] * s.scale[c]; }, [&](int i, float t) { s.group[2 * i + 1] = t; });
        __syncthreads();
    }
    const float *const rstd_of = rstd + static_cast<size_t>(at.n) * d.groups + at.block * g.block_groups;
    if (partial) {
        float *to = partial + (static_cast<size_t>(at.n) * g.parts + at.part) * 2 * d.channels + at.c0;
        for (int c = threadIdx.x; c < at.channels; c += blockDim.x) {
            to[c] = s.channel[c];
            to[d.channels + c] = s.channel[s.channels + c] * rstd_of[group_of(c, d, g)]; /* of du hat */
        }
    }
    if constexpr (!WHOLE) {
        float *to = sums + (static_cast<size_t>(at.n) * g.parts + at.part) * 2 * d.groups + at.block * g.block_groups;
        for (int i = threadIdx.x; i < at.groups; i += blockDim.x) {
            to[i] = s.group[2 * i];
            to[d.groups + i] = s.group[2 * i + 1];
        }
    } else {
        float *merged = s.group + 2 * g.block_groups;
        cg::cluster_group cluster = cg::this_cluster();
        if (g.parts > 1) cluster.sync();
        const float count = static_cast<float>(d.positions) * static_cast<float>(d.per_group);
        for (int i = threadIdx.x; i < 2 * at.groups; i += blockDim.x) {
            float t = 0.0f;
            for (int r = 0; r < g.parts; ++r) t += g.parts > 1 ? cluster.map_shared_rank(s.group, r)[i] : s.group[i];
            merged[i] = t / count;
        }
        if (g.parts > 1) cluster.barrier_arrive(); /* no CTA leaves before the others have read */
        __syncthreads();
        const Less<PACK> l = less_of<PACK>(d, g, at, rstd, merged);
        T *p = dx + at.n * d.gs + (at.first + at.row) * d.gp + at.c0 + at.lane * PACK;
        const size_t jump = g.rows_at_once * d.gp;
#pragma unroll 4
        for (int i = 0; i < at.mine; ++i) {
            Array<PACK> z, du;
            taken<T, PACK>(tile[i * STEP], z);
#pragma unroll
            for (int k = 0; k < N; ++k) {
                z[k] = vadd(z[k], f.less.v[k]);
                du[k] = kept[(i * N + k) * STEP];
            }
            input_gradient<PACK>(z, du, f, l);
            put<T, PACK>(p, z);
            p += jump;
        }
        if (g.parts > 1) cluster.barrier_wait();
    }
}

/* One warp per (sample, group): means over the sample of the tiles' sums. */
__global__ void __launch_bounds__(kThreads)
norm_merge_sums(NormShape d, size_t parts, const float *sums, float *means) {
    const size_t at = static_cast<size_t>(blockIdx.x) * (kThreads / 32) + threadIdx.x / 32;
    if (at >= d.samples * d.groups) return;
    const int lane = threadIdx.x % 32;
    const size_t n = at / d.groups, i = at % d.groups;
    float a = 0.0f, b = 0.0f;
#pragma unroll 8
    for (size_t r = lane; r < parts; r += 32) {
        const float *p = sums + (n * parts + r) * 2 * d.groups + i;
        a += p[0];
        b += p[d.groups];
    }
    a = warp_sum(a);
    b = warp_sum(b);
    const float count = static_cast<float>(d.positions) * static_cast<float>(d.per_group);
    if (lane == 0) {
        means[2 * at] = a / count;
        means[2 * at + 1] = b / count;
    }
}

template <class T, int PACK>
__global__ void __launch_bounds__(kBackwardThreads, 2)
norm_backward_apply(NormShape d, Tiling g, const T *x, const float *gamma, const float *beta, const float *mean,
                    const float *rstd, const float *means, const T *dy, T *dx) {
    const Seat at = seat_of(d, g, gridDim.x - 1 - blockIdx.x);
    const T *from = x + at.n * d.xs + (at.first + at.row) * d.xp + at.c0 + at.lane * PACK;
    const T *from_dy = dy + at.n * d.ys + (at.first + at.row) * d.yp + at.c0 + at.lane * PACK;
    T *to = dx + at.n * d.gs + (at.first + at.row) * d.gp + at.c0 + at.lane * PACK;
    const size_t jump = g.rows_at_once * d.xp, dy_jump = g.rows_at_once * d.yp, to_jump = g.rows_at_once * d.gp;
    const Given<PACK> f = given_of<PACK>(d, g, at, gamma, beta, mean, rstd);
    const size_t first = static_cast<size_t>(at.n) * d.groups + at.block * g.block_groups;
    const Less<PACK> l = less_of<PACK>(d, g, at, rstd, means + 2 * first);
    constexpr int kPairs = kAhead / 2;
    for (int i = 0; i < at.mine; i += kPairs) {
        Held<T, PACK> v[kPairs], w[kPairs];
#pragma unroll
        for (int j = 0; j < kPairs; ++j)
            if (i + j < at.mine) {
                v[j] = *reinterpret_cast<const Held<T, PACK> *>(from + j * jump);
                w[j] = *reinterpret_cast<const Held<T, PACK> *>(from_dy + j * dy_jump);
            }
#pragma unroll
        for (int j = 0; j < kPairs; ++j)
            if (i + j < at.mine) {
                Array<PACK> z, du;
                taken<T, PACK>(v[j], z);
                taken<T, PACK>(w[j], du);
                gradients<PACK>(z, du, f, d.act);
                input_gradient<PACK>(z, du, f, l);
                put<T, PACK>(to + j * to_jump, z);
            }
        from += kPairs * jump;
        from_dy += kPairs * dy_jump;
        to += kPairs * to_jump;
    }
}

/* dbeta and dgamma from the sums of rows [2, channels]. */
struct Parameters {
    int channels;
    float *dgamma, *dbeta;
    __device__ void operator()(size_t c, float sum) const {
        if (c < static_cast<size_t>(channels)) {
            if (dbeta) dbeta[c] = sum;
        } else if (dgamma) {
            dgamma[c - channels] = sum;
        }
    }
};

/* ---- groups wider than a CTA's rows: one CTA per (sample, group) ---- */

/* A long sum in f32: of 16 terms, of 16 such sums, and so on, so that a term of
 * a million is rounded some 80 times on its way and not a million times. */
struct LongSum {
    static constexpr int kLevels = 6;
    float s[kLevels] = {};
    unsigned terms = 0;
    __device__ __forceinline__ void add(float v) {
        s[0] += v;
        ++terms;
#pragma unroll
        for (int i = 1; i < kLevels; ++i) {
            if (terms >> 4 * (i - 1) & 15u) return;
            s[i] += s[i - 1];
            s[i - 1] = 0.0f;
        }
    }
    __device__ __forceinline__ float total() const {
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < kLevels; ++i) t += s[i];
        return t;
    }
};

/* Where there are this many positions or more (LONG), a thread takes eight of a
 * channel together; where there are fewer, one value after the other: 64 x 256 x
 * 272 f32, one group, 88 us in both directions, one by one 426 and 312; forward
 * of 1,000 x 7 x 2,304 bf16, two groups, 49 us and 39, backward of f32 115 and
 * 167. */
constexpr int kForwardLong = 8, kBackwardLong = 4;
/* Channels that are added up before their sum joins the others: 16 of a thread. */
constexpr int kStretch = 16 * kThreads;
/* f(first, how many: a constant) for runs of positions: eights, then what is left. */
template <class F> __device__ __forceinline__ void runs_of(size_t positions, F &&f) {
    size_t p = 0;
    for (; p + 8 <= positions; p += 8) f(p, std::integral_constant<int, 8>{});
    if (positions & 4) f(p, std::integral_constant<int, 4>{}), p += 4;
    if (positions & 2) f(p, std::integral_constant<int, 2>{}), p += 2;
    if (positions & 1) f(p, std::integral_constant<int, 1>{});
}

/* Sum over the CTA; every thread receives it. */
__device__ float block_sum(float v, float *scratch) {
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.0f;
    for (int i = 0; i < kThreads / 32; ++i) t += scratch[i];
    __syncthreads();
    return t;
}

template <class T, bool LONG>
__global__ void __launch_bounds__(kThreads)
norm_forward_wide(NormShape d, const T *x, const float *gamma, const float *beta, T *y, float *mean_out, float *rstd_out) {
    __shared__ float scratch[kThreads / 32];
    const size_t n = blockIdx.x / d.groups;
    const int g = static_cast<int>(blockIdx.x % d.groups);
    const int c0 = g * d.per_group;
    const float count = static_cast<float>(d.positions) * static_cast<float>(d.per_group);
    const T *xs = x + n * d.xs + c0;
    const auto sum_of = [&](auto &&f) { /* f(value, sum): the sum with the value's term */
        std::conditional_t<LONG, LongSum, float> s{};
        if constexpr (LONG) {
            for (int c = threadIdx.x; c < d.per_group; c += kThreads)
                runs_of(d.positions, [&](size_t p, auto many) {
                    constexpr int MANY = decltype(many)::value;
                    float v[MANY], t = 0.0f;
#pragma unroll
                    for (int j = 0; j < MANY; ++j) v[j] = to_float(xs[(p + j) * d.xp + c]);
#pragma unroll
                    for (int j = 0; j < MANY; ++j) t = f(v[j], t);
                    s.add(t);
                });
        } else {
            for (size_t p = 0; p < d.positions; ++p)
                for (int first = 0; first < d.per_group; first += kStretch) {
                    const int end = min(d.per_group - first, kStretch) + first;
                    float t = 0.0f;
                    for (int c = first + threadIdx.x; c < end; c += kThreads) t = f(to_float(xs[p * d.xp + c]), t);
                    s += t;
                }
        }
        if constexpr (LONG) return block_sum(s.total(), scratch);
        else return block_sum(s, scratch);
    };
    const float mean = sum_of([](float v, float t) { return t + v; }) / count;
    const float squares = sum_of([&](float v, float t) { return fmaf(v - mean, v - mean, t); });
    const float rstd = 1.0f / sqrtf(squares / count + d.epsilon);
    if (threadIdx.x == 0 && mean_out) {
        mean_out[blockIdx.x] = mean;
        rstd_out[blockIdx.x] = rstd;
    }
    T *const ys = y + n * d.ys + c0;
    const auto result_of = [&](size_t p, int c, auto many) {
        constexpr int MANY = decltype(many)::value;
        const float scale = rstd * (gamma ? gamma[c0 + c] : 1.0f), shift = beta ? beta[c0 + c] : 0.0f;
        float v[MANY];
#pragma unroll
        for (int j = 0; j < MANY; ++j) v[j] = to_float(xs[(p + j) * d.xp + c]);
#pragma unroll
        for (int j = 0; j < MANY; ++j) v[j] = fmaf(v[j] - mean, scale, shift);
        activate(v, d.act);
#pragma unroll
        for (int j = 0; j < MANY; ++j) ys[(p + j) * d.yp + c] = from_float<T>(v[j]);
    };
    if constexpr (LONG) {
        for (int c = threadIdx.x; c < d.per_group; c += kThreads)
            runs_of(d.positions, [&](size_t p, auto many) { result_of(p, c, many); });
    } else {
        for (size_t p = 0; p < d.positions; ++p)
            for (int c = threadIdx.x; c < d.per_group; c += kThreads) result_of(p, c, std::integral_constant<int, 1>{});
    }
}

/* partial [samples, 2, channels]. */
template <class T, bool LONG>
__global__ void __launch_bounds__(kThreads)
norm_backward_wide(NormShape d, const T *x, const float *gamma, const float *beta, const float *mean_in,
                   const float *rstd_in, const T *dy, T *dx, float *partial) {
    __shared__ float scratch[kThreads / 32];
    const size_t n = blockIdx.x / d.groups;
    const int g = static_cast<int>(blockIdx.x % d.groups);
    const int c0 = g * d.per_group;
    const float mean = mean_in[blockIdx.x], rstd = rstd_in[blockIdx.x];
    const auto gradients_at = [&](size_t p, auto many, int c, float ga, float be, float *hat, float *du) {
        constexpr int MANY = decltype(many)::value;
        float u[MANY];
#pragma unroll
        for (int j = 0; j < MANY; ++j) {
            hat[j] = (to_float(x[n * d.xs + (p + j) * d.xp + c]) - mean) * rstd;
            du[j] = to_float(dy[n * d.ys + (p + j) * d.yp + c]);
            u[j] = fmaf(hat[j], ga, be);
        }
        slopes(u, d.act);
#pragma unroll
        for (int j = 0; j < MANY; ++j) du[j] *= u[j];
    };
    const auto runs = [&](auto &&f) { /* of the channel's positions */
        if constexpr (LONG) {
            runs_of(d.positions, f);
        } else {
            for (size_t p = 0; p < d.positions; ++p) f(p, std::integral_constant<int, 1>{});
        }
    };
    float s1 = 0.0f, s2 = 0.0f;
    for (int first = c0; first < c0 + d.per_group; first += kStretch) {
        const int end = min(c0 + d.per_group - first, kStretch) + first;
        float t1 = 0.0f, t2 = 0.0f;
        for (int c = first + threadIdx.x; c < end; c += kThreads) {
            const float ga = gamma ? gamma[c] : 1.0f, be = beta ? beta[c] : 0.0f;
            std::conditional_t<LONG, LongSum, float> a{}, b{};
            runs([&](size_t p, auto many) {
                constexpr int MANY = decltype(many)::value;
                float hat[MANY], du[MANY];
                gradients_at(p, many, c, ga, be, hat, du);
                if constexpr (LONG) {
                    float ta = 0.0f, tb = 0.0f;
#pragma unroll
                    for (int j = 0; j < MANY; ++j) ta += du[j], tb = fmaf(du[j], hat[j], tb);
                    a.add(ta);
                    b.add(tb);
                } else {
                    a += du[0];
                    b = fmaf(du[0], hat[0], b);
                }
            });
            float of_du, of_du_hat;
            if constexpr (LONG) of_du = a.total(), of_du_hat = b.total();
            else of_du = a, of_du_hat = b;
            partial[n * 2 * d.channels + c] = of_du;
            partial[n * 2 * d.channels + d.channels + c] = of_du_hat;
            t1 = fmaf(ga, of_du, t1);
            t2 = fmaf(ga, of_du_hat, t2);
        }
        s1 += t1;
        s2 += t2;
    }
    const float count = static_cast<float>(d.positions) * static_cast<float>(d.per_group);
    s1 = block_sum(s1, scratch) / count;
    s2 = block_sum(s2, scratch) / count;
    for (int c = c0 + threadIdx.x; c < c0 + d.per_group; c += kThreads) {
        const float ga = gamma ? gamma[c] : 1.0f, be = beta ? beta[c] : 0.0f;
        runs([&](size_t p, auto many) {
            constexpr int MANY = decltype(many)::value;
            float hat[MANY], du[MANY];
            gradients_at(p, many, c, ga, be, hat, du);
#pragma unroll
            for (int j = 0; j < MANY; ++j)
                dx[n * d.gs + (p + j) * d.gp + c] = from_float<T>(rstd * (fmaf(du[j], ga, -s1) - hat[j] * s2));
        });
    }
}

/* ---- host side ---- */

bool norm_shape(const tb_group_norm_desc *d, NormShape *s) {
    if (!d || !d->samples || !d->positions || !d->channels || !d->groups || d->channels > 0x7fffffffu ||
        d->channels % d->groups || !type_known(d->type) || d->activation < TB_ACT_NONE ||
        d->activation > TB_ACT_GELU || !(d->epsilon >= 0.0f))
        return false;
    size_t blocks, all;
    if (!product(d->samples, d->groups, 0x7fffffffu, &blocks) ||
        !product(d->positions, d->channels, SIZE_MAX / 64 / d->samples, &all))
        return false;
    s->samples = d->samples;
    s->positions = d->positions;
    s->channels = static_cast<int>(d->channels);
    s->groups = static_cast<int>(d->groups);
    s->per_group = static_cast<int>(d->channels / d->groups);
    s->xp = d->x_position_stride ? d->x_position_stride : d->channels;
    s->yp = d->y_position_stride ? d->y_position_stride : d->channels;
    s->xs = d->x_sample_stride ? d->x_sample_stride : d->positions * s->xp;
    s->ys = d->y_sample_stride ? d->y_sample_stride : d->positions * s->yp;
    s->gp = d->dx_position_stride ? d->dx_position_stride : d->channels;
    s->gs = d->dx_sample_stride ? d->dx_sample_stride : d->positions * s->gp;
    if (s->xp < d->channels || s->yp < d->channels || s->gp < d->channels) return false;
    s->act = d->activation;
    s->epsilon = d->epsilon;
    return true;
}

/* Bytes of a tile of x at most: six such CTAs (backward, with du: two of 16-bit
 * types, three of f32) share an SM.  64 channels of bf16, of 4,096 maps of 256
 * positions (the same tensors over and over: with others from call to call
 * the backward pass takes 143): 61 us forward, 138 backward; tiles of 16 KB 88 and 232.  1,024 maps
 * of 1,024 positions: 70 and 161 us; tiles of 56 KB 79 and 241; three kernels in
 * the place of clusters 82 and 208.  Where eight such tiles do not hold a map,
 * larger ones in a cluster lose against a second read of x: 512 maps of 4,096
 * positions forward 199 us against 146, of 3,000 backward 392 against 289. */
constexpr size_t kTile = 32768;

/* Tiles for packs of `pack` elements; false where a group is wider than a
 * CTA's rows (or the tiles are too many to count). */
bool tiling_of(const NormShape &d, int pack, size_t size, bool backward, Tiling *g) {
    const int most_threads = backward ? kBackwardThreads : kThreads;
    /* whole groups, whole packs, 128 bytes a row if there are: narrower rows
     * waste sectors, wider ones leave fewer and longer tiles */
    bool found = false;
    for (int i = 1; i <= d.groups && !found; ++i) {
        if (static_cast<size_t>(i) * d.per_group % pack) continue;
        const size_t lanes = static_cast<size_t>(i) * d.per_group / pack;
        if (lanes > static_cast<size_t>(most_threads)) break;
        g->block_groups = i;
        g->lanes = static_cast<int>(lanes);
        found = lanes * pack * size >= 128 || i == d.groups;
    }
    if (!found || d.positions > 0x3fffffffu) return false;
    g->pack = pack;
    g->blocks = (d.groups + g->block_groups - 1) / g->block_groups;
    const size_t packs = d.positions * g->lanes;
    const size_t threads = packs < static_cast<size_t>(most_threads) ? align_up(packs, 32) : most_threads;
    g->threads = static_cast<int>(threads);
    g->rows_at_once = g->threads / g->lanes;
    const size_t turns = kTile / (static_cast<size_t>(most_threads) * pack * size);
    const size_t most = static_cast<size_t>(g->rows_at_once) * (turns ? turns : 1);
    const size_t parts = (d.positions + most - 1) / most;
    const size_t rows = align_up((d.positions + parts - 1) / parts, g->rows_at_once);
    if (product(d.samples * g->blocks, parts, 0x7fffffffu, &g->tiles) == false) return false;
    g->rows = static_cast<int>(rows);
    g->turns = static_cast<int>(rows / g->rows_at_once);
    g->parts = static_cast<int>((d.positions + rows - 1) / rows);
    g->fits = g->parts <= kCluster;
    g->tiles = d.samples * g->blocks * g->parts;
    g->folds = 32 % g->lanes == 0;
    g->sum_rows = g->folds ? g->threads / 32 : g->rows_at_once;
    g->share = 1;
    while (g->share < 32 && g->share * 2 * g->lanes * pack <= g->threads) g->share *= 2;
    const auto magic = [](unsigned by) { return static_cast<unsigned>(0xffffffffull / by); };
    g->magic_parts = magic(g->parts);
    g->magic_blocks = magic(g->blocks);
    g->magic_lanes = magic(g->lanes);
    g->magic_rows = magic(g->rows_at_once);
    g->magic_group = magic(d.per_group);
    return true;
}

/* The widest pack that every row allows. */
int pack_of(const NormShape &d, size_t size, const void *a, size_t as, size_t ap, const void *b, size_t bs, size_t bp) {
    return tb_learn::pack_of(reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | (as | ap | bs | bp) * size |
                                 static_cast<size_t>(d.channels) * size, size);
}

template <auto Kernel, class... Args>
int launch_tiles(const NormShape &d, const Tiling &g, bool clusters, size_t shared, cudaStream_t st, Args... args) {
    if (!allow_shared<Kernel>(shared)) return 0;
    if (!clusters || g.parts == 1) {
        Kernel<<<static_cast<unsigned>(g.tiles), g.threads, shared, st>>>(d, g, args...);
        return launched();
    }
    cudaLaunchConfig_t c{};
    c.gridDim = dim3(static_cast<unsigned>(g.tiles));
    c.blockDim = dim3(static_cast<unsigned>(g.threads));
    c.dynamicSmemBytes = shared;
    c.stream = st;
    cudaLaunchAttribute a{};
    a.id = cudaLaunchAttributeClusterDimension;
    a.val.clusterDim = {static_cast<unsigned>(g.parts), 1, 1};
    c.attrs = &a;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, Kernel, d, g, args...) == cudaSuccess;
}

/* Workspace: the forward pass's partial statistics, or the backward pass's
 * per-channel rows with their column sums, group sums and means. */
size_t forward_bytes(const NormShape &d, const Tiling &g) {
    return (2 * d.samples * d.groups + g.tiles * 2 * g.block_groups) * sizeof(float);
}
size_t backward_bytes(const NormShape &d, size_t parts) {
    const size_t rows = d.samples * parts;
    return ((rows + column_parts(rows)) * 2 * d.channels + (rows + d.samples) * 2 * d.groups) * sizeof(float);
}

unsigned merge_grid(const NormShape &d) {
    return static_cast<unsigned>((d.samples * d.groups + kThreads / 32 - 1) / (kThreads / 32));
}

} /* namespace */

extern "C" size_t tb_cuda_group_norm_workspace(const tb_group_norm_desc *desc) {
    NormShape s;
    if (!norm_shape(desc, &s)) return 0;
    const size_t size = type_size(desc->type);
    size_t need = backward_bytes(s, 1);
    /* for whichever pack the pointers turn out to allow */
    for (int pack : {static_cast<int>(16 / size), static_cast<int>(4 / size), 1}) {
        Tiling g;
        if (s.channels % pack) continue;
        if (tiling_of(s, pack, size, false, &g) && !g.fits && forward_bytes(s, g) > need) need = forward_bytes(s, g);
        if (tiling_of(s, pack, size, true, &g) && backward_bytes(s, g.parts) > need) need = backward_bytes(s, g.parts);
    }
    return need;
}

extern "C" int tb_cuda_group_norm_device(const tb_group_norm_desc *desc, const void *x, const float *gamma,
                                         const float *beta, void *y, float *mean, float *rstd, void *workspace,
                                         void *stream) {
    NormShape s;
    if (!norm_shape(desc, &s) || !x || !y || !workspace || !mean != !rstd) return 0;
    const size_t size = type_size(desc->type);
    if (!aligned(x, size) || !aligned(y, size) || !aligned(gamma, 4) || !aligned(beta, 4) || !aligned(mean, 4) ||
        !aligned(rstd, 4) || !aligned(workspace, 16) || (x == y && (s.xs != s.ys || s.xp != s.yp)) ||
        collide({y, mean, rstd, workspace}, {gamma, beta}) || collide({mean, rstd, workspace}, {x}))
        return 0;
    cudaGetLastError(); /* report these launches only */
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return with_type(desc->type, [&](auto t) {
        using T = decltype(t);
        const T *in = static_cast<const T *>(x);
        T *out = static_cast<T *>(y);
        Tiling g;
        const int pack = pack_of(s, size, x, s.xs, s.xp, y, s.ys, s.yp);
        if (!tiling_of(s, pack, size, false, &g)) {
            const auto kernel = s.positions >= kForwardLong ? norm_forward_wide<T, true> : norm_forward_wide<T, false>;
            kernel<<<static_cast<unsigned>(s.samples * s.groups), kThreads, 0, st>>>(s, in, gamma, beta, out, mean, rstd);
            return launched();
        }
        return with_pack<T>(pack, [&](auto p) {
            constexpr int P = decltype(p)::value;
            if (g.fits)
                return launch_tiles<norm_forward_tiles<T, P, true>>(s, g, true, shared_bytes(g, size, 1, false), st, in, gamma, beta, out, mean,
                                    rstd, static_cast<float *>(nullptr));
            float *means = static_cast<float *>(workspace), *partial = means + 2 * s.samples * s.groups;
            float *m = mean ? mean : means, *r = rstd ? rstd : means + s.samples * s.groups;
            if (!launch_tiles<norm_forward_tiles<T, P, false>>(s, g, false, shared_bytes(g, size, 1, false), st, in, gamma, beta, out, m, r, partial))
                return 0;
            norm_merge<<<merge_grid(s), kThreads, 0, st>>>(s, g, partial, m, r);
            if (!launched()) return 0;
            return launch_tiles<norm_forward_apply<T, P>>(s, g, false, 0, st, in, gamma, beta, m, r, out);
        });
    });
}

extern "C" int tb_cuda_group_norm_backward_device(const tb_group_norm_desc *desc, const void *x, const float *gamma,
                                                  const float *beta, const float *mean, const float *rstd,
                                                  const void *dy, void *dx, float *dgamma, float *dbeta,
                                                  void *workspace, void *stream) {
    NormShape s;
    if (!norm_shape(desc, &s) || !x || !mean || !rstd || !dy || !dx || !workspace) return 0;
    const size_t size = type_size(desc->type);
    if (!aligned(x, size) || !aligned(dy, size) || !aligned(dx, size) || !aligned(gamma, 4) || !aligned(beta, 4) ||
        !aligned(mean, 4) || !aligned(rstd, 4) || !aligned(dgamma, 4) || !aligned(dbeta, 4) ||
        !aligned(workspace, 16) || (dx == dy && (s.gs != s.ys || s.gp != s.yp)) ||
        (dx == x && (s.gs != s.xs || s.gp != s.xp)) ||
        collide({dx, dgamma, dbeta, workspace}, {gamma, beta, mean, rstd}) || collide({dgamma, dbeta, workspace}, {x, dy}))
        return 0;
    cudaGetLastError(); /* report these launches only */
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int ok_rows = with_type(desc->type, [&](auto t) -> int {
        using T = decltype(t);
        const T *in = static_cast<const T *>(x), *grad = static_cast<const T *>(dy);
        T *out = static_cast<T *>(dx);
        Tiling g;
        float *partial = static_cast<float *>(workspace);
        const int both = pack_of(s, size, x, s.xs, s.xp, dy, s.ys, s.yp), own = pack_of(s, size, dx, s.gs, s.gp, dx, s.gs, s.gp);
        const int pack = both < own ? both : own;
        const bool wide = !tiling_of(s, pack, size, true, &g);
        const size_t rows = s.samples * (wide ? 1 : g.parts), parts = column_parts(rows);
        float *columns = partial + rows * 2 * s.channels, *sums = columns + parts * 2 * s.channels;
        float *rows_to = wide || dgamma || dbeta ? partial : nullptr;
        if (wide) {
            const auto kernel = s.positions >= kBackwardLong ? norm_backward_wide<T, true> : norm_backward_wide<T, false>;
            kernel<<<static_cast<unsigned>(s.samples * s.groups), kThreads, 0, st>>>(s, in, gamma, beta, mean, rstd, grad, out,
                                                                                     partial);
            if (!launched()) return 0;
        } else {
            const int ok = with_pack<T>(pack, [&](auto p) {
                constexpr int P = decltype(p)::value;
                if (g.fits)
                    return launch_tiles<norm_backward_tiles<T, P, true>>(s, g, true, shared_bytes(g, size, 2, true), st, in, gamma, beta, mean,
                                        rstd, grad, out, rows_to, sums);
                float *means = sums + rows * 2 * s.groups;
                if (!launch_tiles<norm_backward_tiles<T, P, false>>(s, g, false, shared_bytes(g, size, 2, false), st, in, gamma, beta, mean, rstd,
                                  grad, out, rows_to, sums))
                    return 0;
                norm_merge_sums<<<merge_grid(s), kThreads, 0, st>>>(s, g.parts, sums, means);
                if (!launched()) return 0;
                return launch_tiles<norm_backward_apply<T, P>>(s, g, false, 0, st, in, gamma, beta, mean, rstd, means, grad,
                                    out);
            });
            if (!ok) return 0;
        }
        if (!dgamma && !dbeta) return 1;
        return sum_columns(partial, rows, 2 * static_cast<size_t>(s.channels), Parameters{s.channels, dgamma, dbeta}, st);
    });
    return ok_rows;
}
