/*
 * Group norm with an activation, channels last: forward and backward
 * (include/turbinator/training/cuda_learner.h).
 *
 * Bound: HBM, given that x (and dy) are read once.  A tile is some positions of
 * some whole groups of one sample; a CTA holds a tile in registers, so that mean,
 * variance about that mean, and result come from one read.  Threads form rows
 * of `lanes` packs, each thread keeping its channels over all its positions.
 *
 *   - A sample's groups that fit one tile, or the tiles of one cluster (8 CTAs),
 *     take one kernel: the tiles' statistics meet in distributed shared memory.
 *   - Larger maps take three: each tile's statistics, their merge, and the
 *     result from a second read, last tiles first, while they are in L2.
 *   - A group of more channels than a CTA has threads times its pack takes a
 *     CTA of its own and reads three times.
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

constexpr int kThreads = 256;
constexpr int kCluster = 8; /* CTAs of a cluster at most */

struct NormShape {
    size_t samples, positions;
    int channels, groups, per_group;
    size_t xs, xp, ys, yp; /* strides of samples and positions */
    int act;
    float epsilon;
};

/* Tiles of a sample: `parts` of the positions by `blocks` of whole groups. */
struct Tiling {
    int pack;                /* elements of a load */
    int block_groups, lanes; /* groups and packs of a tile's row */
    int blocks, threads, rows_at_once;
    size_t rows;             /* positions of a part */
    size_t parts;
    bool fits;               /* the parts fit one cluster */
};

__device__ __forceinline__ float activate(float u, int act) {
    if (act == TB_ACT_SILU) return u * fast_sigmoid(u);
    if (act == TB_ACT_RELU) return u > 0.0f || u != u ? u : 0.0f;
    if (act == TB_ACT_GELU) return 0.5f * u * (1.0f + erff(u * 0.70710678f));
    return u;
}

__device__ __forceinline__ float slope(float u, int act) {
    if (act == TB_ACT_SILU) {
        const float s = fast_sigmoid(u);
        return s * (1.0f + u * (1.0f - s));
    }
    if (act == TB_ACT_RELU) return u > 0.0f ? 1.0f : 0.0f;
    if (act == TB_ACT_GELU) return 0.5f * (1.0f + erff(u * 0.70710678f)) + u * expf(-0.5f * u * u) * 0.39894228f;
    return 1.0f;
}

/* ---- a tile ---- */

/* Packs that a thread holds: 32 registers' worth. */
template <class T, int PACK> constexpr int kHeld = PACK * sizeof(T) == 16 ? 8 : 32;

/* Where a CTA and its thread are. */
struct Seat {
    size_t n, part;
    int block, lane, row, c0; /* c0: the tile's first channel */
    size_t first;             /* the tile's first position */
    int rows;                 /* its positions */
    bool in;                  /* the thread has a place in the rows */
    int mine;                 /* positions of the thread */
};

__device__ __forceinline__ Seat seat_of(const NormShape &d, const Tiling &g, size_t tile) {
    Seat s;
    s.part = tile % g.parts; /* the parts of a cluster are neighbours */
    s.block = static_cast<int>(tile / g.parts % g.blocks);
    s.n = tile / g.parts / g.blocks;
    s.c0 = s.block * g.block_groups * d.per_group;
    s.lane = threadIdx.x % g.lanes;
    s.row = threadIdx.x / g.lanes;
    s.first = s.part * g.rows;
    const size_t left = d.positions - s.first;
    s.rows = static_cast<int>(left < g.rows ? left : g.rows);
    s.in = s.row < g.rows_at_once;
    s.mine = s.in && s.row < s.rows ? (s.rows - s.row + g.rows_at_once - 1) / g.rows_at_once : 0;
    return s;
}

template <class T, int PACK, int HELD>
__device__ __forceinline__ void load_tile(Held<T, PACK> (&v)[HELD], const T *p, size_t stride, const Seat &s, const Tiling &g) {
    p += (s.first + s.row) * stride + s.c0 + s.lane * PACK;
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        if (i < s.mine) v[i] = *reinterpret_cast<const Held<T, PACK> *>(p);
        p += g.rows_at_once * stride;
    }
}

/* ---- sums over a tile ---- */

/* Shared memory of a tile: rows of per-channel partial sums (pitch channels +
 * 4), channel totals, and per group four values. */
struct Sums {
    float *rows, *channel, *group;
    int pitch;
};
__device__ __forceinline__ Sums sums_of(float *shared, const NormShape &d, const Tiling &g) {
    Sums s;
    const int channels = g.lanes * g.pack;
    s.pitch = channels + 4;
    s.rows = shared;
    s.channel = shared + g.rows_at_once * s.pitch;
    s.group = s.channel + 2 * ((channels + 3) & ~3);
    return s;
}
size_t sums_bytes(const Tiling &g) {
    const size_t channels = static_cast<size_t>(g.lanes) * g.pack;
    return (g.rows_at_once * (channels + 4) + 2 * ((channels + 3) & ~size_t(3)) + 4 * g.block_groups) * sizeof(float);
}

/* channel[c] = the sum over the CTA's rows of each thread's own[PACK]; ends
 * with the totals visible to all. */
template <int PACK>
__device__ __forceinline__ void channel_totals(const float (&own)[PACK], float *channel, const Sums &s, const Seat &at,
                                               const Tiling &g) {
    if (at.in) {
        float *to = s.rows + at.row * s.pitch + at.lane * PACK;
        if constexpr (PACK % 4 == 0) {
#pragma unroll
            for (int v = 0; v < PACK; v += 4)
                *reinterpret_cast<float4 *>(to + v) = make_float4(own[v], own[v + 1], own[v + 2], own[v + 3]);
        } else {
#pragma unroll
            for (int v = 0; v < PACK; ++v) to[v] = own[v];
        }
    }
    __syncthreads();
    /* `share` neighbouring threads for each channel */
    const int channels = g.lanes * PACK;
    int share = 1;
    while (share < 32 && share * 2 * channels <= static_cast<int>(blockDim.x)) share *= 2;
    const int mine = threadIdx.x % share;
    for (int base = 0; base < channels; base += blockDim.x / share) {
        const int c = base + threadIdx.x / share;
        float t = 0.0f;
        if (c < channels)
            for (int r = mine; r < g.rows_at_once; r += share) t += s.rows[r * s.pitch + c];
        for (int o = 1; o < share; o *= 2) t += __shfl_xor_sync(0xffffffffu, t, o);
        if (c < channels && mine == 0) channel[c] = t;
    }
    __syncthreads();
}

/* f(group, sum over its channels of value(channel)) for each of the tile's groups, by one thread each. */
template <class Value, class F>
__device__ __forceinline__ void group_totals(const NormShape &d, const Tiling &g, Value &&value, F &&f) {
    if (d.per_group <= 32) {
        for (int i = threadIdx.x; i < g.block_groups; i += blockDim.x) {
            float t = 0.0f;
            for (int c = i * d.per_group; c < (i + 1) * d.per_group; ++c) t += value(c);
            f(i, t);
        }
    } else {
        for (int i = threadIdx.x / 32; i < g.block_groups; i += blockDim.x / 32) {
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
template <class T, int PACK, int HELD>
__device__ __forceinline__ void tile_statistics(const Held<T, PACK> (&v)[HELD], const Sums &s, const Seat &at, const NormShape &d,
                                                const Tiling &g) {
    float own[PACK];
#pragma unroll
    for (int k = 0; k < PACK; ++k) own[k] = 0.0f;
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (i < at.mine) {
            float e[PACK];
            unpack(v[i], e);
#pragma unroll
            for (int k = 0; k < PACK; ++k) own[k] += e[k];
        }
    channel_totals<PACK>(own, s.channel, s, at, g);
    const float count = static_cast<float>(at.rows) * static_cast<float>(d.per_group);
    group_totals(d, g, [&](int c) { return s.channel[c]; }, [&](int i, float t) { s.group[2 * i] = t / count; });
    __syncthreads();
    float mean[PACK];
#pragma unroll
    for (int k = 0; k < PACK; ++k) {
        mean[k] = at.in ? s.group[2 * ((at.lane * PACK + k) / d.per_group)] : 0.0f;
        own[k] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (i < at.mine) {
            float e[PACK];
            unpack(v[i], e);
#pragma unroll
            for (int k = 0; k < PACK; ++k) {
                const float off = e[k] - mean[k];
                own[k] = fmaf(off, off, own[k]);
            }
        }
    channel_totals<PACK>(own, s.channel, s, at, g);
    group_totals(d, g, [&](int c) { return s.channel[c]; }, [&](int i, float t) { s.group[2 * i + 1] = t; });
    __syncthreads();
}

/* A thread's channels: u = (x - mean) scale + shift. */
template <int PACK> struct Affine {
    float mean[PACK], scale[PACK], shift[PACK];
};

template <class T, int PACK, int HELD>
__device__ __forceinline__ void write_tile(const Held<T, PACK> (&v)[HELD], const Affine<PACK> &f, T *p, size_t stride, int act,
                                           const Seat &s, const Tiling &g) {
    p += (s.first + s.row) * stride + s.c0 + s.lane * PACK;
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        if (i < s.mine) {
            float e[PACK];
            unpack(v[i], e);
#pragma unroll
            for (int k = 0; k < PACK; ++k) e[k] = activate(fmaf(e[k] - f.mean[k], f.scale[k], f.shift[k]), act);
            *reinterpret_cast<Held<T, PACK> *>(p) = packed<T, PACK>(e);
        }
        p += g.rows_at_once * stride;
    }
}

/* The tile's statistics and, where the whole sample's groups are in the
 * cluster, its result; else the statistics go to partial [samples, blocks,
 * parts, 2 block_groups]. */
template <class T, int PACK, bool WHOLE>
__global__ void __launch_bounds__(kThreads, 3)
norm_forward_tiles(NormShape d, Tiling g, const T *x, const float *gamma, const float *beta, T *y, float *mean_out,
                   float *rstd_out, float *partial) {
    extern __shared__ __align__(16) float shared[];
    constexpr int HELD = kHeld<T, PACK>;
    const Seat at = seat_of(d, g, blockIdx.x);
    const Sums s = sums_of(shared, d, g);
    Held<T, PACK> v[HELD];
    load_tile(v, x + at.n * d.xs, d.xp, at, g);
    tile_statistics(v, s, at, d, g);
    if constexpr (!WHOLE) {
        for (int i = threadIdx.x; i < 2 * g.block_groups; i += blockDim.x)
            partial[static_cast<size_t>(blockIdx.x) * 2 * g.block_groups + i] = s.group[i];
    } else {
        float *merged = s.group + 2 * g.block_groups;
        cg::cluster_group cluster = cg::this_cluster();
        if (g.parts > 1) cluster.sync();
        for (int i = threadIdx.x; i < g.block_groups; i += blockDim.x) {
            float mean = s.group[2 * i], squares = s.group[2 * i + 1];
            const float total = static_cast<float>(d.positions) * static_cast<float>(d.per_group);
            if (g.parts > 1) { /* in the parts' order */
                float sum = 0.0f;
                for (unsigned r = 0; r < g.parts; ++r) {
                    const float rows = static_cast<float>(r + 1 < g.parts ? g.rows : d.positions - r * g.rows);
                    sum += rows * cluster.map_shared_rank(s.group, r)[2 * i];
                }
                mean = sum / static_cast<float>(d.positions);
                squares = 0.0f;
                for (unsigned r = 0; r < g.parts; ++r) {
                    const float rows = static_cast<float>(r + 1 < g.parts ? g.rows : d.positions - r * g.rows);
                    const float *other = cluster.map_shared_rank(s.group, r) + 2 * i;
                    const float off = other[0] - mean;
                    squares += fmaf(rows * static_cast<float>(d.per_group) * off, off, other[1]);
                }
            }
            const float rstd = 1.0f / sqrtf(squares / total + d.epsilon);
            merged[2 * i] = mean;
            merged[2 * i + 1] = rstd;
            if (mean_out && at.part == 0) {
                const size_t to = at.n * d.groups + at.block * g.block_groups + i;
                mean_out[to] = mean;
                rstd_out[to] = rstd;
            }
        }
        if (g.parts > 1) cluster.barrier_arrive(); /* no CTA leaves before the others have read */
        __syncthreads();
        Affine<PACK> f;
#pragma unroll
        for (int k = 0; k < PACK; ++k) {
            const int c = at.lane * PACK + k, i = at.in ? c / d.per_group : 0;
            f.mean[k] = merged[2 * i];
            f.scale[k] = merged[2 * i + 1] * (gamma && at.in ? gamma[at.c0 + c] : 1.0f);
            f.shift[k] = beta && at.in ? beta[at.c0 + c] : 0.0f;
        }
        write_tile(v, f, y + at.n * d.ys, d.yp, d.act, at, g);
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
    const auto rows = [&](size_t r) { return static_cast<float>(r + 1 < g.parts ? g.rows : d.positions - r * g.rows); };
    float sum = 0.0f;
    for (size_t r = lane; r < g.parts; r += 32) sum += rows(r) * p[r * pitch];
    const float mean = warp_sum(sum) / static_cast<float>(d.positions);
    float squares = 0.0f;
    for (size_t r = lane; r < g.parts; r += 32) {
        const float off = p[r * pitch] - mean;
        squares += fmaf(rows(r) * static_cast<float>(d.per_group) * off, off, p[r * pitch + 1]);
    }
    squares = warp_sum(squares);
    if (lane == 0) {
        mean_out[at] = mean;
        rstd_out[at] = 1.0f / sqrtf(squares / (static_cast<float>(d.positions) * static_cast<float>(d.per_group)) + d.epsilon);
    }
}

/* The result from given statistics. */
template <class T, int PACK>
__global__ void __launch_bounds__(kThreads, 3)
norm_forward_apply(NormShape d, Tiling g, const T *x, const float *gamma, const float *beta, const float *mean,
                   const float *rstd, T *y) {
    constexpr int HELD = kHeld<T, PACK>;
    const Seat at = seat_of(d, g, gridDim.x - 1 - blockIdx.x);
    Held<T, PACK> v[HELD];
    load_tile(v, x + at.n * d.xs, d.xp, at, g);
    Affine<PACK> f;
#pragma unroll
    for (int k = 0; k < PACK; ++k) {
        const int c = at.c0 + (at.in ? at.lane * PACK + k : 0);
        const size_t i = at.n * d.groups + c / d.per_group;
        f.mean[k] = mean[i];
        f.scale[k] = rstd[i] * (gamma ? gamma[c] : 1.0f);
        f.shift[k] = beta ? beta[c] : 0.0f;
    }
    write_tile(v, f, y + at.n * d.ys, d.yp, d.act, at, g);
}

/* ---- backward ---- */

/* hat = (x - mean) rstd, u = hat gamma + beta. */
template <int PACK> struct Given {
    float mean[PACK], rstd[PACK], gamma[PACK], beta[PACK];
};
template <int PACK>
__device__ __forceinline__ Given<PACK> given_of(const NormShape &d, const Seat &at, const float *gamma, const float *beta,
                                                const float *mean, const float *rstd) {
    Given<PACK> f;
#pragma unroll
    for (int k = 0; k < PACK; ++k) {
        const int c = at.c0 + (at.in ? at.lane * PACK + k : 0);
        const size_t i = at.n * d.groups + c / d.per_group;
        f.mean[k] = mean[i];
        f.rstd[k] = rstd[i];
        f.gamma[k] = gamma ? gamma[c] : 1.0f;
        f.beta[k] = beta ? beta[c] : 0.0f;
    }
    return f;
}

/* Leaves per channel the sums of du in s.channel, of du hat behind them, and per
 * group those of du gamma and du gamma hat in s.group; visible to all. */
template <class T, int PACK, int HELD>
__device__ __forceinline__ void tile_gradients(const Held<T, PACK> (&v)[HELD], const Held<T, PACK> (&w)[HELD],
                                               const Given<PACK> &f, const float *gamma, const Sums &s, const Seat &at,
                                               const NormShape &d, const Tiling &g) {
    float a[PACK], b[PACK];
#pragma unroll
    for (int k = 0; k < PACK; ++k) a[k] = b[k] = 0.0f;
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (i < at.mine) {
            float e[PACK], dy[PACK];
            unpack(v[i], e);
            unpack(w[i], dy);
#pragma unroll
            for (int k = 0; k < PACK; ++k) {
                const float hat = (e[k] - f.mean[k]) * f.rstd[k];
                const float du = dy[k] * slope(fmaf(hat, f.gamma[k], f.beta[k]), d.act);
                a[k] += du;
                b[k] = fmaf(du, hat, b[k]);
            }
        }
    float *const second = s.channel + ((g.lanes * PACK + 3) & ~3);
    channel_totals<PACK>(a, s.channel, s, at, g);
    channel_totals<PACK>(b, second, s, at, g);
    const auto weighted = [&](const float *t) { return [=](int c) { return t[c] * (gamma ? gamma[at.c0 + c] : 1.0f); }; };
    group_totals(d, g, weighted(s.channel), [&](int i, float t) { s.group[2 * i] = t; });
    group_totals(d, g, weighted(second), [&](int i, float t) { s.group[2 * i + 1] = t; });
    __syncthreads();
}

/* dx = rstd (du gamma - m1 - hat m2); m1, m2: the group's means of du gamma, du gamma hat. */
template <class T, int PACK, int HELD>
__device__ __forceinline__ void write_gradients(const Held<T, PACK> (&v)[HELD], const Held<T, PACK> (&w)[HELD],
                                                const Given<PACK> &f, const float (&m1)[PACK], const float (&m2)[PACK], T *p,
                                                const NormShape &d, const Seat &s, const Tiling &g) {
    p += (s.first + s.row) * d.xp + s.c0 + s.lane * PACK;
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        if (i < s.mine) {
            float e[PACK], dy[PACK];
            unpack(v[i], e);
            unpack(w[i], dy);
#pragma unroll
            for (int k = 0; k < PACK; ++k) {
                const float hat = (e[k] - f.mean[k]) * f.rstd[k];
                const float du = dy[k] * slope(fmaf(hat, f.gamma[k], f.beta[k]), d.act);
                e[k] = f.rstd[k] * (fmaf(du, f.gamma[k], -m1[k]) - hat * m2[k]);
            }
            *reinterpret_cast<Held<T, PACK> *>(p) = packed<T, PACK>(e);
        }
        p += g.rows_at_once * d.xp;
    }
}

/* The tile's sums and, where the whole sample's groups are in the cluster, dx.
 * Per-channel sums go to partial [samples, parts, 2, channels], and where the
 * sample is larger the groups' to sums [samples, parts, 2, groups]. */
template <class T, int PACK, bool WHOLE>
__global__ void __launch_bounds__(kThreads, 2)
norm_backward_tiles(NormShape d, Tiling g, const T *x, const float *gamma, const float *beta, const float *mean,
                    const float *rstd, const T *dy, T *dx, float *partial, float *sums) {
    extern __shared__ __align__(16) float shared[];
    constexpr int HELD = kHeld<T, PACK>;
    const Seat at = seat_of(d, g, blockIdx.x);
    const Sums s = sums_of(shared, d, g);
    Held<T, PACK> v[HELD], w[HELD];
    load_tile(v, x + at.n * d.xs, d.xp, at, g);
    load_tile(w, dy + at.n * d.ys, d.yp, at, g);
    const Given<PACK> f = given_of<PACK>(d, at, gamma, beta, mean, rstd);
    tile_gradients(v, w, f, gamma, s, at, d, g);
    const int channels = g.lanes * PACK, second = (channels + 3) & ~3;
    if (partial) {
        float *to = partial + (at.n * g.parts + at.part) * 2 * d.channels + at.c0;
        for (int c = threadIdx.x; c < channels; c += blockDim.x) {
            to[c] = s.channel[c];
            to[d.channels + c] = s.channel[second + c];
        }
    }
    if constexpr (!WHOLE) {
        float *to = sums + (at.n * g.parts + at.part) * 2 * d.groups + at.block * g.block_groups;
        for (int i = threadIdx.x; i < g.block_groups; i += blockDim.x) {
            to[i] = s.group[2 * i];
            to[d.groups + i] = s.group[2 * i + 1];
        }
    } else {
        float *merged = s.group + 2 * g.block_groups;
        cg::cluster_group cluster = cg::this_cluster();
        if (g.parts > 1) cluster.sync();
        const float count = static_cast<float>(d.positions) * static_cast<float>(d.per_group);
        for (int i = threadIdx.x; i < 2 * g.block_groups; i += blockDim.x) {
            float t = 0.0f;
            for (unsigned r = 0; r < g.parts; ++r)
                t += g.parts > 1 ? cluster.map_shared_rank(s.group, r)[i] : s.group[i];
            merged[i] = t / count;
        }
        if (g.parts > 1) cluster.barrier_arrive(); /* no CTA leaves before the others have read */
        __syncthreads();
        float m1[PACK], m2[PACK];
#pragma unroll
        for (int k = 0; k < PACK; ++k) {
            const int i = at.in ? (at.lane * PACK + k) / d.per_group : 0;
            m1[k] = merged[2 * i];
            m2[k] = merged[2 * i + 1];
        }
        write_gradients(v, w, f, m1, m2, dx + at.n * d.xs, d, at, g);
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
__global__ void __launch_bounds__(kThreads, 2)
norm_backward_apply(NormShape d, Tiling g, const T *x, const float *gamma, const float *beta, const float *mean,
                    const float *rstd, const float *means, const T *dy, T *dx) {
    constexpr int HELD = kHeld<T, PACK>;
    const Seat at = seat_of(d, g, gridDim.x - 1 - blockIdx.x);
    Held<T, PACK> v[HELD], w[HELD];
    load_tile(v, x + at.n * d.xs, d.xp, at, g);
    load_tile(w, dy + at.n * d.ys, d.yp, at, g);
    const Given<PACK> f = given_of<PACK>(d, at, gamma, beta, mean, rstd);
    float m1[PACK], m2[PACK];
#pragma unroll
    for (int k = 0; k < PACK; ++k) {
        const size_t i = at.n * d.groups + (at.c0 + (at.in ? at.lane * PACK + k : 0)) / d.per_group;
        m1[k] = means[2 * i];
        m2[k] = means[2 * i + 1];
    }
    write_gradients(v, w, f, m1, m2, dx + at.n * d.xs, d, at, g);
}

/* dbeta and dgamma from parts [rows, 2, channels]. */
__global__ void __launch_bounds__(kThreads)
norm_parameters(const float *parts, size_t rows, int channels, float *dgamma, float *dbeta) {
    const int c = blockIdx.x * kThreads + threadIdx.x;
    if (c >= 2 * channels) return;
    float s = 0.0f;
    for (size_t r = 0; r < rows; ++r) s += parts[r * 2 * channels + c];
    if (c < channels) {
        if (dbeta) dbeta[c] = s;
    } else if (dgamma) {
        dgamma[c - channels] = s;
    }
}

/* ---- groups wider than a CTA's rows: one CTA per (sample, group) ---- */

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

template <class T>
__global__ void __launch_bounds__(kThreads)
norm_forward_wide(NormShape d, const T *x, const float *gamma, const float *beta, T *y, float *mean_out, float *rstd_out) {
    __shared__ float scratch[kThreads / 32];
    const size_t n = blockIdx.x / d.groups;
    const int g = static_cast<int>(blockIdx.x % d.groups);
    const int c0 = g * d.per_group;
    const float count = static_cast<float>(d.positions) * static_cast<float>(d.per_group);
    const T *xs = x + n * d.xs + c0;
    float s = 0.0f;
    for (size_t p = 0; p < d.positions; ++p)
        for (int c = threadIdx.x; c < d.per_group; c += kThreads) s += to_float(xs[p * d.xp + c]);
    const float mean = block_sum(s, scratch) / count;
    s = 0.0f;
    for (size_t p = 0; p < d.positions; ++p)
        for (int c = threadIdx.x; c < d.per_group; c += kThreads) {
            const float v = to_float(xs[p * d.xp + c]) - mean;
            s = fmaf(v, v, s);
        }
    const float rstd = 1.0f / sqrtf(block_sum(s, scratch) / count + d.epsilon);
    if (threadIdx.x == 0 && mean_out) {
        mean_out[blockIdx.x] = mean;
        rstd_out[blockIdx.x] = rstd;
    }
    for (size_t p = 0; p < d.positions; ++p)
        for (int c = threadIdx.x; c < d.per_group; c += kThreads) {
            const float scale = rstd * (gamma ? gamma[c0 + c] : 1.0f);
            const float u = fmaf(to_float(xs[p * d.xp + c]) - mean, scale, beta ? beta[c0 + c] : 0.0f);
            y[n * d.ys + p * d.yp + c0 + c] = from_float<T>(activate(u, d.act));
        }
}

/* partial [samples, 2, channels]. */
template <class T>
__global__ void __launch_bounds__(kThreads)
norm_backward_wide(NormShape d, const T *x, const float *gamma, const float *beta, const float *mean_in,
                   const float *rstd_in, const T *dy, T *dx, float *partial) {
    __shared__ float scratch[kThreads / 32];
    const size_t n = blockIdx.x / d.groups;
    const int g = static_cast<int>(blockIdx.x % d.groups);
    const int c0 = g * d.per_group;
    const float mean = mean_in[blockIdx.x], rstd = rstd_in[blockIdx.x];
    float s1 = 0.0f, s2 = 0.0f;
    const auto gradient = [&](size_t p, int c, float ga, float be, float *hat) {
        *hat = (to_float(x[n * d.xs + p * d.xp + c]) - mean) * rstd;
        return to_float(dy[n * d.ys + p * d.yp + c]) * slope(fmaf(*hat, ga, be), d.act);
    };
    for (int c = c0 + threadIdx.x; c < c0 + d.per_group; c += kThreads) {
        const float ga = gamma ? gamma[c] : 1.0f, be = beta ? beta[c] : 0.0f;
        float a = 0.0f, b = 0.0f, hat;
        for (size_t p = 0; p < d.positions; ++p) {
            const float du = gradient(p, c, ga, be, &hat);
            a += du;
            b = fmaf(du, hat, b);
        }
        partial[n * 2 * d.channels + c] = a;
        partial[n * 2 * d.channels + d.channels + c] = b;
        s1 = fmaf(ga, a, s1);
        s2 = fmaf(ga, b, s2);
    }
    const float count = static_cast<float>(d.positions) * static_cast<float>(d.per_group);
    s1 = block_sum(s1, scratch) / count;
    s2 = block_sum(s2, scratch) / count;
    for (int c = c0 + threadIdx.x; c < c0 + d.per_group; c += kThreads) {
        const float ga = gamma ? gamma[c] : 1.0f, be = beta ? beta[c] : 0.0f;
        float hat;
        for (size_t p = 0; p < d.positions; ++p) {
            const float du = gradient(p, c, ga, be, &hat);
            dx[n * d.xs + p * d.xp + c] = from_float<T>(rstd * (fmaf(du, ga, -s1) - hat * s2));
        }
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
    if (s->xp < d->channels || s->yp < d->channels) return false;
    s->act = d->activation;
    s->epsilon = d->epsilon;
    return true;
}

/* Tiles for packs of `pack` elements; false where a group is wider than a
 * CTA's rows (or the tiles are too many to count). */
bool tiling_of(const NormShape &d, int pack, size_t size, Tiling *g) {
    const int held = pack * size == 16 ? 8 : 32;
    /* whole groups, whole packs, 128 bytes a row if there are: narrower rows
     * waste sectors, wider ones leave fewer and longer tiles */
    int best = 0;
    for (int i = 1; i <= d.groups && !best; ++i) {
        if (d.groups % i || static_cast<size_t>(i) * d.per_group % pack) continue;
        const size_t lanes = static_cast<size_t>(i) * d.per_group / pack;
        if (lanes > kThreads) break;
        g->block_groups = i;
        g->lanes = static_cast<int>(lanes);
        if (lanes * pack * size >= 128) best = i;
        else if (i == d.groups) best = i;
        else continue;
    }
    if (!best) return false;
    g->pack = pack;
    g->blocks = d.groups / g->block_groups;
    const size_t packs = d.positions * g->lanes;
    const size_t threads = packs < kThreads ? align_up(packs, 32) : kThreads;
    g->threads = static_cast<int>(threads < static_cast<size_t>(g->lanes) ? align_up(g->lanes, 32) : threads);
    g->rows_at_once = g->threads / g->lanes;
    const size_t most = static_cast<size_t>(g->rows_at_once) * held;
    g->parts = (d.positions + most - 1) / most;
    g->rows = (d.positions + g->parts - 1) / g->parts;
    g->parts = (d.positions + g->rows - 1) / g->rows;
    g->fits = g->parts <= kCluster;
    size_t tiles;
    return product(d.samples * g->blocks, g->parts, 0x7fffffffu, &tiles);
}

/* The widest pack that every row allows: 16 bytes, 4 bytes, an element. */
int pack_of(const NormShape &d, size_t size, const void *a, size_t as, size_t ap, const void *b, size_t bs, size_t bp) {
    const size_t all = reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | (as | ap | bs | bp) * size |
                       static_cast<size_t>(d.channels) * size;
    if (all % 16 == 0) return static_cast<int>(16 / size);
    return all % 4 == 0 ? static_cast<int>(4 / size) : 1;
}

/* Calls f with the pack as a constant. */
template <class T, class F> int with_pack(int pack, F &&f) {
    if (pack == 16 / static_cast<int>(sizeof(T))) return f(std::integral_constant<int, 16 / static_cast<int>(sizeof(T))>{});
    if constexpr (sizeof(T) == 2)
        if (pack == 2) return f(std::integral_constant<int, 2>{});
    return f(std::integral_constant<int, 1>{});
}

template <class Kernel, class... Args>
int launch_tiles(Kernel kernel, const NormShape &d, const Tiling &g, bool clusters, size_t shared, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t c{};
    c.gridDim = dim3(static_cast<unsigned>(d.samples * g.blocks * g.parts));
    c.blockDim = dim3(static_cast<unsigned>(g.threads));
    c.dynamicSmemBytes = shared;
    c.stream = st;
    cudaLaunchAttribute a{};
    if (clusters && g.parts > 1) {
        a.id = cudaLaunchAttributeClusterDimension;
        a.val.clusterDim = {static_cast<unsigned>(g.parts), 1, 1};
        c.attrs = &a;
        c.numAttrs = 1;
    }
    return cudaLaunchKernelEx(&c, kernel, d, g, args...) == cudaSuccess;
}

/* Workspace: the forward pass's partial statistics, or the backward pass's
 * per-channel rows with their column sums, group sums and means. */
size_t forward_bytes(const NormShape &d, const Tiling &g) {
    return (2 * d.samples * d.groups + d.samples * g.parts * 2 * d.groups) * sizeof(float);
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
        if (s.channels % pack || !tiling_of(s, pack, size, &g)) continue;
        const size_t f = g.fits ? 0 : forward_bytes(s, g), b = backward_bytes(s, g.parts);
        need = f > need ? f : need;
        need = b > need ? b : need;
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
        !aligned(rstd, 4) || !aligned(workspace, 16) || (x == y && (s.xs != s.ys || s.xp != s.yp)))
        return 0;
    cudaGetLastError(); /* report these launches only */
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return with_type(desc->type, [&](auto t) {
        using T = decltype(t);
        const T *in = static_cast<const T *>(x);
        T *out = static_cast<T *>(y);
        Tiling g;
        const int pack = pack_of(s, size, x, s.xs, s.xp, y, s.ys, s.yp);
        if (!tiling_of(s, pack, size, &g)) {
            norm_forward_wide<T><<<static_cast<unsigned>(s.samples * s.groups), kThreads, 0, st>>>(s, in, gamma, beta, out,
                                                                                             mean, rstd);
            return launched();
        }
        return with_pack<T>(pack, [&](auto p) {
            constexpr int P = decltype(p)::value;
            if (g.fits)
                return launch_tiles(norm_forward_tiles<T, P, true>, s, g, true, sums_bytes(g), st, in, gamma, beta, out, mean,
                                    rstd, static_cast<float *>(nullptr));
            float *means = static_cast<float *>(workspace), *partial = means + 2 * s.samples * s.groups;
            float *m = mean ? mean : means, *r = rstd ? rstd : means + s.samples * s.groups;
            if (!launch_tiles(norm_forward_tiles<T, P, false>, s, g, false, sums_bytes(g), st, in, gamma, beta, out, m, r, partial))
                return 0;
            norm_merge<<<merge_grid(s), kThreads, 0, st>>>(s, g, partial, m, r);
            if (!launched()) return 0;
            return launch_tiles(norm_forward_apply<T, P>, s, g, false, 0, st, in, gamma, beta, m, r, out);
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
        !aligned(workspace, 16) || (dx == dy && (s.xs != s.ys || s.xp != s.yp)))
        return 0;
    cudaGetLastError(); /* report these launches only */
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int ok_rows = with_type(desc->type, [&](auto t) -> int {
        using T = decltype(t);
        const T *in = static_cast<const T *>(x), *grad = static_cast<const T *>(dy);
        T *out = static_cast<T *>(dx);
        Tiling g;
        float *partial = static_cast<float *>(workspace);
        const uintptr_t both = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(dx);
        const int pack = pack_of(s, size, reinterpret_cast<const void *>(both), s.xs, s.xp, dy, s.ys, s.yp);
        const bool wide = !tiling_of(s, pack, size, &g);
        const size_t rows = s.samples * (wide ? 1 : g.parts), parts = column_parts(rows);
        float *columns = partial + rows * 2 * s.channels, *sums = columns + parts * 2 * s.channels;
        float *rows_to = wide || dgamma || dbeta ? partial : nullptr;
        if (wide) {
            norm_backward_wide<T><<<static_cast<unsigned>(s.samples * s.groups), kThreads, 0, st>>>(
                s, in, gamma, beta, mean, rstd, grad, out, partial);
            if (!launched()) return 0;
        } else {
            const int ok = with_pack<T>(pack, [&](auto p) {
                constexpr int P = decltype(p)::value;
                if (g.fits)
                    return launch_tiles(norm_backward_tiles<T, P, true>, s, g, true, sums_bytes(g), st, in, gamma, beta, mean,
                                        rstd, grad, out, rows_to, sums);
                float *means = sums + rows * 2 * s.groups;
                if (!launch_tiles(norm_backward_tiles<T, P, false>, s, g, false, sums_bytes(g), st, in, gamma, beta, mean, rstd,
                                  grad, out, rows_to, sums))
                    return 0;
                norm_merge_sums<<<merge_grid(s), kThreads, 0, st>>>(s, g.parts, sums, means);
                if (!launched()) return 0;
                return launch_tiles(norm_backward_apply<T, P>, s, g, false, 0, st, in, gamma, beta, mean, rstd, means, grad,
                                    out);
            });
            if (!ok) return 0;
        }
        if (!dgamma && !dbeta) return 1;
        column_sums<<<dim3(static_cast<unsigned>((2 * s.channels + 31) / 32), static_cast<unsigned>(parts)), kColumnThreads,
                      0, st>>>(partial, rows, 2 * static_cast<size_t>(s.channels), columns);
        if (!launched()) return 0;
        norm_parameters<<<(2 * s.channels + kThreads - 1) / kThreads, kThreads, 0, st>>>(columns, parts, s.channels, dgamma,
                                                                                        dbeta);
        return launched();
    });
    return ok_rows;
}
