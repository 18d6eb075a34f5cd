/*
 * Orthogonalising updates by Newton-Schulz products
 * (include/turbinator/training/cuda_learner.h).
 *
 * x = g / (|g| + epsilon), then `steps` times S = b A + c A A with A = x x^T
 * and x = a x + S x (for a matrix taller than wide A = x^T x and x = a x + x S:
 * no transposes, the tensor cores take either order).  Three products a step,
 * A and S symmetric, so that a little over half of their tiles are computed and
 * the others mirrored.
 *
 * x, A and S are kept times 2^12 as pairs of f16 values, the second what the
 * rounding of the first left, 2^11 higher: 22 bits for values down to 2^-26 (a
 * unit matrix's share is some 2^-5 to 2^-12) and 2^-48 absolute below, so that rows
 * far smaller than others keep their digits.  A product of pairs is three
 * products of f16 (the fourth is below 2^-22); the polynomial multiplies an
 * error in a direction of a small singular value by up to a^steps, 485 for five
 * steps of the quintic, so that plain bf16 products leave errors of 2 to 3 % in
 * the result and f16 ones 0.2 to 0.4 %, pairs 1e-6.
 */
#include <algorithm>

#include "tb_tensor.cuh"

using namespace tb_learn;
using tb_tensor::Matrices;
using tb_tensor::Operands;
using tb_tensor::Tile;

namespace {

constexpr float kUp = 4096.0f; /* of every kept value */
constexpr float kDown = 1.0f / 4096.0f;
constexpr float kLowUp = 1 << tb_tensor::kPlaneRise<2>; /* of the second plane beyond that */
constexpr float kLowDown = 1.0f / kLowUp;
__device__ __forceinline__ float joined(__half high, __half low) { return fmaf(__half2float(low), kLowDown, __half2float(high)); }
__device__ __forceinline__ void part(float v, __half *high, __half *low) {
    *high = __float2half_rn(v);
    *low = __float2half_rn((v - __half2float(*high)) * kLowUp);
}

/* A stack of matrices as two planes: the second `plane` elements on. */
struct Pair {
    __half *at;
    size_t line, matrix, plane;
    __device__ __forceinline__ float get(size_t i) const { return joined(at[i], at[plane + i]); }
    __device__ __forceinline__ void put(size_t i, float v) const { part(v, &at[i], &at[plane + i]); }
};

/* ---- x = g / (|g| + epsilon) ---- */

constexpr int kNormThreads = 256;
constexpr size_t kMostParts = 512;  /* of a matrix */
constexpr size_t kPartValues = 2048; /* of a part at least */
constexpr size_t kManyParts = 8192;  /* of all matrices */

struct Given {
    size_t rows, columns, matrix_stride, row_stride, rows_a_part;
    int lanes; /* that take a row together, a power of two */
};

/* Calls f(row, column, values) for this lane's packs of the part of the matrix
 * that blockIdx.x takes, four under way at once. */
template <int PACK, class T, class F> __device__ __forceinline__ void each_pack(const Given &d, const T *from, F &&f) {
    const size_t first = blockIdx.x * d.rows_a_part, last = min(first + d.rows_a_part, d.rows);
    const unsigned team = threadIdx.x / d.lanes, teams = kNormThreads / d.lanes, lane = threadIdx.x - team * d.lanes;
    for (size_t r = first + team; r < last; r += teams)
        for (size_t c = lane * PACK; c < d.columns; c += static_cast<size_t>(d.lanes) * PACK * 4) {
            Held<T, PACK> h[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const size_t at = c + static_cast<size_t>(i) * d.lanes * PACK;
                if (at < d.columns) h[i] = *reinterpret_cast<const Held<T, PACK> *>(from + r * d.row_stride + at);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const size_t at = c + static_cast<size_t>(i) * d.lanes * PACK;
                float e[PACK];
                if (at < d.columns) unpack(h[i], e), f(r, at, e);
            }
        }
}

/* The squares are summed in 64 bits: those of f32 may pass f32's range either way. */
template <class T, int PACK>
__global__ void __launch_bounds__(kNormThreads) squares(Given d, const T *g, double *sums) {
    __shared__ double parts[kNormThreads / 32];
    later_may_start();
    const T *from = g + blockIdx.y * d.matrix_stride;
    double s = 0.0;
    each_pack<PACK>(d, from, [&](size_t, size_t, const float (&e)[PACK]) {
#pragma unroll
        for (int i = 0; i < PACK; ++i) s = fma(static_cast<double>(e[i]), static_cast<double>(e[i]), s);
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (threadIdx.x % 32 == 0) parts[threadIdx.x / 32] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < kNormThreads / 32; ++i) s += parts[i];
        sums[blockIdx.y * gridDim.x + blockIdx.x] = s;
    }
}

template <class T, int PACK>
__global__ void __launch_bounds__(kNormThreads) normalise(Given d, const T *g, const double *sums, double epsilon, Pair x) {
    __shared__ double scale;
    later_may_start();
    after_earlier();
    if (threadIdx.x < 32) {
        double s = 0.0;
        for (unsigned i = threadIdx.x; i < gridDim.x; i += 32) s += sums[blockIdx.y * gridDim.x + i];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        /* nothing stays nothing; a matrix with an infinity or a NaN becomes NaN */
        if (threadIdx.x == 0) scale = s == 0.0 ? 0.0 : isfinite(s) ? kUp / (sqrt(s) + epsilon) : s - s;
    }
    __syncthreads();
    const double up = scale;
    const float near = static_cast<float>(up); /* where f32 holds it, the products do too */
    const bool plain = fabsf(near) < 1e30f && (near > 1e-30f || up == 0.0);
    const T *from = g + blockIdx.y * d.matrix_stride;
    __half *to = x.at + blockIdx.y * x.matrix;
    each_pack<PACK>(d, from, [&](size_t r, size_t c, const float (&e)[PACK]) {
        Pack<__half, PACK> high, low;
#pragma unroll
        for (int i = 0; i < PACK; ++i) {
            const float v = plain ? e[i] * near : static_cast<float>(static_cast<double>(e[i]) * up);
            part(v, &high.v[i], &low.v[i]);
        }
        *reinterpret_cast<Pack<__half, PACK> *>(to + r * x.line + c) = high;
        *reinterpret_cast<Pack<__half, PACK> *>(to + x.plane + r * x.line + c) = low;
    });
}

/* ---- the products ---- */

/* Tiles of a matrix [height, width] of the output; symmetric: those that touch
 * m >= n, each mirrored where the tile across the diagonal is not computed. */
struct Plan {
    int matrices, width, height, depth, tile_m, tile_n;
    bool symmetric;
    int tiles_m, per;

    __host__ __device__ int first(int n) const { return symmetric ? n * tile_n / tile_m : 0; }
    void count() {
        tiles_m = (width + tile_m - 1) / tile_m;
        per = 0;
        for (int n = 0; n * tile_n < height; ++n) per += tiles_m - first(n);
    }
    __device__ __forceinline__ Tile tile(int t) const {
        const int z = t / per;
        int in = t - z * per, n = 0, m;
        if (symmetric) {
            for (; in >= tiles_m - first(n); ++n) in -= tiles_m - first(n);
            m = first(n) + in;
        } else {
            n = in / tiles_m;
            m = in - n * tiles_m;
        }
        Tile r;
        r.m0 = m * tile_m;
        r.n0 = n * tile_n;
        r.columns = min(tile_n, height - r.n0);
        r.k0 = 0;
        r.depth = depth;
        r.az = r.bz = r.which = z;
        return r;
    }
    /* Whether what lies across the diagonal from row m of the 32 columns from c is in no tile. */
    __device__ __forceinline__ bool mirrored(const Tile &t, int m, int c) const {
        return symmetric && (t.n0 + c) / tile_m < first(m / tile_n);
    }
};

struct Nothing {};

constexpr int kBoxBytes = 32 * 32 * sizeof(__half);

/* 32 columns of 32 rows of the tensor cores as pairs, [column][row] (or
 * [row][column]) in a warp's staging, and from there in whole boxes: to global
 * memory directly, 64 bytes at a time, a tile's storing took twice as long. */
struct Boxes {
    int lane;
    __half *at;
    __device__ __forceinline__ float get(int i) const { return joined(at[i * 32 + lane], at[1024 + i * 32 + lane]); }
    __device__ __forceinline__ void put(int i, float v, __half *high, __half *low) const {
        part(v, high, low);
        at[i * 32 + lane] = *high;
        at[1024 + i * 32 + lane] = *low;
    }
    __device__ __forceinline__ void across(const __half (&high)[32], const __half (&low)[32]) const {
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
            Pack<__half, 8> h, l;
#pragma unroll
            for (int j = 0; j < 8; ++j) h.v[j] = high[i + j], l.v[j] = low[i + j];
            *reinterpret_cast<Pack<__half, 8> *>(at + lane * 32 + i) = h;
            *reinterpret_cast<Pack<__half, 8> *>(at + 1024 + lane * 32 + i) = l;
        }
    }
};

/* A = x x^T, or S = b A + c A A. */
struct SquareJob {
    static constexpr bool kRagged = false;
    static constexpr int kStaging = 2 * kBoxBytes;
    using Shared = Nothing;
    CUtensorMap out, old; /* boxes of 32 x 32 */
    Plan plan;
    Pair to, from; /* the same */
    bool second;   /* S */
    float b, c;
    __device__ void setup(Shared &) const {}
    __device__ int tiles(const Shared &) const { return plan.matrices * plan.per; }
    __device__ Tile tile(const Shared &, int t) const { return plan.tile(t); }
    __device__ __forceinline__ void ask(const Tile &t, int m, int c0, tb_tensor::Staging &s) const {
        if (second && m - s.lane < plan.width) s.load(&old, m - s.lane, t.n0 + c0, t.which, plan.matrices, kBoxBytes);
    }
    __device__ __forceinline__ bool store(const Tile &t, int m, int c0, float (&v)[32], tb_tensor::Staging &s) const {
        const int x = m - s.lane, y = t.n0 + c0;
        if (x >= plan.width) return true;
        const Boxes boxes{s.lane, reinterpret_cast<__half *>(s.at)};
        __half high[32], low[32];
        if (second) {
            if (!s.loaded()) return false;
#pragma unroll
            for (int i = 0; i < 32; ++i) boxes.put(i, fmaf(c, v[i] * kDown, b * boxes.get(i)), &high[i], &low[i]);
        } else {
            s.free();
#pragma unroll
            for (int i = 0; i < 32; ++i) boxes.put(i, v[i] * kDown, &high[i], &low[i]);
        }
        s.store(&out, x, y, t.which, plan.matrices, kBoxBytes);
        if (plan.mirrored(t, x, c0)) {
            s.free();
            boxes.across(high, low);
            s.store(&out, y, x, t.which, plan.matrices, kBoxBytes);
        }
        return true;
    }
    __device__ __forceinline__ void store_joined(const Tile &t, int m, int c0, const uint32_t (&r)[8]) const {
        if (m >= plan.width) return;
        const size_t base = t.which * to.matrix;
        __half *down = to.at + base + (t.n0 + c0) * to.line + m;
        const size_t was = base + (t.n0 + c0) * from.line + m;
        Pack<__half, 8> high, low;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float e = __uint_as_float(r[i]) * kDown;
            if (second && c0 + i < t.columns) e = fmaf(c, e, b * from.get(was + i * from.line));
            part(e, &high.v[i], &low.v[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c0 + i < t.columns) {
                down[i * to.line] = high.v[i];
                down[to.plane + i * to.line] = low.v[i];
            }
        if (plan.mirrored(t, m, c0)) { /* a line's end is a multiple of eight */
            __half *across = to.at + base + m * to.line + t.n0 + c0;
            *reinterpret_cast<Pack<__half, 8> *>(across) = high;
            *reinterpret_cast<Pack<__half, 8> *>(across + to.plane) = low;
        }
    }
};

/* x = a x + S x; the last step's goes to the output. */
template <class T> struct StepJob {
    static constexpr bool kRagged = false;
    static constexpr int kStaging = 2 * kBoxBytes;
    using Shared = Nothing;
    CUtensorMap x, next; /* boxes of 32 x 32 */
    Plan plan;
    Pair to, from; /* the same */
    T *last; /* or NULL */
    size_t row_stride, matrix_stride;
    float a, scale;
    __device__ void setup(Shared &) const {}
    __device__ int tiles(const Shared &) const { return plan.matrices * plan.per; }
    __device__ Tile tile(const Shared &, int t) const { return plan.tile(t); }
    __device__ __forceinline__ void ask(const Tile &t, int m, int c0, tb_tensor::Staging &s) const {
        if (m - s.lane < plan.width) s.load(&x, m - s.lane, t.n0 + c0, t.which, plan.matrices, kBoxBytes);
    }
    __device__ __forceinline__ bool store(const Tile &t, int m, int c0, float (&v)[32], tb_tensor::Staging &s) const {
        const int left = m - s.lane, y = t.n0 + c0;
        if (left >= plan.width) return true;
        const Boxes boxes{s.lane, reinterpret_cast<__half *>(s.at)};
        if (!s.loaded()) return false;
        if (last) {
            T *o = last + t.which * matrix_stride + y * row_stride + m;
#pragma unroll
            for (int i = 0; i < 32; ++i, o += row_stride)
                if (m < plan.width && c0 + i < t.columns) *o = from_float<T>(fmaf(a, boxes.get(i), v[i] * kDown) * kDown * scale);
            __syncwarp(); /* the next boxes come where these were */
        } else {
            __half high, low;
#pragma unroll
            for (int i = 0; i < 32; ++i) boxes.put(i, fmaf(a, boxes.get(i), v[i] * kDown), &high, &low);
            s.store(&next, left, y, t.which, plan.matrices, kBoxBytes);
        }
        return true;
    }
    __device__ __forceinline__ void store_joined(const Tile &t, int m, int c0, const uint32_t (&r)[8]) const {
        if (m >= plan.width) return;
        const size_t n = t.n0 + c0, at = t.which * from.matrix + n * from.line + m;
        float e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            e[i] = c0 + i < t.columns ? fmaf(a, from.get(at + i * from.line), __uint_as_float(r[i]) * kDown) : 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c0 + i < t.columns) {
                if (last) last[t.which * matrix_stride + (n + i) * row_stride + m] = from_float<T>(e[i] * kDown * scale);
                else to.put(at + i * to.line, e[i]);
            }
    }
};

struct OrthogonalShape {
    size_t matrices, rows, columns, small, in_matrix, in_row, out_matrix, out_row;
    bool tall;
};
bool orthogonal_shape(const tb_orthogonalise_desc *d, OrthogonalShape *s) {
    if (!d || !d->matrices || !d->rows || !d->columns || !type_known(d->type) || d->steps < 1 || d->steps > 64 ||
        d->rows > TB_ORTHOGONALISE_MAX_SIDE || d->columns > TB_ORTHOGONALISE_MAX_SIDE || d->matrices > 65535 ||
        !(d->epsilon >= 0.0f))
        return false;
    s->matrices = d->matrices;
    s->rows = d->rows;
    s->columns = d->columns;
    s->tall = s->rows > s->columns;
    s->small = s->tall ? s->columns : s->rows;
    s->in_row = d->in_row_stride ? d->in_row_stride : s->columns;
    s->out_row = d->out_row_stride ? d->out_row_stride : s->columns;
    if (s->in_row < s->columns || s->out_row < s->columns) return false;
    size_t in, out, all;
    if (!product(s->rows, s->in_row, SIZE_MAX / 64, &in) || !product(s->rows, s->out_row, SIZE_MAX / 64, &out)) return false;
    s->in_matrix = d->in_matrix_stride ? d->in_matrix_stride : in;
    s->out_matrix = d->out_matrix_stride ? d->out_matrix_stride : out;
    return s->in_matrix >= in && s->out_matrix >= out && product(s->matrices, s->in_matrix, SIZE_MAX / 64, &all) &&
           product(s->matrices, s->out_matrix, SIZE_MAX / 64, &all) &&
           product(s->matrices, ((s->rows + 31) / 32) * ((s->columns + 127) / 128), 0x7fffffffu, &all);
}
size_t line_of(size_t width) { return align_up(width, 8); }
size_t pair_bytes(size_t matrices, size_t rows, size_t width) { return align_up(matrices * rows * line_of(width) * 4, 256); }
size_t sums_bytes(size_t matrices) { return align_up(matrices * kMostParts * sizeof(double), 256); }

Pair take_pair(unsigned char **scratch, size_t matrices, size_t rows, size_t width) {
    const Pair p{reinterpret_cast<__half *>(*scratch), line_of(width), rows * line_of(width), matrices * rows * line_of(width)};
    *scratch += pair_bytes(matrices, rows, width);
    return p;
}
Matrices matrices_of(const Pair &p, size_t matrices, size_t rows, size_t width) {
    return Matrices{p.at, width, rows, matrices * 2, p.line, p.matrix, 2};
}

/* A symmetric product of one tile of rows has nothing across its diagonal to leave out. */
bool half_needed(size_t small) { return small > static_cast<size_t>(tb_tensor::kRows); }

tb_tensor::Fit plan_fit(int matrices, size_t height, size_t width, size_t depth, bool square, bool outer) {
    const auto tiles = [&](int columns, int m) {
        Plan plan{matrices, static_cast<int>(width), static_cast<int>(height), 0, m, columns, square && half_needed(height)};
        plan.count();
        return static_cast<size_t>(matrices) * plan.per;
    };
    return tb_tensor::best_fit(2, outer ? 64 : 32, height, (depth + 63) / 64, true, tiles, tiles);
}

tb_tensor::Fit square_fit(const OrthogonalShape &s, bool first) {
    return plan_fit(static_cast<int>(s.matrices), s.small, s.small, !first ? s.small : s.tall ? s.rows : s.columns, true, first && s.tall);
}
tb_tensor::Fit step_fit(const OrthogonalShape &s) {
    return plan_fit(static_cast<int>(s.matrices), s.rows, s.columns, s.small, false, false);
}

} /* namespace */

extern "C" size_t tb_cuda_orthogonalise_workspace(const tb_orthogonalise_desc *desc) {
    OrthogonalShape s;
    if (!orthogonal_shape(desc, &s)) return 0;
    return sums_bytes(s.matrices) + 2 * pair_bytes(s.matrices, s.rows, s.columns) + 2 * pair_bytes(s.matrices, s.small, s.small) +
           std::max({square_fit(s, true).room(), square_fit(s, false).room(), step_fit(s).room()});
}

extern "C" int tb_cuda_orthogonalise_device(const tb_orthogonalise_desc *desc, const void *g, void *out, void *workspace,
                                            void *stream) {
    OrthogonalShape s;
    int device;
    if (!orthogonal_shape(desc, &s) || !g || !out || !workspace) return 0;
    const size_t size = type_size(desc->type);
    if (!aligned(g, size) || !aligned(out, size) || !aligned(workspace, 16) || workspace == g || workspace == out ||
        (g == out && (s.in_row != s.out_row || s.in_matrix != s.out_matrix)))
        return 0;
    const int sms = multiprocessors(&device);
    Operands ops{};
    if (!sms || !(ops.status = tb_status_slot(stream))) return 0;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaGetLastError(); /* report these launches only */
    unsigned char *scratch = static_cast<unsigned char *>(workspace);
    double *sums = reinterpret_cast<double *>(scratch);
    scratch += sums_bytes(s.matrices);
    Pair x = take_pair(&scratch, s.matrices, s.rows, s.columns), next = take_pair(&scratch, s.matrices, s.rows, s.columns);
    const Pair square = take_pair(&scratch, s.matrices, s.small, s.small), poly = take_pair(&scratch, s.matrices, s.small, s.small);
    ops.type = 0;
    ops.sums = reinterpret_cast<uint32_t *>(scratch);
    ops.a_plane = ops.b_plane = static_cast<int>(s.matrices);
    return with_type(desc->type, [&](auto t) {
        using T = decltype(t);
        const int pack = pack_of(reinterpret_cast<uintptr_t>(g) | (s.in_row | s.columns | (s.matrices > 1 ? s.in_matrix : 0)) * size, size);
        size_t parts = (s.rows * s.columns + kPartValues - 1) / kPartValues;
        parts = std::min({parts, kMostParts, s.rows, std::max<size_t>(16, kManyParts / s.matrices)});
        Given given{s.rows, s.columns, s.in_matrix, s.in_row, (s.rows + parts - 1) / parts, 1};
        while (given.lanes < kNormThreads && static_cast<size_t>(given.lanes) * pack < s.columns) given.lanes *= 2;
        const dim3 grid(static_cast<unsigned>(parts), static_cast<unsigned>(s.matrices));
        const int normalised = with_pack<T>(pack, [&](auto p) {
            constexpr int P = decltype(p)::value;
            squares<T, P><<<grid, kNormThreads, 0, st>>>(given, static_cast<const T *>(g), sums);
            if (!launched()) return 0;
            return launch_early(normalise<T, P>, grid, kNormThreads, 0, 1, st, given, static_cast<const T *>(g),
                                static_cast<const double *>(sums), static_cast<double>(desc->epsilon), x);
        });
        if (!normalised) return 0;
        const int z = static_cast<int>(s.matrices), small = static_cast<int>(s.small);
        const int wide = static_cast<int>(s.columns), high = static_cast<int>(s.rows);
        const tb_tensor::Fit square_fits[2] = {square_fit(s, true), square_fit(s, false)}, whole_fit = step_fit(s);
        for (int step = 0; step < desc->steps; ++step) {
            const Matrices mx = matrices_of(x, s.matrices, s.rows, s.columns), mn = matrices_of(next, s.matrices, s.rows, s.columns);
            const Matrices ma = matrices_of(square, s.matrices, s.small, s.small), mp = matrices_of(poly, s.matrices, s.small, s.small);
            for (const bool first : {true, false}) {
                const tb_tensor::Fit &fit = square_fits[first ? 0 : 1];
                const int squared = tb_tensor::with_fit<2>(fit, [&](auto n, auto pair) {
                    constexpr int NT = decltype(n)::value;
                    constexpr bool PAIR = decltype(pair)::value;
                    SquareJob job{};
                    job.plan = Plan{z, small, small, !first ? small : s.tall ? high : wide, tb_tensor::Shape<NT, 2, PAIR>::kTileM, NT, half_needed(s.small)};
                    job.plan.count();
                    job.to = first ? square : poly;
                    job.from = square;
                    job.second = !first;
                    job.b = desc->b;
                    job.c = desc->c;
                    ops.parts = fit.parts;
                    const Matrices &from = first ? mx : ma;
                    return tb_tensor::encode<NT, PAIR>(&ops, from, first && s.tall, from, first && s.tall) &&
                                   tb_tensor::encode(&job.out, first ? ma : mp, 32, 32) && tb_tensor::encode(&job.old, ma, 32, 32) &&
                                   tb_tensor::launch_products<NT, 2, false, PAIR>(ops, job, fit.tiles, sms, st)
                               ? 1 : 0;
                });
                if (!squared) return 0;
            }
            const tb_tensor::Fit &fit = whole_fit;
            ops.parts = fit.parts;
            const int stepped = tb_tensor::with_fit<2>(fit, [&](auto n, auto pair) {
                constexpr int NT = decltype(n)::value;
                constexpr bool PAIR = decltype(pair)::value;
                StepJob<T> job{};
                job.plan = Plan{z, wide, high, small, tb_tensor::Shape<NT, 2, PAIR>::kTileM, NT, false};
                job.plan.count();
                job.to = next;
                job.from = x;
                job.last = step + 1 == desc->steps ? static_cast<T *>(out) : nullptr;
                job.row_stride = s.out_row;
                job.matrix_stride = s.out_matrix;
                job.a = desc->a;
                job.scale = desc->scale;
                /* x S: A is S (its own transpose), B is x; S x: A is x with its columns as m, B is S */
                return (s.tall ? tb_tensor::encode<NT, PAIR>(&ops, mp, false, mx, false)
                               : tb_tensor::encode<NT, PAIR>(&ops, mx, true, mp, false)) &&
                               tb_tensor::encode(&job.x, mx, 32, 32) && tb_tensor::encode(&job.next, mn, 32, 32) &&
                               tb_tensor::launch_products<NT, 2, false, PAIR>(ops, job, fit.tiles, sms, st)
                           ? 1 : 0;
            });
            if (!stepped) return 0;
            const Pair swap = x;
            x = next;
            next = swap;
        }
        return 1;
    });
}
