/*
 * The experts' products, forward and both gradients, and the same in 8-bit
 * integers (include/turbinator/training/cuda_learner.h).
 *
 * y[p] = x[p] W_e and dx[p] = dy[p] W_e^T are one job: rows of one expert (up
 * to 256, taken as they come: the tensor cores issue as many columns) against
 * 128 of the output's channels; tiles of one set of rows follow each other, so
 * the rows stay in L2 and so do the expert's weights.  Where an expert's rows
 * start is read on the device.  dW_e = sum_p x[p]^T dy[p] sums over a run of
 * rows that ends anywhere: what the last 16 of a run reads of the next
 * expert's rows is cleared in shared memory.  The contiguous dimension of
 * every output lies in the tensor core's rows (tb_tensor.cuh).
 *
 * f32 tensors are laid out as three bf16 planes that sum to them exactly (8
 * bits each, held higher and higher) and multiplied as six pairs, small ones
 * first; what is left out is below 2^-24 of the factors.  Rows that do not start on 16 bytes are laid
 * out anew too, in the workspace.
 */
#include <algorithm>

#include "tb_tensor.cuh"

using namespace tb_learn;
using tb_tensor::Matrices;
using tb_tensor::Operands;
using tb_tensor::Tile;

namespace {

constexpr int kMaxExperts = TB_ROUTE_MAX_EXPERTS;

struct Runs { /* of rows, one for each expert */
    const int32_t *offsets; /* NULL: one expert, all rows */
    int experts, rows;
};
/* Expert e's rows: offsets taken into [0, rows], a run that would end before its start is empty. */
__device__ __forceinline__ int run_start(const Runs &r, int e) {
    return r.offsets ? min(max(r.offsets[e], 0), r.rows) : 0;
}
__device__ __forceinline__ int run_end(const Runs &r, int e, int start) {
    return r.offsets ? max(min(max(r.offsets[e + 1], 0), r.rows), start) : r.rows;
}

template <class T> __device__ __forceinline__ T stored(uint32_t r) { return from_float<T>(__uint_as_float(r)); }

/* ---- O[p, m] = sum_k X[p, k] W_e[m, k] ---- */

template <class T, int NT> struct RowJob {
    static constexpr bool kRagged = false;
    static constexpr int kStaging = 0;
    struct Shared {
        int first[kMaxExperts + 1]; /* tile of rows that each expert's start with */
        int start[kMaxExperts], end[kMaxExperts];
    };
    Runs runs;
    int width, depth, tile_m, tiles_m;
    T *out;
    size_t out_stride;

    __device__ void setup(Shared &s) const {
        for (int e = threadIdx.x; e < runs.experts; e += blockDim.x) {
            s.start[e] = run_start(runs, e);
            s.end[e] = run_end(runs, e, s.start[e]);
        }
        __syncthreads();
        if (threadIdx.x < 32) {
            int before = 0, past = 0; /* tiles and rows of the experts so far: a run begins behind all others, */
            for (int base = 0; base < runs.experts; base += 32) { /* so that there are no more tiles than room for their sums */
                const int e = base + threadIdx.x;
                int start = max(e < runs.experts ? s.start[e] : 0, past);
#pragma unroll
                for (int o = 1; o < 32; o *= 2) start = max(start, __shfl_up_sync(0xffffffffu, start, o));
                const int end = max(e < runs.experts ? s.end[e] : 0, start);
                int n = (end - start + NT - 1) / NT;
#pragma unroll
                for (int o = 1; o < 32; o *= 2) {
                    const int v = __shfl_up_sync(0xffffffffu, n, o);
                    if (threadIdx.x >= o) n += v;
                }
                if (e < runs.experts) s.start[e] = start, s.end[e] = end, s.first[e + 1] = before + n;
                before += __shfl_sync(0xffffffffu, n, 31);
                past = __shfl_sync(0xffffffffu, end, 31);
            }
            if (threadIdx.x == 0) s.first[0] = 0;
        }
    }
    __device__ int tiles(const Shared &s) const { return s.first[runs.experts] * tiles_m; }
    __device__ Tile tile(const Shared &s, int t) const {
        const int of = t / tiles_m;
        int low = 0, high = runs.experts; /* first[low] <= of < first[high] */
        while (high - low > 1) {
            const int mid = (low + high) / 2;
            if (s.first[mid] <= of) low = mid;
            else high = mid;
        }
        Tile r;
        r.m0 = (t - of * tiles_m) * tile_m;
        r.n0 = s.start[low] + (of - s.first[low]) * NT;
        r.columns = min(NT, s.end[low] - r.n0);
        r.k0 = 0;
        r.depth = depth;
        r.az = low;
        r.bz = 0;
        r.which = low;
        return r;
    }
    __device__ __forceinline__ void store(const Shared &, const Tile &t, int m, int c, const uint32_t (&r)[8]) const {
        if (m >= width) return;
        T *o = out + (t.n0 + c) * out_stride + m;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < t.columns) o[i * out_stride] = stored<T>(r[i]);
    }
};

/* The same of 8-bit integers, scaled by row and channel. */
template <class T, int NT> struct IntegerJob : RowJob<T, NT> {
    const float *row_scale, *channel_scale;
    __device__ __forceinline__ void store(const typename RowJob<T, NT>::Shared &, const Tile &t, int m, int c,
                                          const uint32_t (&r)[8]) const {
        if (m >= this->width) return;
        T *o = this->out + (t.n0 + c) * this->out_stride + m;
        const float s = channel_scale[static_cast<size_t>(t.which) * this->width + m];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < t.columns)
                o[i * this->out_stride] = from_float<T>(static_cast<float>(static_cast<int>(r[i])) * (row_scale[t.n0 + c + i] * s));
    }
};

/* ---- O_e[n, m] = sum_p B[p, n] A[p, m] over expert e's rows ---- */

template <class T, int NT> struct SumJob {
    static constexpr bool kRagged = true;
    static constexpr int kStaging = 0;
    struct Shared {};
    Runs runs;
    int width, height, tile_m, tiles_m, tiles_n;
    T *out;
    size_t row_stride, matrix_stride;

    __device__ void setup(Shared &) const {}
    __device__ int tiles(const Shared &) const { return runs.experts * tiles_m * tiles_n; }
    __device__ Tile tile(const Shared &, int t) const {
        const int per = tiles_m * tiles_n, e = t / per, in = t - e * per, tn = in / tiles_m;
        Tile r;
        r.m0 = (in - tn * tiles_m) * tile_m;
        r.n0 = tn * NT;
        r.columns = min(NT, height - r.n0);
        r.k0 = run_start(runs, e);
        r.depth = run_end(runs, e, r.k0) - r.k0;
        r.az = r.bz = 0;
        r.which = e;
        return r;
    }
    __device__ __forceinline__ void store(const Shared &, const Tile &t, int m, int c, const uint32_t (&r)[8]) const {
        if (m >= width) return;
        T *o = out + t.which * matrix_stride + (t.n0 + c) * row_stride + m;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < t.columns) o[i * row_stride] = stored<T>(r[i]);
    }
};

/* ---- few rows ---- */

/* Where the rows are few, as in acting, the weights are what is read, once, and
 * a product is a warp's sum over a row of weights, against up to four rows. */
constexpr int kFewThreads = 256, kFewRows = 4;

/* The dot product of 16 bytes (or 4, or an element) of weights and a row. */
template <class T, int PACK> struct FewPack {
    using Sum = float;
    Held<T, PACK> h;
    __device__ __forceinline__ void load(const T *p) { h = *reinterpret_cast<const Held<T, PACK> *>(p); }
    __device__ __forceinline__ void load_once(const T *p) { h = tb_learn::load_once<T, PACK>(p); }
    __device__ __forceinline__ float dot(const FewPack &o, float sum) const {
        float a[PACK], b[PACK];
        unpack(h, a);
        unpack(o.h, b);
#pragma unroll
        for (int i = 0; i < PACK; ++i) sum = fmaf(a[i], b[i], sum);
        return sum;
    }
};
template <int PACK> struct FewPack<int8_t, PACK> {
    using Sum = int;
    static constexpr int kWords = PACK >= 4 ? PACK / 4 : 1;
    int w[kWords];
    __device__ __forceinline__ void load(const int8_t *p) {
        if constexpr (PACK == 16) {
            const int4 v = *reinterpret_cast<const int4 *>(p);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else if constexpr (PACK == 4) {
            w[0] = *reinterpret_cast<const int *>(p);
        } else {
            w[0] = *p;
        }
    }
    __device__ __forceinline__ void load_once(const int8_t *p) {
        if constexpr (PACK == 16) {
            const int4 v = __ldcs(reinterpret_cast<const int4 *>(p));
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else {
            load(p);
        }
    }
    __device__ __forceinline__ int dot(const FewPack &o, int sum) const {
        if constexpr (PACK == 1) return sum + w[0] * o.w[0];
#pragma unroll
        for (int i = 0; i < kWords; ++i) sum = __dp4a(w[i], o.w[i], sum);
        return sum;
    }
};

struct FewShape {
    int width, depth; /* of the output, of the sums */
    size_t x_stride, w_row, w_matrix, out_stride;
};

/* The expert whose run row is in and where that ends, -1 (and `last`) for none; by a warp. */
__device__ __forceinline__ int expert_of(const Runs &runs, int row, int last, int lane, int *end) {
    *end = last;
    for (int base = 0; base < runs.experts; base += 32) {
        const int mine = base + lane, from = mine < runs.experts ? run_start(runs, mine) : runs.rows;
        const int to = mine < runs.experts ? run_end(runs, mine, from) : from;
        const unsigned has = __ballot_sync(0xffffffffu, from <= row && row < to);
        if (has) {
            *end = __shfl_sync(0xffffffffu, to, __ffs(has) - 1);
            return base + __ffs(has) - 1;
        }
    }
    return -1;
}

/* W: of rows and weights, f32, bf16, f16 or 8 bits; T: of the output. */
template <class W, class T, int PACK>
__global__ void __launch_bounds__(kFewThreads)
few_rows(FewShape d, Runs runs, const W *x, const W *weight, T *out, const float *row_scale, const float *channel_scale) {
    using Sum = typename FewPack<W, PACK>::Sum;
    constexpr int kAhead = 8; /* packs of a row of weights under way at once */
    const int lane = threadIdx.x % 32, m = blockIdx.x * (kFewThreads / 32) + threadIdx.x / 32;
    const int last = min(static_cast<int>(blockIdx.y + 1) * kFewRows, runs.rows);
    after_earlier();
    if (m >= d.width) return;
    for (int row = blockIdx.y * kFewRows, count; row < last; row += count) {
        int e = 0, start = 0, end = last; /* the row's expert and its run */
        if (runs.experts == 1) { /* not waited for before the weights */
            start = run_start(runs, 0);
            end = run_end(runs, 0, start);
            count = last - row;
        } else {
            e = expert_of(runs, row, last, lane, &end);
            count = e < 0 ? 1 : min(end, last) - row;
            if (e < 0) continue; /* no expert's: left as it was */
        }
        const W *w = weight + e * d.w_matrix + m * d.w_row, *from = x + row * d.x_stride;
        Sum sum[kFewRows] = {};
        for (int k = lane * PACK; k < d.depth; k += 32 * PACK * kAhead) {
            FewPack<W, PACK> a[kAhead], b;
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                if (k + i * 32 * PACK < d.depth) a[i].load_once(w + k + i * 32 * PACK);
#pragma unroll
            for (int r = 0; r < kFewRows; ++r)
                if (r < count) {
#pragma unroll
                    for (int i = 0; i < kAhead; ++i)
                        if (k + i * 32 * PACK < d.depth) {
                            b.load(from + r * d.x_stride + k + i * 32 * PACK);
                            sum[r] = a[i].dot(b, sum[r]);
                        }
                }
        }
#pragma unroll
        for (int r = 0; r < kFewRows; ++r) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], o);
            if (lane == r && r < count && row + r >= start && row + r < end) {
                float v = static_cast<float>(sum[r]);
                if constexpr (std::is_same<W, int8_t>::value)
                    v *= row_scale[row + r] * channel_scale[static_cast<size_t>(e) * d.width + m];
                out[(row + r) * d.out_stride + m] = from_float<T>(v);
            }
        }
    }
}

/* The same where the weights lie the other way, [sum][channel]: a lane takes a
 * channel, a CTA's 32 warps every 32nd k, and their sums meet in shared memory.
 * For f32 alone (1 x 4,096 x 4,096: 27 us against 72 on the tensor cores where the
 * weights lie in L2, 45 where they do not; 16 bytes a lane: 61): of 16 bits the tensor cores' parts of a sum are faster (bf16
 * 9 us, this way 30). */
constexpr int kAcrossThreads = 1024, kAcrossWarps = kAcrossThreads / 32;
__global__ void __launch_bounds__(kAcrossThreads)
few_rows_across(FewShape d, Runs runs, const float *x, const float *weight, float *out) {
    __shared__ float parts[kAcrossWarps][kFewRows][32];
    constexpr int kAhead = 8; /* rows of weights under way at once */
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, m = blockIdx.x * 32 + lane;
    const int last = min(static_cast<int>(blockIdx.y + 1) * kFewRows, runs.rows);
    after_earlier();
    for (int row = blockIdx.y * kFewRows, count; row < last; row += count) {
        int end;
        const int e = expert_of(runs, row, last, lane, &end);
        count = e < 0 ? 1 : min(end, last) - row;
        if (e < 0) continue; /* no expert's: left as it was */
        const float *w = weight + e * d.w_matrix + m, *from = x + row * d.x_stride;
        float sum[kFewRows] = {};
        if (m < d.width)
            for (int k = warp; k < d.depth; k += kAcrossWarps * kAhead) {
                float a[kAhead];
#pragma unroll
                for (int i = 0; i < kAhead; ++i)
                    if (k + i * kAcrossWarps < d.depth) a[i] = __ldcs(w + (k + i * kAcrossWarps) * d.w_row);
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    if (k + i * kAcrossWarps >= d.depth) break;
#pragma unroll
                    for (int r = 0; r < kFewRows; ++r)
                        if (r < count) sum[r] = fmaf(a[i], from[r * d.x_stride + k + i * kAcrossWarps], sum[r]);
                }
            }
#pragma unroll
        for (int r = 0; r < kFewRows; ++r) parts[warp][r][lane] = sum[r];
        __syncthreads();
        if (warp < count && m < d.width) {
            float v = 0.0f;
#pragma unroll
            for (int p = 0; p < kAcrossWarps; ++p) v += parts[p][warp][lane];
            out[(row + warp) * d.out_stride + m] = v;
        }
        __syncthreads();
    }
}

/* dW where an expert has few rows: what is written is most of the work.  A warp
 * takes four lines of an expert's gradient, [line][column], lanes along them. */
constexpr int kFewLines = 4;
template <class T, int PACK>
__global__ void __launch_bounds__(kFewThreads)
few_sums(int width, int height, size_t line_stride, size_t column_stride, size_t w_row, size_t w_matrix, Runs runs, const T *lines,
         const T *columns, T *out) {
    const int lane = threadIdx.x % 32, n0 = (blockIdx.x * (kFewThreads / 32) + threadIdx.x / 32) * kFewLines, e = blockIdx.y;
    after_earlier();
    if (n0 >= height) return;
    const int start = run_start(runs, e), end = run_end(runs, e, start);
    for (int m = lane * PACK; m < width; m += 32 * PACK) {
        float sum[kFewLines][PACK] = {};
        for (int p = start; p < end; ++p) {
            float b[PACK];
            unpack(*reinterpret_cast<const Held<T, PACK> *>(columns + p * column_stride + m), b);
#pragma unroll
            for (int i = 0; i < kFewLines; ++i)
                if (n0 + i < height) {
                    const float a = to_float(lines[p * line_stride + n0 + i]);
#pragma unroll
                    for (int j = 0; j < PACK; ++j) sum[i][j] = fmaf(a, b[j], sum[i][j]);
                }
        }
#pragma unroll
        for (int i = 0; i < kFewLines; ++i)
            if (n0 + i < height) store_once<T, PACK>(out + e * w_matrix + (n0 + i) * w_row + m, packed<T, PACK>(sum[i]));
    }
}

/* Up to eight rows, and some 2^25 products of theirs: 1 x 4,096 x 4,096 of 8 bits
 * 6.2 us against 7.7 by tiles, of bf16 6.7 against 9.1, 8 x 1,024 x 1,024 4.0
 * against 4.8; 8 x 8,192 x 8,192 47 against 12.  f32 weights are laid out as planes
 * for the tensor cores, 16 bytes moved for each of 4: rows up to a dozen an expert
 * (8 x 4,096 x 4,096: 32 us against 72), up to four where the weights' rows lie
 * across the sum (4 x 4,096 x 4,096: 30 against 72, 8: 57). */
bool few(size_t rows, size_t experts, size_t in, size_t out, bool wide, bool across) {
    if (in > 1u << 30 || out > 1u << 30) return false; /* 32-bit places, some packs ahead */
    if (wide) return rows <= (across ? 4 : 12) * experts;
    return !across && rows <= 8 && static_cast<double>(rows) * in * out <= 33554432.0;
}

template <class W, class T>
int few_product(const FewShape &d, const Runs &runs, const W *x, const W *weight, T *out, const float *row_scale,
                const float *channel_scale, cudaStream_t st) {
    const size_t bits = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(weight) |
                        (d.x_stride | d.w_row | d.w_matrix | static_cast<size_t>(d.depth)) * sizeof(W);
    const dim3 grid(static_cast<unsigned>((d.width + kFewThreads / 32 - 1) / (kFewThreads / 32)),
                    static_cast<unsigned>((runs.rows + kFewRows - 1) / kFewRows));
    const auto launch = [&](auto p) {
        return launch_early(few_rows<W, T, decltype(p)::value>, grid, kFewThreads, 0, 1, st, d, runs, x, weight, out, row_scale, channel_scale);
    };
    if (bits % 16 == 0) return launch(std::integral_constant<int, 16 / static_cast<int>(sizeof(W))>{});
    if constexpr (sizeof(W) < 4)
        if (bits % 4 == 0) return launch(std::integral_constant<int, 4 / static_cast<int>(sizeof(W))>{});
    return launch(std::integral_constant<int, 1>{});
}

inline int few_product_across(const FewShape &d, const Runs &runs, const float *x, const float *weight, float *out, cudaStream_t st) {
    const dim3 grid(static_cast<unsigned>((d.width + 31) / 32), static_cast<unsigned>((runs.rows + kFewRows - 1) / kFewRows));
    return launch_early(few_rows_across, grid, kAcrossThreads, 0, 1, st, d, runs, x, weight, out);
}

/* Rows of lines and columns; out [experts][height][width]. */
template <class T>
int few_gradient(int width, int height, size_t line_stride, size_t column_stride, size_t w_row, size_t w_matrix, const Runs &runs,
                 const T *lines, const T *columns, T *out, cudaStream_t st) {
    const size_t bits = reinterpret_cast<uintptr_t>(columns) | reinterpret_cast<uintptr_t>(out) |
                        (column_stride | w_row | w_matrix | static_cast<size_t>(width)) * sizeof(T);
    return with_pack<T>(pack_of(bits, sizeof(T)), [&](auto p) {
        constexpr int P = decltype(p)::value, kLines = kFewThreads / 32 * kFewLines;
        const dim3 grid(static_cast<unsigned>((height + kLines - 1) / kLines), static_cast<unsigned>(runs.experts));
        return launch_early(few_sums<T, P>, grid, kFewThreads, 0, 1, st, width, height, line_stride, column_stride, w_row, w_matrix, runs, lines,
                            columns, out);
    });
}

/* ---- laying operands out ---- */

struct Layout {
    size_t width, rows, count, row_stride, matrix_stride; /* of the source */
    size_t line;                                          /* of the copy: a multiple of 16 bytes */
    const void *from;
    void *to;
    const int32_t *first, *last; /* of the rows that are any expert's, or NULL: all */
};
constexpr int kMostLayouts = 3;
struct Layouts {
    Layout of[kMostLayouts];
    int count;
};

/* A value's planes: three bf16 that sum to it, the second held 2^7 and the third
 * 2^14 higher (the first alone where it is no finite number).  So f32's smallest
 * normal numbers keep 22 bits; at one scale the third plane of what is below
 * 2^-112 fell under bf16's least values, an error of 1.5e-5 at 2^-118. */
__device__ __forceinline__ void planes_of(float v, __nv_bfloat16 (&p)[3]) {
    p[0] = __float2bfloat16_rn(v);
    if (__hisinf(p[0]) && isfinite(v)) p[0] = __float2bfloat16_rz(v); /* rounded past the largest */
    constexpr float kUp = 1 << tb_tensor::kPlaneRise<3>;
    const float rest = isfinite(v) ? (v - __bfloat162float(p[0])) * kUp : 0.0f;
    p[1] = __float2bfloat16_rn(rest);
    p[2] = __float2bfloat16_rn((rest - __bfloat162float(p[1])) * kUp);
}

constexpr int kLayThreads = 256;
/* N neighbours of a line. */
template <class T, int N> __device__ __forceinline__ void lay_some(const Layout &d, const T (&v)[N], size_t at, size_t plane) {
    if constexpr (sizeof(T) == 4) {
        Pack<__nv_bfloat16, N> part[3];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            __nv_bfloat16 p[3];
            planes_of(v[i], p);
#pragma unroll
            for (int j = 0; j < 3; ++j) part[j].v[i] = p[j];
        }
#pragma unroll
        for (int j = 0; j < 3; ++j) *reinterpret_cast<Pack<__nv_bfloat16, N> *>(static_cast<__nv_bfloat16 *>(d.to) + at + j * plane) = part[j];
    } else {
        Pack<T, N> part;
#pragma unroll
        for (int i = 0; i < N; ++i) part.v[i] = v[i];
        *reinterpret_cast<Pack<T, N> *>(static_cast<T *>(d.to) + at) = part;
    }
}
/* A warp a line at a time, two neighbours a lane, or four where an f32 line
 * lies on 16 bytes; blockIdx.y: of the tensors. */
template <class T>
__global__ void __launch_bounds__(kLayThreads) lay_out(const __grid_constant__ Layouts all) {
    const Layout &d = all.of[blockIdx.y];
    const size_t lines = d.rows * d.count, plane = lines * d.line;
    const int lane = threadIdx.x % 32;
    const size_t begin = d.first ? static_cast<size_t>(max(*d.first, 0)) : 0;
    const size_t end = d.last ? min(static_cast<size_t>(max(*d.last, 0)), lines) : lines;
    for (size_t i = begin + static_cast<size_t>(blockIdx.x) * (kLayThreads / 32) + threadIdx.x / 32; i < end;
         i += static_cast<size_t>(gridDim.x) * (kLayThreads / 32)) {
        const size_t z = d.count > 1 ? i / d.rows : 0, r = i - z * d.rows;
        const T *from = static_cast<const T *>(d.from) + z * d.matrix_stride + r * d.row_stride;
        if (sizeof(T) == 4 && d.width % 4 == 0 && (reinterpret_cast<uintptr_t>(from) & 15) == 0) {
            for (size_t c = lane * 4; c < d.line; c += 128) { /* a line's length is a multiple of eight */
                T v[4] = {};
                if (c < d.width) {
                    const Pack<T, 4> p = *reinterpret_cast<const Pack<T, 4> *>(from + c);
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] = p.v[j];
                }
                lay_some(d, v, i * d.line + c, plane);
            }
        } else {
            for (size_t c = lane * 2; c < d.line; c += 64) {
                T v[2] = {};
                if (c < d.width) v[0] = from[c];
                if (c + 1 < d.width) v[1] = from[c + 1];
                lay_some(d, v, i * d.line + c, plane);
            }
        }
    }
}

/* A tensor of a call, and where it lies for the tensor cores. */
struct Source {
    const void *at;
    size_t width, rows, count, row_stride, matrix_stride;
    const int32_t *first = nullptr, *last = nullptr; /* of its rows that are any expert's */
};
/* Elements of a laid-out line, and bytes of the whole. */
size_t line_of(size_t width, size_t size) { return align_up(width, 16 / size); }
size_t laid_bytes(size_t width, size_t rows, size_t count, bool wide, size_t size) {
    return align_up(line_of(width, size) * rows * count * (wide ? 3 : 1) * size, 256);
}

/* Notes a tensor to be laid out, if it has to be. */
template <class T> void lay(const Source &s, size_t size, unsigned char **scratch, Layouts *all, Matrices *m) {
    const bool wide = sizeof(T) == 4;
    *m = Matrices{s.at, s.width, s.rows, s.count, s.row_stride, s.matrix_stride, size};
    if (!wide && m->straight()) return;
    const size_t line = line_of(s.width, size);
    all->of[all->count++] = Layout{s.width, s.rows, s.count, s.row_stride, s.matrix_stride, line, s.at, *scratch, s.first, s.last};
    *m = Matrices{*scratch, s.width, s.rows, s.count * (wide ? 3 : 1), line, line * s.rows, size};
    *scratch += laid_bytes(s.width, s.rows, s.count, wide, size);
}
/* Lays out what has been noted, in one launch. */
template <class T> int laid(const Layouts &all, int sms, cudaStream_t st) {
    size_t most = 0;
    for (int i = 0; i < all.count; ++i) most = std::max(most, all.of[i].rows * all.of[i].count);
    if (!most) return 1;
    const size_t blocks = std::min((most + kLayThreads / 32 - 1) / (kLayThreads / 32), static_cast<size_t>(sms) * 8);
    lay_out<T><<<dim3(static_cast<unsigned>(blocks), all.count), kLayThreads, 0, st>>>(all);
    return launched();
}

/* ---- shapes ---- */

struct ProductShape {
    size_t rows, experts, in, out, x_stride, dx_stride, y_stride, w_row, w_matrix;
    bool turned; /* weights [out, in] */
    size_t size;
    bool wide;
};

bool product_shape(const tb_expert_product_desc *d, ProductShape *s) {
    if (!d || !d->rows || !d->experts || !d->in_width || !d->out_width || !type_known(d->type) ||
        d->experts > kMaxExperts || d->rows > 0x7fffff00u || d->in_width > 0x7fffff00u || d->out_width > 0x7fffff00u ||
        (d->weight_order != TB_WEIGHT_IN_OUT && d->weight_order != TB_WEIGHT_OUT_IN))
        return false;
    s->rows = d->rows;
    s->experts = d->experts;
    s->in = d->in_width;
    s->out = d->out_width;
    s->turned = d->weight_order == TB_WEIGHT_OUT_IN;
    s->x_stride = d->in_stride ? d->in_stride : s->in;
    s->dx_stride = d->din_stride ? d->din_stride : s->in;
    s->y_stride = d->out_stride ? d->out_stride : s->out;
    const size_t w_width = s->turned ? s->in : s->out, w_rows = s->turned ? s->out : s->in;
    s->w_row = d->weight_row_stride ? d->weight_row_stride : w_width;
    size_t all;
    if (s->w_row < w_width || !product(w_rows, s->w_row, SIZE_MAX / 64, &all)) return false;
    s->w_matrix = d->weight_expert_stride ? d->weight_expert_stride : all;
    s->wide = d->type == TB_TYPE_F32;
    s->size = type_size(d->type);
    return s->x_stride >= s->in && s->dx_stride >= s->in && s->y_stride >= s->out && s->w_matrix >= all &&
           product(s->rows, s->x_stride, SIZE_MAX / 64, &all) && product(s->rows, s->dx_stride, SIZE_MAX / 64, &all) &&
           product(s->rows, s->y_stride, SIZE_MAX / 64, &all) && product(s->experts, s->w_matrix, SIZE_MAX / 64, &all) &&
           product(s->experts * ((s->in + 63) / 64), (s->out + 63) / 64, 0x7fffffffu, &all) &&
           product((s->out + 127) / 128, s->rows / 32 + s->experts, 0x7fffffffu, &all) &&
           product((s->in + 127) / 128, s->rows / 32 + s->experts, 0x7fffffffu, &all);
}
Source rows_of(const void *at, size_t width, size_t rows, size_t stride, const int32_t *offsets, size_t experts) {
    return {at, width, rows, 1, stride, 0, offsets, offsets ? offsets + experts : nullptr};
}
Source x_of(const ProductShape &s, const void *x, const int32_t *offsets) { return rows_of(x, s.in, s.rows, s.x_stride, offsets, s.experts); }
Source y_of(const ProductShape &s, const void *y, const int32_t *offsets) { return rows_of(y, s.out, s.rows, s.y_stride, offsets, s.experts); }
Source w_of(const ProductShape &s, const void *w) {
    return {w, s.turned ? s.in : s.out, s.turned ? s.out : s.in, s.experts, s.w_row, s.w_matrix};
}
size_t laid_room(const Source &s, bool wide) { return laid_bytes(s.width, s.rows, s.count, wide, 2); }

int kind_of(int type) { return type == TB_TYPE_F16 ? 0 : 1; }
int tiles_of(size_t width, int tile) { return static_cast<int>((width + tile - 1) / tile); }

/* Tiles of rows: an expert's last is half full on average. */
tb_tensor::Fit rows_fit(int planes, size_t rows, size_t experts, size_t width, size_t blocks) {
    const size_t average = (rows + experts - 1) / experts;
    return tb_tensor::best_fit(
        planes, 32, average, blocks, true,
        [&](int columns, int m) {
            const size_t of_rows = experts > 1 && average > static_cast<size_t>(columns) ? rows / columns + experts / 2
                                                                                         : (average + columns - 1) / columns * experts;
            return of_rows * tiles_of(width, m);
        },
        [&](int columns, int m) { return (rows / columns + experts) * tiles_of(width, m); });
}
tb_tensor::Fit sums_fit(int planes, size_t rows, size_t experts, size_t width, size_t height) {
    const auto tiles = [&](int columns, int m) { return experts * tiles_of(width, m) * tiles_of(height, columns); };
    return tb_tensor::best_fit(planes, 64, height, ((rows + experts - 1) / experts + 63) / 64, true, tiles, tiles);
}

/* O [rows, width] of type T, from operands laid out. */
template <class T>
int rows_product(Operands ops, const Matrices &w, bool w_outer, const Matrices &x, const Runs &runs, size_t width,
                 size_t depth, void *out, size_t out_stride, void *sums, int sms, cudaStream_t st) {
    constexpr int PLANES = sizeof(T) == 4 ? 3 : 1;
    const tb_tensor::Fit fit = rows_fit(PLANES, runs.rows, runs.experts, width, (depth + 63) / 64);
    ops.parts = fit.parts;
    ops.sums = static_cast<uint32_t *>(sums);
    return tb_tensor::with_fit<PLANES>(fit, [&](auto n, auto pair) {
        constexpr int NT = decltype(n)::value;
        constexpr bool PAIR = decltype(pair)::value;
        constexpr int TM = tb_tensor::Shape<NT, PLANES, PAIR>::kTileM;
        if (!tb_tensor::encode<NT, PAIR>(&ops, w, w_outer, x, false)) return 0;
        ops.a_plane = runs.experts;
        ops.b_plane = 1;
        const RowJob<T, NT> job{runs, static_cast<int>(width), static_cast<int>(depth), TM, tiles_of(width, TM), static_cast<T *>(out), out_stride};
        return tb_tensor::launch_products<NT, PLANES, false, PAIR>(ops, job, fit.tiles, sms, st);
    });
}

} /* namespace */

extern "C" size_t tb_cuda_experts_product_workspace(const tb_expert_product_desc *desc) {
    ProductShape s;
    if (!product_shape(desc, &s)) return 0;
    const int planes = s.wide ? 3 : 1;
    const size_t sums = std::max({rows_fit(planes, s.rows, s.experts, s.out, (s.in + 63) / 64).room(),
                                  rows_fit(planes, s.rows, s.experts, s.in, (s.out + 63) / 64).room(),
                                  sums_fit(planes, s.rows, s.experts, s.turned ? s.in : s.out, s.turned ? s.out : s.in).room()});
    return laid_room(x_of(s, nullptr, nullptr), s.wide) + laid_room(y_of(s, nullptr, nullptr), s.wide) + laid_room(w_of(s, nullptr), s.wide) + sums;
}

extern "C" int tb_cuda_experts_product_device(const tb_expert_product_desc *desc, const void *x, const void *weight,
                                              const int32_t *offsets, void *y, void *workspace, void *stream) {
    ProductShape s;
    int device;
    if (!product_shape(desc, &s) || !x || !weight || !y || !workspace || (!offsets && s.experts > 1)) return 0;
    if (!aligned(x, s.size) || !aligned(weight, s.size) || !aligned(y, s.size) || !aligned(offsets, 4) ||
        !aligned(workspace, 16) || collide({y, workspace}, {x, weight, offsets}))
        return 0;
    const int sms = multiprocessors(&device);
    Operands ops{};
    if (!sms || !(ops.status = tb_status_slot(stream))) return 0;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaGetLastError(); /* report these launches only */
    ops.type = kind_of(desc->type);
    const Runs runs{offsets, static_cast<int>(s.experts), static_cast<int>(s.rows)};
    return with_type(desc->type, [&](auto t) -> int {
        using T = decltype(t);
        const bool by_rows = few(s.rows, s.experts, s.in, s.out, s.wide, !s.turned);
        if constexpr (sizeof(T) == 4)
            if (!s.turned && by_rows)
                return few_product_across({static_cast<int>(s.out), static_cast<int>(s.in), s.x_stride, s.w_row, s.w_matrix, s.y_stride}, runs,
                                             static_cast<const T *>(x), static_cast<const T *>(weight), static_cast<T *>(y), st);
        if (s.turned && by_rows)
            return few_product<T, T>({static_cast<int>(s.out), static_cast<int>(s.in), s.x_stride, s.w_row, s.w_matrix, s.y_stride}, runs,
                                     static_cast<const T *>(x), static_cast<const T *>(weight), static_cast<T *>(y), nullptr, nullptr, st);
        unsigned char *scratch = static_cast<unsigned char *>(workspace);
        Matrices mw, mx;
        Layouts all{};
        lay<T>(w_of(s, weight), 2, &scratch, &all, &mw);
        lay<T>(x_of(s, x, offsets), 2, &scratch, &all, &mx);
        return laid<T>(all, sms, st) &&
               rows_product<T>(ops, mw, !s.turned, mx, runs, s.out, s.in, y, s.y_stride, scratch, sms, st);
    });
}

extern "C" int tb_cuda_experts_product_backward_device(const tb_expert_product_desc *desc, const void *x,
                                                       const void *weight, const int32_t *offsets, const void *dy,
                                                       void *dx, void *dweight, void *workspace, void *stream) {
    ProductShape s;
    int device;
    if (!product_shape(desc, &s) || (!x && dweight) || (!weight && dx) || !dy || (!dx && !dweight) || !workspace ||
        (!offsets && s.experts > 1))
        return 0;
    if (!aligned(x, s.size) || !aligned(weight, s.size) || !aligned(dy, s.size) || !aligned(dx, s.size) ||
        !aligned(dweight, s.size) || !aligned(offsets, 4) || !aligned(workspace, 16) ||
        collide({dx, dweight, workspace}, {x, weight, offsets, dy}))
        return 0;
    const int sms = multiprocessors(&device);
    Operands ops{};
    if (!sms || !(ops.status = tb_status_slot(stream))) return 0;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaGetLastError(); /* report these launches only */
    ops.type = kind_of(desc->type);
    const Runs runs{offsets, static_cast<int>(s.experts), static_cast<int>(s.rows)};
    return with_type(desc->type, [&](auto t) {
        using T = decltype(t);
        const T *g = static_cast<const T *>(dy), *w = static_cast<const T *>(weight), *in = static_cast<const T *>(x);
        if (dx && few(s.rows, s.experts, s.in, s.out, s.wide, s.turned)) {
            const FewShape d{static_cast<int>(s.in), static_cast<int>(s.out), s.y_stride, s.w_row, s.w_matrix, s.dx_stride};
            int ok = 0;
            if (!s.turned) ok = few_product<T, T>(d, runs, g, w, static_cast<T *>(dx), nullptr, nullptr, st);
            if constexpr (sizeof(T) == 4)
                if (s.turned) ok = few_product_across(d, runs, g, w, static_cast<T *>(dx), st);
            if (!ok) return 0;
            dx = nullptr;
        }
        if (dweight && few(s.rows, s.experts, s.in, s.out, s.wide, false)) {
            const int width = static_cast<int>(s.turned ? s.in : s.out), height = static_cast<int>(s.turned ? s.out : s.in);
            if (!few_gradient<T>(width, height, s.turned ? s.y_stride : s.x_stride, s.turned ? s.x_stride : s.y_stride, s.w_row, s.w_matrix, runs,
                                 s.turned ? g : in, s.turned ? in : g, static_cast<T *>(dweight), st))
                return 0;
            dweight = nullptr;
        }
        if (!dx && !dweight) return 1;
        unsigned char *scratch = static_cast<unsigned char *>(workspace);
        Matrices mw, mx, my;
        Layouts all{};
        lay<T>(y_of(s, dy, offsets), 2, &scratch, &all, &my);
        if (dx) lay<T>(w_of(s, weight), 2, &scratch, &all, &mw);
        if (dweight) lay<T>(x_of(s, x, offsets), 2, &scratch, &all, &mx);
        if (!laid<T>(all, sms, st)) return 0;
        if (dx && !rows_product<T>(ops, mw, s.turned, my, runs, s.in, s.out, dx, s.dx_stride, scratch, sms, st)) return 0;
        if (!dweight) return 1;
        /* weights [in, out]: n counts in, m out; [out, in] the other way */
        const size_t width = s.turned ? s.in : s.out, height = s.turned ? s.out : s.in;
        constexpr int PLANES = sizeof(T) == 4 ? 3 : 1;
        const tb_tensor::Fit fit = sums_fit(PLANES, s.rows, s.experts, width, height);
        ops.parts = fit.parts;
        ops.sums = reinterpret_cast<uint32_t *>(scratch);
        return tb_tensor::with_fit<PLANES>(fit, [&](auto n, auto pair) {
            constexpr int NT = decltype(n)::value;
            constexpr bool PAIR = decltype(pair)::value;
            constexpr int TM = tb_tensor::Shape<NT, PLANES, PAIR>::kTileM;
            if constexpr (NT < tb_tensor::kChunk) return 0;
            if (!tb_tensor::encode<NT, PAIR>(&ops, s.turned ? mx : my, true, s.turned ? my : mx, true)) return 0;
            ops.a_plane = ops.b_plane = 1;
            const int tiles_m = tiles_of(width, TM), tiles_n = tiles_of(height, NT);
            const SumJob<T, NT> job{runs, static_cast<int>(width), static_cast<int>(height), TM, tiles_m, tiles_n,
                                    static_cast<T *>(dweight), s.w_row, s.w_matrix};
            return tb_tensor::launch_products<NT, PLANES, false, PAIR>(ops, job, fit.tiles, sms, st);
        });
    });
}

/* ---- 8-bit integers ---- */

namespace {

constexpr int kQuantThreads = 256;

/* A team of a warp or a CTA a row: its largest magnitude, then its values, up
 * to HELD packs a thread of which stay in registers.  A row whose largest magnitude
 * has no finite reciprocal times 127 counts as zero; one with an infinity or a
 * NaN gets the scale NaN. */
template <class T, int PACK, int TEAM, int HELD>
__global__ void __launch_bounds__(kQuantThreads)
quantise_rows(size_t rows, size_t width, size_t x_stride, size_t q_stride, const T *x, int8_t *q, float *scale) {
    __shared__ float most[kQuantThreads / 32];
    __shared__ int wrong[kQuantThreads / 32];
    const size_t row = static_cast<size_t>(blockIdx.x) * (kQuantThreads / TEAM) + threadIdx.x / TEAM;
    const unsigned lane = threadIdx.x % TEAM;
    later_may_start();
    if (TEAM == 32 && row >= rows) return;
    const T *from = x + row * x_stride;
    float m = 0.0f;
    bool bad = false;
    const auto look = [&](const Held<T, PACK> &h) {
        float e[PACK];
        unpack(h, e);
#pragma unroll
        for (int i = 0; i < PACK; ++i) {
            m = fmaxf(m, fabsf(e[i]));
            bad |= !(fabsf(e[i]) <= 3.402823466e38f);
        }
    };
    const size_t first = static_cast<size_t>(lane) * PACK, step = TEAM * PACK;
    Held<T, PACK> held[HELD];
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (first + i * step < width) held[i] = load_once<T, PACK>(from + first + i * step);
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (first + i * step < width) look(held[i]);
    for (size_t c = first + HELD * step; c < width; c += step) look(*reinterpret_cast<const Held<T, PACK> *>(from + c));
    m = warp_max(m);
    bad = __any_sync(0xffffffffu, bad);
    if constexpr (TEAM > 32) {
        if (threadIdx.x % 32 == 0) most[threadIdx.x / 32] = m, wrong[threadIdx.x / 32] = bad;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kQuantThreads / 32; ++i) m = fmaxf(m, most[i]), bad |= wrong[i] != 0;
    }
    float up = __fmul_rn(__frcp_rn(m), 127.0f);
    const bool none = bad || !(up <= 3.402823466e38f);
    if (none) up = 0.0f;
    const auto put = [&](size_t c, const Held<T, PACK> &h) {
        float e[PACK];
        unpack(h, e);
        Pack<int8_t, PACK> out;
#pragma unroll
        for (int i = 0; i < PACK; ++i) out.v[i] = none ? 0 : static_cast<int8_t>(__float2int_rn(e[i] * up));
        *reinterpret_cast<Pack<int8_t, PACK> *>(q + row * q_stride + c) = out;
    };
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (first + i * step < width) put(first + i * step, held[i]);
    for (size_t c = first + HELD * step; c < width; c += step) put(c, *reinterpret_cast<const Held<T, PACK> *>(from + c));
    if (lane == 0) scale[row] = bad ? __int_as_float(0x7fc00000) : none ? 0.0f : __fdiv_rn(m, 127.0f);
}
/* Rows for all warps of the GPU, each held by its warp: 16,384 x 4,096 bf16 43 us, a
 * CTA a row 50. */
constexpr size_t kQuantManyRows = 2048;

struct IntegerShape {
    size_t rows, experts, in, out, x_stride, y_stride, w_row, w_matrix;
};
bool integer_shape(const tb_expert_product_i8_desc *d, IntegerShape *s) {
    if (!d || !d->rows || !d->experts || !d->in_width || !d->out_width || !type_known(d->type) ||
        d->experts > kMaxExperts || d->rows > 0x7fffff00u || d->in_width > TB_I8_MAX_WIDTH || d->out_width > 0x7fffff00u)
        return false;
    s->rows = d->rows;
    s->experts = d->experts;
    s->in = d->in_width;
    s->out = d->out_width;
    s->x_stride = d->in_stride ? d->in_stride : s->in;
    s->y_stride = d->out_stride ? d->out_stride : s->out;
    s->w_row = d->weight_row_stride ? d->weight_row_stride : s->in;
    size_t all;
    if (s->w_row < s->in || !product(s->out, s->w_row, SIZE_MAX / 64, &all)) return false;
    s->w_matrix = d->weight_expert_stride ? d->weight_expert_stride : all;
    return s->x_stride >= s->in && s->y_stride >= s->out && s->w_matrix >= all &&
           product(s->rows, s->x_stride, SIZE_MAX / 64, &all) && product(s->rows, s->y_stride, SIZE_MAX / 64, &all) &&
           product(s->experts, s->w_matrix, SIZE_MAX / 64, &all) &&
           product((s->out + 127) / 128, s->rows / 32 + s->experts, 0x7fffffffu, &all);
}

} /* namespace */

extern "C" int tb_cuda_quantise_rows_device(const tb_quantise_desc *desc, const void *x, int8_t *q, float *scale,
                                            void *stream) {
    if (!desc || !desc->rows || !desc->width || !type_known(desc->type) || desc->rows > 0x7fffffffu || !x || !q || !scale)
        return 0;
    const size_t x_stride = desc->x_stride ? desc->x_stride : desc->width, q_stride = desc->q_stride ? desc->q_stride : desc->width;
    const size_t size = type_size(desc->type);
    size_t all;
    if (x_stride < desc->width || q_stride < desc->width || !product(desc->rows, x_stride, SIZE_MAX / 64, &all) ||
        !product(desc->rows, q_stride, SIZE_MAX / 64, &all) || !aligned(x, size) || !aligned(scale, 4) ||
        collide({q, scale}, {x}))
        return 0;
    cudaGetLastError(); /* report this launch only */
    return with_type(desc->type, [&](auto t) {
        using T = decltype(t);
        /* a pack of x and the q that it becomes both start on their own size */
        const size_t bits = reinterpret_cast<uintptr_t>(x) | (x_stride | desc->width) * size |
                            (reinterpret_cast<uintptr_t>(q) | q_stride) * size;
        return with_pack<T>(pack_of(bits, size), [&](auto p) {
            constexpr int P = decltype(p)::value;
            const cudaStream_t st = static_cast<cudaStream_t>(stream);
            constexpr int kTeams = kQuantThreads / 32;
            if (desc->rows >= kQuantManyRows && desc->width <= static_cast<size_t>(32) * P * 16)
                quantise_rows<T, P, 32, 16><<<static_cast<unsigned>((desc->rows + kTeams - 1) / kTeams), kQuantThreads, 0, st>>>(
                    desc->rows, desc->width, x_stride, q_stride, static_cast<const T *>(x), q, scale);
            else
                quantise_rows<T, P, kQuantThreads, 4><<<static_cast<unsigned>(desc->rows), kQuantThreads, 0, st>>>(
                    desc->rows, desc->width, x_stride, q_stride, static_cast<const T *>(x), q, scale);
            return launched();
        });
    });
}

extern "C" size_t tb_cuda_experts_product_i8_workspace(const tb_expert_product_i8_desc *desc) {
    IntegerShape s;
    if (!integer_shape(desc, &s)) return 0;
    return laid_bytes(s.in, s.rows, 1, false, 1) + laid_bytes(s.in, s.out, s.experts, false, 1) +
           rows_fit(1, s.rows, s.experts, s.out, (s.in + 127) / 128).room();
}

extern "C" int tb_cuda_experts_product_i8_device(const tb_expert_product_i8_desc *desc, const int8_t *q,
                                                 const float *q_scale, const int8_t *weight, const float *weight_scale,
                                                 const int32_t *offsets, void *y, void *workspace, void *stream) {
    IntegerShape s;
    int device;
    if (!integer_shape(desc, &s) || !q || !q_scale || !weight || !weight_scale || !y || !workspace || (!offsets && s.experts > 1))
        return 0;
    if (!aligned(q_scale, 4) || !aligned(weight_scale, 4) || !aligned(offsets, 4) || !aligned(y, type_size(desc->type)) ||
        !aligned(workspace, 16) || collide({y, workspace}, {q, q_scale, weight, weight_scale, offsets}))
        return 0;
    const int sms = multiprocessors(&device);
    Operands ops{};
    if (!sms || !(ops.status = tb_status_slot(stream))) return 0;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaGetLastError(); /* report these launches only */
    ops.type = 1;
    const Runs runs{offsets, static_cast<int>(s.experts), static_cast<int>(s.rows)};
    if (few(s.rows, s.experts, s.in, s.out, false, false))
        return with_type(desc->type, [&](auto t) {
            using T = decltype(t);
            return few_product<int8_t, T>({static_cast<int>(s.out), static_cast<int>(s.in), s.x_stride, s.w_row, s.w_matrix, s.y_stride}, runs,
                                          q, weight, static_cast<T *>(y), q_scale, weight_scale, st);
        });
    unsigned char *scratch = static_cast<unsigned char *>(workspace);
    Matrices mw, mx;
    Layouts all{};
    lay<int8_t>({weight, s.in, s.out, s.experts, s.w_row, s.w_matrix}, 1, &scratch, &all, &mw);
    lay<int8_t>(rows_of(q, s.in, s.rows, s.x_stride, offsets, s.experts), 1, &scratch, &all, &mx);
    if (!laid<int8_t>(all, sms, st)) return 0;
    const tb_tensor::Fit fit = rows_fit(1, s.rows, s.experts, s.out, (s.in + 127) / 128);
    ops.parts = fit.parts;
    ops.sums = reinterpret_cast<uint32_t *>(scratch);
    return with_type(desc->type, [&](auto t) {
        using T = decltype(t);
        return tb_tensor::with_fit<1>(fit, [&](auto n, auto pair) {
            constexpr int NT = decltype(n)::value;
            constexpr bool PAIR = decltype(pair)::value;
            constexpr int TM = tb_tensor::Shape<NT, 1, PAIR>::kTileM;
            if (!tb_tensor::encode<NT, PAIR>(&ops, mw, false, mx, false)) return 0;
            const int tiles_m = tiles_of(s.out, TM);
            IntegerJob<T, NT> job;
            static_cast<RowJob<T, NT> &>(job) = RowJob<T, NT>{runs, static_cast<int>(s.out), static_cast<int>(s.in), TM,
                                                              tiles_m, static_cast<T *>(y), s.y_stride};
            job.row_scale = q_scale;
            job.channel_scale = weight_scale;
            return tb_tensor::launch_products<NT, 1, true, PAIR>(ops, job, fit.tiles, sms, st);
        });
    });
}
