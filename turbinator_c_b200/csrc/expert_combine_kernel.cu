/*
 * The experts' rows back to their tokens: weighted sum and its gradient
 * (include/turbinator/training/cuda_learner.h).
 *
 * Bound: HBM; every named row is read once and every token's row read or
 * written once.  Rows move in packs of 16 bytes; the slots of a token are few
 * and known from one load, so the loads of all its rows are under way together.
 * The forward pass gives a team of up to 32 lanes a token and 32 packs of its
 * width; the backward pass gives a token one to eight warps, whose parts of
 * <dout, row> meet in shared memory, in order.  Backward of 16,384 tokens x 8
 * slots x 1,024 bf16: 113 us, 5.1 TB/s; 129 with a whole warp summing each slot.
 */
#include "tb_learner.cuh"

using namespace tb_learn;

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kAhead = 4; /* rows of a token under way at once; backward two: 132 us for 112, eight: 143 */

struct CombineShape {
    size_t tokens, rows, width, rows_stride, out_stride;
    int top_k;
};

/* lanes: of a team, a power of two; chunks: of lanes packs each, of a row. */
template <class T, int PACK>
__global__ void __launch_bounds__(kThreads)
combine_forward(CombineShape d, int lanes, int chunks, const T *rows, const int32_t *position, const float *weights, T *out) {
    using V = typename Values<PACK>::V;
    constexpr int N = Values<PACK>::kCount;
    const size_t team = (static_cast<size_t>(blockIdx.x) * kThreads + threadIdx.x) / lanes;
    const int lane = threadIdx.x % lanes;
    const size_t t = team / chunks, c = ((team - t * chunks) * lanes + lane) * PACK;
    const bool there = t < d.tokens;
    Array<PACK> sum;
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] = vall<V>(0.0f);
    for (int first = 0; first < d.top_k; first += lanes) { /* a slot for each lane */
        int32_t p = -1;
        float w = 1.0f;
        if (there && first + lane < d.top_k) {
            p = position[t * d.top_k + first + lane];
            if (p >= 0 && static_cast<size_t>(p) >= d.rows) p = -1;
            if (weights) w = weights[t * d.top_k + first + lane];
        }
        const int slots = min(d.top_k - first, lanes);
        for (int j = 0; j < slots; j += kAhead) {
            Held<T, PACK> v[kAhead];
            int32_t row[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                row[k] = __shfl_sync(0xffffffffu, p, min(j + k, slots - 1), lanes);
                if (j + k >= slots || c >= d.width) row[k] = -1;
                if (row[k] >= 0) v[k] = load_once<T, PACK>(rows + row[k] * d.rows_stride + c);
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const V s = vall<V>(__shfl_sync(0xffffffffu, w, min(j + k, slots - 1), lanes));
                if (row[k] < 0) continue;
                float e[PACK];
                unpack(v[k], e);
#pragma unroll
                for (int i = 0; i < N; ++i) sum[i] = vfma(s, vload<V>(e + 2 * i), sum[i]);
            }
        }
    }
    if (!there || c >= d.width) return;
    float e[PACK];
#pragma unroll
    for (int i = 0; i < N; ++i) vstore(e + 2 * i, sum[i]);
    *reinterpret_cast<Held<T, PACK> *>(out + t * d.out_stride + c) = packed<T, PACK>(e);
}

/* `warps` (1, 2, 4 or 8) take a token, every warps-th chunk of 32 packs each. */
template <class T, int PACK>
__global__ void __launch_bounds__(kThreads)
combine_backward(CombineShape d, int warps, const T *rows, const int32_t *position, const float *weights, const T *dout,
                 T *drows, float *dweights) {
    using V = typename Values<PACK>::V;
    constexpr int N = Values<PACK>::kCount;
    __shared__ float dots[kWarps][TB_ROUTE_MAX_TOP_K];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, part = warp % warps;
    const size_t t = static_cast<size_t>(blockIdx.x) * (kWarps / warps) + warp / warps;
    int32_t p = -1;
    float w = 1.0f;
    if (t < d.tokens && lane < d.top_k) {
        p = position[t * d.top_k + lane];
        if (p >= 0 && static_cast<size_t>(p) >= d.rows) p = -1;
        if (weights) w = weights[t * d.top_k + lane];
    }
    dots[warp][lane] = 0.0f;
    __syncwarp();
    if (t < d.tokens)
        for (size_t base = static_cast<size_t>(part) * 32 * PACK; base < d.width; base += static_cast<size_t>(warps) * 32 * PACK) {
            const size_t c = base + lane * PACK;
            const bool in = c < d.width;
            Array<PACK> g;
            {
                float e[PACK];
                Held<T, PACK> v{};
                if (in) v = *reinterpret_cast<const Held<T, PACK> *>(dout + t * d.out_stride + c);
                unpack(v, e);
#pragma unroll
                for (int i = 0; i < N; ++i) g[i] = vload<V>(e + 2 * i);
            }
            for (int j = 0; j < d.top_k; j += kAhead) {
                Held<T, PACK> v[kAhead];
                int32_t row[kAhead];
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    row[k] = __shfl_sync(0xffffffffu, p, min(j + k, d.top_k - 1));
                    if (j + k >= d.top_k || !in) row[k] = -1;
                    if (row[k] >= 0 && dweights)
                        v[k] = load_once<T, PACK>(rows + row[k] * d.rows_stride + c);
                }
                float dot[kAhead];
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    const V s = vall<V>(__shfl_sync(0xffffffffu, w, min(j + k, d.top_k - 1)));
                    dot[k] = 0.0f;
                    if (row[k] >= 0) {
                        float e[PACK];
#pragma unroll
                        for (int i = 0; i < N; ++i) vstore(e + 2 * i, vmul(s, g[i]));
                        store_once<T, PACK>(drows + row[k] * d.rows_stride + c, packed<T, PACK>(e));
                        if (dweights) {
                            unpack(v[k], e);
                            V sum = vall<V>(0.0f);
#pragma unroll
                            for (int i = 0; i < N; ++i) sum = vfma(g[i], vload<V>(e + 2 * i), sum);
                            float both[2] = {0.0f, 0.0f};
                            vstore(both, sum);
                            dot[k] = both[0] + both[1];
                        }
                    }
                }
                if (dweights) { /* each half of the warp sums half of the slots, and so on, down to eight lanes a slot */
                    int spread = 16;
#pragma unroll
                    for (int n = kAhead / 2; n; n /= 2, spread /= 2) {
                        const bool high = lane & spread;
#pragma unroll
                        for (int k = 0; k < n; ++k) {
                            const float mine = high ? dot[k + n] : dot[k];
                            dot[k] = mine + __shfl_xor_sync(0xffffffffu, high ? dot[k] : dot[k + n], spread);
                        }
                    }
                    for (; spread; spread /= 2) dot[0] += __shfl_xor_sync(0xffffffffu, dot[0], spread);
                    const int slot = j + lane / (32 / kAhead);
                    if (lane % (32 / kAhead) == 0 && slot < d.top_k) dots[warp][slot] += dot[0];
                }
            }
        }
    if (!dweights) return;
    __syncthreads();
    if (t < d.tokens && part == 0 && lane < d.top_k) {
        float sum = 0.0f;
        for (int i = 0; i < warps; ++i) sum += dots[warp + i][lane];
        dweights[t * d.top_k + lane] = sum;
    }
}

bool combine_shape(const tb_expert_combine_desc *d, CombineShape *s) {
    if (!d || !d->tokens || !d->rows || !d->width || d->top_k < 1 || d->top_k > TB_ROUTE_MAX_TOP_K ||
        !type_known(d->type) || d->rows > 0x7fffffffu)
        return false;
    size_t slots, all;
    if (!product(d->tokens, d->top_k, 0x7fffffffu, &slots)) return false;
    s->tokens = d->tokens;
    s->rows = d->rows;
    s->width = d->width;
    s->rows_stride = d->rows_stride ? d->rows_stride : d->width;
    s->out_stride = d->out_stride ? d->out_stride : d->width;
    s->top_k = d->top_k;
    return s->rows_stride >= d->width && s->out_stride >= d->width &&
           product(d->rows, s->rows_stride, SIZE_MAX / 64, &all) && product(d->tokens, s->out_stride, SIZE_MAX / 64, &all);
}

/* Calls f with the widest pack that every row of the tensors allows, as a
 * constant; 8 bytes too, for the widths that are no multiple of 16 (30,783
 * tokens x 9 slots x 124 bf16: 21 us, in packs of 4 bytes 34). */
template <class T, class F>
int with_row_pack(const CombineShape &s, const void *a, const void *b, const void *c, F &&f) {
    const size_t bits = reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c) |
                        (s.rows_stride | s.out_stride | s.width) * sizeof(T);
    if (bits % 16 == 8) return f(std::integral_constant<int, 8 / static_cast<int>(sizeof(T))>{});
    return with_pack<T>(pack_of(bits, sizeof(T)), f);
}

} /* namespace */

extern "C" int tb_cuda_combine_experts_device(const tb_expert_combine_desc *desc, const void *rows,
                                              const int32_t *position, const float *weights, void *out,
                                              void *stream) {
    CombineShape s;
    if (!combine_shape(desc, &s) || !rows || !position || !out) return 0;
    const size_t size = type_size(desc->type);
    if (!aligned(rows, size) || !aligned(out, size) || !aligned(position, 4) || !aligned(weights, 4) ||
        collide({out}, {rows, position, weights}))
        return 0;
    cudaGetLastError(); /* report this launch only */
    return with_type(desc->type, [&](auto t) {
        using T = decltype(t);
        return with_row_pack<T>(s, rows, out, nullptr, [&](auto p) {
            constexpr int P = decltype(p)::value;
            const size_t packs = (s.width + P - 1) / P;
            int lanes = 1;
            while (lanes < 32 && static_cast<size_t>(lanes) < packs) lanes *= 2;
            /* narrower teams where they idle less: 30,000 tokens x 4 x 320 bf16
             * 23 us for 29, 29,875 x 3 x 35 f32 13.7 for 17.3 */
            const auto places = [&](size_t n) { return (packs + n - 1) / n * n; };
            while (lanes > 8 && places(lanes / 2) * 5 <= places(lanes) * 4) lanes /= 2;
            const size_t chunks = (packs + lanes - 1) / lanes;
            size_t teams;
            if (!product(s.tokens, chunks, 0x7fffffffull * (kThreads / lanes) , &teams) || chunks > 0x7fffffffu) return 0;
            combine_forward<T, P><<<static_cast<unsigned>((teams * lanes + kThreads - 1) / kThreads), kThreads, 0,
                                    static_cast<cudaStream_t>(stream)>>>(
                s, lanes, static_cast<int>(chunks), static_cast<const T *>(rows), position, weights, static_cast<T *>(out));
            return launched();
        });
    });
}

extern "C" int tb_cuda_combine_experts_backward_device(const tb_expert_combine_desc *desc, const void *rows,
                                                       const int32_t *position, const float *weights,
                                                       const void *dout, void *drows, float *dweights,
                                                       void *stream) {
    CombineShape s;
    if (!combine_shape(desc, &s) || (!rows && dweights) || !position || !dout || !drows) return 0;
    const size_t size = type_size(desc->type);
    if (!aligned(rows, size) || !aligned(dout, size) || !aligned(drows, size) || !aligned(position, 4) ||
        !aligned(weights, 4) || !aligned(dweights, 4) ||
        collide({drows, dweights}, {rows, position, weights, dout}))
        return 0;
    cudaGetLastError(); /* report this launch only */
    return with_type(desc->type, [&](auto t) {
        using T = decltype(t);
        return with_row_pack<T>(s, rows, dout, drows, [&](auto p) {
            constexpr int P = decltype(p)::value;
            int warps = 1;
            while (warps < kWarps && static_cast<size_t>(warps) * 32 * P < s.width) warps *= 2;
            const size_t per = kWarps / warps;
            combine_backward<T, P><<<static_cast<unsigned>((s.tokens + per - 1) / per), kThreads, 0,
                                     static_cast<cudaStream_t>(stream)>>>(
                s, warps, static_cast<const T *>(rows), position, weights, static_cast<const T *>(dout),
                static_cast<T *>(drows), dweights);
            return launched();
        });
    });
}
