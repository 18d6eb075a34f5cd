/*
 * Tokens handed out to their experts, weights applied on the way, and the
 * gradient (include/turbinator/training/cuda_learner.h).
 *
 * Bound: HBM; a row of the output is written once, a token's row read from L2
 * by all but the first of its slots.  16,384 tokens x 8 slots x 1,024 bf16, a tenth
 * without slots: 107 us, 43 % of the copy rate; a lane has one pack under way, and
 * waits for its slot and then for its token before it has that.  The gradient reads
 * every slot's row once, as a whole, by the warp that holds its token: 80 us, 72
 * without weights (a token's chunks spread over four warps, four rows ahead: 89).
 * Two rows are asked for at a time and nothing while they are summed.
 */
#include "tb_learner.cuh"

using namespace tb_learn;

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kAhead = 2; /* rows of a token under way at once */
constexpr int kHeld = 4;  /* chunks of a row, of 32 packs, under way at once */

struct HandShape {
    size_t tokens, rows, width, rows_stride, token_stride;
    int top_k;
};

/* lanes: of a team that takes a row's chunk of `lanes` packs; chunks: of a row. */
template <class T, int PACK>
__global__ void __launch_bounds__(kThreads)
hand_out(HandShape d, int lanes, int chunks, const T *x, const int32_t *order, const float *weights, T *rows) {
    const size_t team = (static_cast<size_t>(blockIdx.x) * kThreads + threadIdx.x) / lanes;
    const int lane = threadIdx.x % lanes;
    const size_t p = team / chunks, c = ((team - p * chunks) * lanes + lane) * PACK;
    if (p >= d.rows || c >= d.width) return;
    const int32_t slot = order[p];
    if (slot < 0 || static_cast<size_t>(slot) >= d.tokens * d.top_k) return;
    Held<T, PACK> v = *reinterpret_cast<const Held<T, PACK> *>(x + static_cast<size_t>(slot / d.top_k) * d.token_stride + c);
    if (weights) {
        const float w = weights[slot];
        float e[PACK];
        unpack(v, e);
#pragma unroll
        for (int i = 0; i < PACK; ++i) e[i] *= w;
        v = packed<T, PACK>(e);
    }
    store_once<T, PACK>(rows + p * d.rows_stride + c, v);
}

/* A warp a token: kHeld chunks of 32 packs of its x and of the sums stay in
 * registers while its slots' rows pass by, two at a time, each read as a whole. */
template <class T, int PACK>
__global__ void __launch_bounds__(kThreads, 2)
hand_out_backward(HandShape d, const T *x, const int32_t *position, const float *weights, const T *drows, T *dx, float *dweights) {
    using V = typename Values<PACK>::V;
    constexpr int N = Values<PACK>::kCount;
    const int lane = threadIdx.x % 32;
    const size_t t = static_cast<size_t>(blockIdx.x) * kWarps + threadIdx.x / 32;
    if (t >= d.tokens) return;
    int32_t p = -1;
    float w = 1.0f, dot = 0.0f; /* of slot `lane` */
    if (lane < d.top_k) {
        p = position[t * d.top_k + lane];
        if (p >= 0 && static_cast<size_t>(p) >= d.rows) p = -1;
        if (weights) w = weights[t * d.top_k + lane];
    }
    for (size_t base = lane * PACK; base - lane * PACK < d.width; base += kHeld * 32 * PACK) {
        Array<PACK> g[kHeld], sum[kHeld];
#pragma unroll
        for (int h = 0; h < kHeld; ++h) {
            float e[PACK];
            Held<T, PACK> v{};
            if (dweights && base + h * 32 * PACK < d.width) v = load_once<T, PACK>(x + t * d.token_stride + base + h * 32 * PACK);
            unpack(v, e);
#pragma unroll
            for (int i = 0; i < N; ++i) g[h][i] = vload<V>(e + 2 * i), sum[h][i] = vall<V>(0.0f);
        }
        for (int j = 0; j < d.top_k; j += kAhead) {
            Held<T, PACK> v[kAhead][kHeld];
            int32_t row[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                row[k] = __shfl_sync(0xffffffffu, p, min(j + k, d.top_k - 1));
                if (j + k >= d.top_k) row[k] = -1;
#pragma unroll
                for (int h = 0; h < kHeld; ++h)
                    if (row[k] >= 0 && base + h * 32 * PACK < d.width)
                        v[k][h] = load_once<T, PACK>(drows + row[k] * d.rows_stride + base + h * 32 * PACK);
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (row[k] < 0) continue; /* the same for the whole warp */
                const V s = vall<V>(__shfl_sync(0xffffffffu, w, j + k));
                V of = vall<V>(0.0f);
#pragma unroll
                for (int h = 0; h < kHeld; ++h) {
                    if (base + h * 32 * PACK >= d.width) continue;
                    float e[PACK];
                    unpack(v[k][h], e);
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const V r = vload<V>(e + 2 * i);
                        sum[h][i] = vfma(s, r, sum[h][i]);
                        of = vfma(g[h][i], r, of);
                    }
                }
                if (dweights) {
                    float both[2] = {0.0f, 0.0f};
                    vstore(both, of);
                    const float all = warp_sum(both[0] + both[1]);
                    if (lane == j + k) dot += all;
                }
            }
        }
#pragma unroll
        for (int h = 0; h < kHeld; ++h)
            if (dx && base + h * 32 * PACK < d.width) {
                float e[PACK];
#pragma unroll
                for (int i = 0; i < N; ++i) vstore(e + 2 * i, sum[h][i]);
                *reinterpret_cast<Held<T, PACK> *>(dx + t * d.token_stride + base + h * 32 * PACK) = packed<T, PACK>(e);
            }
    }
    if (dweights && lane < d.top_k) dweights[t * d.top_k + lane] = dot;
}

bool hand_shape(const tb_expert_combine_desc *d, HandShape *s) {
    if (!d || !d->tokens || !d->rows || !d->width || d->top_k < 1 || d->top_k > TB_ROUTE_MAX_TOP_K ||
        !type_known(d->type) || d->rows > 0x7fffffffu)
        return false;
    size_t slots, all;
    if (!product(d->tokens, d->top_k, 0x7fffffffu, &slots)) return false;
    s->tokens = d->tokens;
    s->rows = d->rows;
    s->width = d->width;
    s->rows_stride = d->rows_stride ? d->rows_stride : d->width;
    s->token_stride = d->out_stride ? d->out_stride : d->width;
    s->top_k = d->top_k;
    return s->rows_stride >= d->width && s->token_stride >= d->width &&
           product(d->rows, s->rows_stride, SIZE_MAX / 64, &all) && product(d->tokens, s->token_stride, SIZE_MAX / 64, &all);
}

/* Calls f with the widest pack that every row of the tensors allows, as a
 * constant: 16, 8 or 4 bytes or an element. */
template <class T, class F>
int with_row_pack(const HandShape &s, const void *a, const void *b, const void *c, F &&f) {
    const size_t bits = reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c) |
                        (s.rows_stride | s.token_stride | s.width) * sizeof(T);
    if (bits % 16 == 8) return f(std::integral_constant<int, 8 / static_cast<int>(sizeof(T))>{});
    return with_pack<T>(pack_of(bits, sizeof(T)), f);
}

} /* namespace */

extern "C" int tb_cuda_hand_out_experts_device(const tb_expert_combine_desc *desc, const void *x, const int32_t *order,
                                               const float *weights, void *rows, void *stream) {
    HandShape s;
    if (!hand_shape(desc, &s) || !x || !order || !rows) return 0;
    const size_t size = type_size(desc->type);
    if (!aligned(x, size) || !aligned(rows, size) || !aligned(order, 4) || !aligned(weights, 4) ||
        collide({rows}, {x, order, weights}))
        return 0;
    cudaGetLastError(); /* report this launch only */
    return with_type(desc->type, [&](auto t) {
        using T = decltype(t);
        return with_row_pack<T>(s, x, rows, nullptr, [&](auto p) {
            constexpr int P = decltype(p)::value;
            const size_t packs = (s.width + P - 1) / P;
            int lanes = 1;
            while (lanes < 32 && static_cast<size_t>(lanes) < packs) lanes *= 2;
            const auto places = [&](size_t n) { return (packs + n - 1) / n * n; };
            while (lanes > 8 && places(lanes / 2) * 5 <= places(lanes) * 4) lanes /= 2;
            const size_t chunks = (packs + lanes - 1) / lanes;
            size_t teams;
            if (!product(s.rows, chunks, 0x7fffffffull * (kThreads / lanes), &teams) || chunks > 0x7fffffffu) return 0;
            hand_out<T, P><<<static_cast<unsigned>((teams * lanes + kThreads - 1) / kThreads), kThreads, 0,
                             static_cast<cudaStream_t>(stream)>>>(s, lanes, static_cast<int>(chunks), static_cast<const T *>(x),
                                                                  order, weights, static_cast<T *>(rows));
            return launched();
        });
    });
}

extern "C" int tb_cuda_hand_out_experts_backward_device(const tb_expert_combine_desc *desc, const void *x,
                                                        const int32_t *position, const float *weights, const void *drows,
                                                        void *dx, float *dweights, void *stream) {
    HandShape s;
    if (!hand_shape(desc, &s) || (!x && dweights) || !position || !drows || (!dx && !dweights)) return 0;
    const size_t size = type_size(desc->type);
    if (!aligned(x, size) || !aligned(drows, size) || !aligned(dx, size) || !aligned(position, 4) || !aligned(weights, 4) ||
        !aligned(dweights, 4) || collide({dx, dweights}, {x, position, weights, drows}))
        return 0;
    cudaGetLastError(); /* report this launch only */
    return with_type(desc->type, [&](auto t) {
        using T = decltype(t);
        return with_row_pack<T>(s, x, drows, dx, [&](auto p) {
            constexpr int P = decltype(p)::value;
            hand_out_backward<T, P><<<static_cast<unsigned>((s.tokens + kWarps - 1) / kWarps), kThreads, 0,
                                      static_cast<cudaStream_t>(stream)>>>(
                s, static_cast<const T *>(x), position, weights, static_cast<const T *>(drows), static_cast<T *>(dx), dweights);
            return launched();
        });
    });
}
