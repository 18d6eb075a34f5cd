/*
 * The experts' rows back to their tokens: weighted sum and its gradient
 * (include/turbinator/training/cuda_learner.h).
 */
#include "tb_learner.cuh"

using namespace tb_learn;

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

struct CombineShape {
    size_t tokens, rows, width, rows_stride, out_stride;
    int top_k;
};

/* One warp per token. */
template <class T>
__global__ void __launch_bounds__(kThreads)
combine_forward(CombineShape d, const T *rows, const int32_t *position, const float *weights, T *out) {
    const size_t t = static_cast<size_t>(blockIdx.x) * kWarps + threadIdx.x / 32;
    if (t >= d.tokens) return;
    for (size_t c = threadIdx.x % 32; c < d.width; c += 32) {
        float s = 0.0f;
        for (int j = 0; j < d.top_k; ++j) {
            const int32_t p = position[t * d.top_k + j];
            if (p < 0 || static_cast<size_t>(p) >= d.rows) continue;
            s += (weights ? weights[t * d.top_k + j] : 1.0f) * to_float(rows[p * d.rows_stride + c]);
        }
        out[t * d.out_stride + c] = from_float<T>(s);
    }
}

template <class T>
__global__ void __launch_bounds__(kThreads)
combine_backward(CombineShape d, const T *rows, const int32_t *position, const float *weights, const T *dout,
                 T *drows, float *dweights) {
    const size_t t = static_cast<size_t>(blockIdx.x) * kWarps + threadIdx.x / 32;
    if (t >= d.tokens) return;
    for (int j = 0; j < d.top_k; ++j) {
        const int32_t p = position[t * d.top_k + j];
        const bool there = p >= 0 && static_cast<size_t>(p) < d.rows;
        float dot = 0.0f;
        if (there) {
            const float w = weights ? weights[t * d.top_k + j] : 1.0f;
            for (size_t c = threadIdx.x % 32; c < d.width; c += 32) {
                const float g = to_float(dout[t * d.out_stride + c]);
                if (dweights) dot += g * to_float(rows[p * d.rows_stride + c]);
                drows[p * d.rows_stride + c] = from_float<T>(w * g);
            }
        }
        dot = warp_sum(dot);
        if (dweights && threadIdx.x % 32 == 0) dweights[t * d.top_k + j] = dot;
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

unsigned combine_grid(const CombineShape &s) { return static_cast<unsigned>((s.tokens + kWarps - 1) / kWarps); }

} /* namespace */

extern "C" int tb_cuda_combine_experts_device(const tb_expert_combine_desc *desc, const void *rows,
                                              const int32_t *position, const float *weights, void *out,
                                              void *stream) {
    CombineShape s;
    if (!combine_shape(desc, &s) || !rows || !position || !out || rows == out) return 0;
    const size_t size = type_size(desc->type);
    if (!aligned(rows, size) || !aligned(out, size) || !aligned(position, 4) || !aligned(weights, 4)) return 0;
    cudaGetLastError(); /* report this launch only */
    return with_type(desc->type, [&](auto t) {
        using T = decltype(t);
        combine_forward<T><<<combine_grid(s), kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
            s, static_cast<const T *>(rows), position, weights, static_cast<T *>(out));
        return launched();
    });
}

extern "C" int tb_cuda_combine_experts_backward_device(const tb_expert_combine_desc *desc, const void *rows,
                                                       const int32_t *position, const float *weights,
                                                       const void *dout, void *drows, float *dweights,
                                                       void *stream) {
    CombineShape s;
    if (!combine_shape(desc, &s) || (!rows && dweights) || !position || !dout || !drows || drows == rows ||
        drows == dout)
        return 0;
    const size_t size = type_size(desc->type);
    if (!aligned(rows, size) || !aligned(dout, size) || !aligned(drows, size) || !aligned(position, 4) ||
        !aligned(weights, 4) || !aligned(dweights, 4))
        return 0;
    cudaGetLastError(); /* report this launch only */
    return with_type(desc->type, [&](auto t) {
        using T = decltype(t);
        combine_backward<T><<<combine_grid(s), kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
            s, static_cast<const T *>(rows), position, weights, static_cast<const T *>(dout),
            static_cast<T *>(drows), dweights);
        return launched();
    });
}
