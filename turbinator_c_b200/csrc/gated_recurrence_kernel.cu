/*
 * Gated linear recurrence with resets: forward and backward
 * (include/turbinator/training/cuda_learner.h).
 */
#include "tb_learner.cuh"

using namespace tb_learn;

namespace {

constexpr int kThreads = 128;
constexpr int kCheckpoint = TB_RECURRENCE_CHECKPOINT;

struct RecurrenceShape {
    size_t sequences, steps, channels;
    size_t is, it, os, ot, gs, gt; /* strides of sequences and steps: inputs, h, gradients */
    float scale;
};

__device__ __forceinline__ float softplus(float l) { return fmaxf(l, 0.0f) + log1pf(expf(-fabsf(l))); }
__device__ __forceinline__ float sigmoid(float v) { return 1.0f / (1.0f + expf(-v)); }

__device__ __forceinline__ size_t live_steps(const RecurrenceShape &d, const int32_t *lengths, size_t b) {
    if (!lengths) return d.steps;
    const int32_t n = lengths[b];
    return n < 0 ? 0 : static_cast<size_t>(n) < d.steps ? static_cast<size_t>(n) : d.steps;
}

struct Gates {
    float log_a, a, beta, open, gate, x;
};

template <class T>
__device__ __forceinline__ Gates gates_of(const T *x, const T *rec, const T *inp, size_t at, float rate, bool reset) {
    Gates g;
    g.open = sigmoid(to_float(rec[at]));
    g.gate = sigmoid(to_float(inp[at]));
    g.x = to_float(x[at]);
    g.log_a = rate * g.open;
    g.a = reset ? 0.0f : expf(g.log_a);
    g.beta = reset ? 1.0f : sqrtf(-expm1f(2.0f * g.log_a));
    return g;
}

/* One thread per (sequence, channel). */
template <class T>
__global__ void __launch_bounds__(kThreads)
recurrence_forward(RecurrenceShape d, const T *x, const T *rec, const T *inp, const float *decay,
                   const uint8_t *reset, const int32_t *lengths, const float *state_in, T *h, float *state_out,
                   float *checkpoints) {
    const size_t i = static_cast<size_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (i >= d.sequences * d.channels) return;
    const size_t b = i / d.channels, c = i % d.channels;
    const size_t live = live_steps(d, lengths, b), saved = (d.steps + kCheckpoint - 1) / kCheckpoint;
    const float rate = -d.scale * softplus(decay[c]);
    float s = state_in ? state_in[i] : 0.0f;
    for (size_t t = 0; t < d.steps; ++t) {
        if (checkpoints && t % kCheckpoint == 0) checkpoints[(b * saved + t / kCheckpoint) * d.channels + c] = s;
        float out = 0.0f;
        if (t < live) {
            const Gates g = gates_of(x, rec, inp, b * d.is + t * d.it + c, rate, reset && reset[b * d.steps + t]);
            s = g.a * s + g.beta * g.gate * g.x;
            out = s;
        }
        h[b * d.os + t * d.ot + c] = from_float<T>(out);
    }
    if (state_out) state_out[i] = s;
}

/* One thread per (sequence, channel); partial [sequences, channels]. */
template <class T>
__global__ void __launch_bounds__(kThreads)
recurrence_backward(RecurrenceShape d, const T *x, const T *rec, const T *inp, const float *decay,
                    const uint8_t *reset, const int32_t *lengths, const float *checkpoints, const T *dh,
                    const float *dstate_out, T *dx, T *drec, T *dinp, float *partial, float *dstate_in) {
    const size_t i = static_cast<size_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (i >= d.sequences * d.channels) return;
    const size_t b = i / d.channels, c = i % d.channels;
    const size_t live = live_steps(d, lengths, b), saved = (d.steps + kCheckpoint - 1) / kCheckpoint;
    const float rate = -d.scale * softplus(decay[c]);
    float carry = dstate_out ? dstate_out[i] : 0.0f, sum = 0.0f;
    for (size_t k = saved; k-- > 0;) {
        float before[kCheckpoint];
        float s = checkpoints[(b * saved + k) * d.channels + c];
#pragma unroll
        for (int j = 0; j < kCheckpoint; ++j) {
            const size_t t = k * kCheckpoint + j;
            before[j] = s;
            if (t < live) {
                const Gates g = gates_of(x, rec, inp, b * d.is + t * d.it + c, rate, reset && reset[b * d.steps + t]);
                s = g.a * s + g.beta * g.gate * g.x;
            }
        }
#pragma unroll
        for (int j = kCheckpoint - 1; j >= 0; --j) {
            const size_t t = k * kCheckpoint + j;
            if (t >= d.steps) continue;
            const size_t to = b * d.gs + t * d.gt + c;
            float gx = 0.0f, gr = 0.0f, gi = 0.0f;
            if (t < live) {
                const bool anew = reset && reset[b * d.steps + t];
                const Gates g = gates_of(x, rec, inp, b * d.is + t * d.it + c, rate, anew);
                const float total = to_float(dh[b * d.os + t * d.ot + c]) + carry;
                const float u = g.gate * g.x;
                carry = g.a * total;
                gx = total * g.beta * g.gate;
                gi = gx * g.x * (1.0f - g.gate);
                if (!anew && g.beta > 0.0f) {
                    const float dlog = carry * (before[j] - g.a / g.beta * u);
                    gr = dlog * g.log_a * (1.0f - g.open);
                    sum += dlog * g.open;
                }
            }
            dx[to] = from_float<T>(gx);
            drec[to] = from_float<T>(gr);
            dinp[to] = from_float<T>(gi);
        }
    }
    if (dstate_in) dstate_in[i] = carry;
    partial[i] = sum;
}

__global__ void __launch_bounds__(kThreads)
recurrence_decay(RecurrenceShape d, const float *decay, const float *partial, float *ddecay) {
    const size_t c = static_cast<size_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (c >= d.channels) return;
    float s = 0.0f;
    for (size_t b = 0; b < d.sequences; ++b) s += partial[b * d.channels + c];
    ddecay[c] = -d.scale * sigmoid(decay[c]) * s;
}

bool recurrence_shape(const tb_gated_recurrence_desc *d, RecurrenceShape *s) {
    if (!d || !d->sequences || !d->steps || !d->channels || !type_known(d->type) || !(d->decay_scale >= 0.0f) ||
        d->steps > 0x7fffffffu)
        return false;
    size_t rows, all;
    if (!product(d->sequences, d->channels, 0x7fffffffu, &rows) || !product(rows, d->steps, SIZE_MAX / 64, &all))
        return false;
    s->sequences = d->sequences;
    s->steps = d->steps;
    s->channels = d->channels;
    s->it = d->in_step_stride ? d->in_step_stride : d->channels;
    s->ot = d->out_step_stride ? d->out_step_stride : d->channels;
    s->gt = d->grad_step_stride ? d->grad_step_stride : d->channels;
    s->is = d->in_sequence_stride ? d->in_sequence_stride : d->steps * s->it;
    s->os = d->out_sequence_stride ? d->out_sequence_stride : d->steps * s->ot;
    s->gs = d->grad_sequence_stride ? d->grad_sequence_stride : d->steps * s->gt;
    s->scale = d->decay_scale;
    return s->it >= d->channels && s->ot >= d->channels && s->gt >= d->channels;
}

} /* namespace */

extern "C" size_t tb_cuda_gated_recurrence_workspace(const tb_gated_recurrence_desc *desc) {
    RecurrenceShape s;
    if (!recurrence_shape(desc, &s)) return 0;
    return s.sequences * s.channels * sizeof(float);
}

extern "C" int tb_cuda_gated_recurrence_device(const tb_gated_recurrence_desc *desc, const void *x,
                                               const void *recurrence_gate, const void *input_gate,
                                               const float *decay, const uint8_t *reset, const int32_t *lengths,
                                               const float *state_in, void *h, float *state_out,
                                               float *checkpoints, void *workspace, void *stream) {
    RecurrenceShape s;
    if (!recurrence_shape(desc, &s) || !x || !recurrence_gate || !input_gate || !decay || !h || !workspace) return 0;
    const size_t size = type_size(desc->type);
    if (!aligned(x, size) || !aligned(recurrence_gate, size) || !aligned(input_gate, size) || !aligned(h, size) ||
        !aligned(decay, 4) || !aligned(lengths, 4) || !aligned(state_in, 4) || !aligned(state_out, 4) ||
        !aligned(checkpoints, 4) || !aligned(workspace, 16) || h == x || h == recurrence_gate || h == input_gate)
        return 0;
    cudaGetLastError(); /* report these launches only */
    return with_type(desc->type, [&](auto t) {
        using T = decltype(t);
        const unsigned grid = static_cast<unsigned>((s.sequences * s.channels + kThreads - 1) / kThreads);
        recurrence_forward<T><<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
            s, static_cast<const T *>(x), static_cast<const T *>(recurrence_gate),
            static_cast<const T *>(input_gate), decay, reset, lengths, state_in, static_cast<T *>(h), state_out,
            checkpoints);
        return launched();
    });
}

extern "C" int tb_cuda_gated_recurrence_backward_device(
    const tb_gated_recurrence_desc *desc, const void *x, const void *recurrence_gate, const void *input_gate,
    const float *decay, const uint8_t *reset, const int32_t *lengths, const float *checkpoints, const void *dh,
    const float *dstate_out, void *dx, void *drecurrence_gate, void *dinput_gate, float *ddecay, float *dstate_in,
    void *workspace, void *stream) {
    RecurrenceShape s;
    if (!recurrence_shape(desc, &s) || !x || !recurrence_gate || !input_gate || !decay || !checkpoints || !dh ||
        !dx || !drecurrence_gate || !dinput_gate || !workspace)
        return 0;
    const size_t size = type_size(desc->type);
    if (!aligned(x, size) || !aligned(recurrence_gate, size) || !aligned(input_gate, size) || !aligned(dh, size) ||
        !aligned(dx, size) || !aligned(drecurrence_gate, size) || !aligned(dinput_gate, size) ||
        !aligned(decay, 4) || !aligned(lengths, 4) || !aligned(checkpoints, 4) || !aligned(dstate_out, 4) ||
        !aligned(ddecay, 4) || !aligned(dstate_in, 4) || !aligned(workspace, 16))
        return 0;
    const void *in[] = {x, recurrence_gate, input_gate, dh}, *out[] = {dx, drecurrence_gate, dinput_gate};
    for (int i = 0; i < 3; ++i) {
        for (const void *p : in)
            if (out[i] == p) return 0;
        if (out[i] == out[(i + 1) % 3]) return 0;
    }
    cudaGetLastError(); /* report these launches only */
    return with_type(desc->type, [&](auto t) {
        using T = decltype(t);
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        float *partial = static_cast<float *>(workspace);
        const unsigned grid = static_cast<unsigned>((s.sequences * s.channels + kThreads - 1) / kThreads);
        recurrence_backward<T><<<grid, kThreads, 0, st>>>(
            s, static_cast<const T *>(x), static_cast<const T *>(recurrence_gate),
            static_cast<const T *>(input_gate), decay, reset, lengths, checkpoints, static_cast<const T *>(dh),
            dstate_out, static_cast<T *>(dx), static_cast<T *>(drecurrence_gate), static_cast<T *>(dinput_gate),
            partial, dstate_in);
        if (!launched()) return 0;
        if (ddecay)
            recurrence_decay<<<static_cast<unsigned>((s.channels + kThreads - 1) / kThreads), kThreads, 0, st>>>(
                s, decay, partial, ddecay);
        return launched();
    });
}
