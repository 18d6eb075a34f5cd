/*
 * Group norm with an activation, channels last: forward and backward
 * (include/turbinator/training/cuda_learner.h).
 */
#include "tb_learner.cuh"

using namespace tb_learn;

namespace {

constexpr int kThreads = 256;

struct NormShape {
    size_t samples, positions;
    int channels, groups, per_group;
    size_t xs, xp, ys, yp; /* strides of samples and positions */
    int act;
    float epsilon;
};

__device__ __forceinline__ float activate(float u, int act) {
    if (act == TB_ACT_SILU) return u / (1.0f + expf(-u));
    if (act == TB_ACT_RELU) return u > 0.0f || u != u ? u : 0.0f;
    if (act == TB_ACT_GELU) return 0.5f * u * (1.0f + erff(u * 0.70710678f));
    return u;
}

__device__ __forceinline__ float slope(float u, int act) {
    if (act == TB_ACT_SILU) {
        const float s = 1.0f / (1.0f + expf(-u));
        return s * (1.0f + u * (1.0f - s));
    }
    if (act == TB_ACT_RELU) return u > 0.0f ? 1.0f : 0.0f;
    if (act == TB_ACT_GELU) return 0.5f * (1.0f + erff(u * 0.70710678f)) + u * expf(-0.5f * u * u) * 0.39894228f;
    return 1.0f;
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

/* One CTA per (sample, group). */
template <class T>
__global__ void __launch_bounds__(kThreads)
norm_forward(NormShape d, const T *x, const float *gamma, const float *beta, T *y, float *mean_out, float *rstd_out) {
    __shared__ float scratch[kThreads / 32];
    const size_t n = blockIdx.x / d.groups;
    const int g = static_cast<int>(blockIdx.x % d.groups);
    const int c0 = g * d.per_group;
    const size_t total = d.positions * d.per_group;
    const T *xs = x + n * d.xs + c0;
    float s = 0.0f;
    for (size_t i = threadIdx.x; i < total; i += kThreads)
        s += to_float(xs[i / d.per_group * d.xp + i % d.per_group]);
    const float mean = block_sum(s, scratch) / static_cast<float>(total);
    s = 0.0f;
    for (size_t i = threadIdx.x; i < total; i += kThreads) {
        const float v = to_float(xs[i / d.per_group * d.xp + i % d.per_group]) - mean;
        s += v * v;
    }
    const float rstd = 1.0f / sqrtf(block_sum(s, scratch) / static_cast<float>(total) + d.epsilon);
    if (threadIdx.x == 0 && mean_out) {
        mean_out[blockIdx.x] = mean;
        rstd_out[blockIdx.x] = rstd;
    }
    for (size_t i = threadIdx.x; i < total; i += kThreads) {
        const size_t p = i / d.per_group;
        const int c = static_cast<int>(i % d.per_group);
        const float u = (to_float(xs[p * d.xp + c]) - mean) * rstd * (gamma ? gamma[c0 + c] : 1.0f) +
                        (beta ? beta[c0 + c] : 0.0f);
        y[n * d.ys + p * d.yp + c0 + c] = from_float<T>(activate(u, d.act));
    }
}

/* One CTA per (sample, group); partial [samples, 2, channels]. */
template <class T>
__global__ void __launch_bounds__(kThreads)
norm_backward(NormShape d, const T *x, const float *gamma, const float *beta, const float *mean_in,
              const float *rstd_in, const T *dy, T *dx, float *partial) {
    __shared__ float scratch[kThreads / 32];
    const size_t n = blockIdx.x / d.groups;
    const int g = static_cast<int>(blockIdx.x % d.groups);
    const int c0 = g * d.per_group;
    const float mean = mean_in[blockIdx.x], rstd = rstd_in[blockIdx.x];
    float s1 = 0.0f, s2 = 0.0f;
    for (int c = c0; c < c0 + d.per_group; ++c) {
        const float ga = gamma ? gamma[c] : 1.0f, be = beta ? beta[c] : 0.0f;
        float a = 0.0f, b = 0.0f;
        for (size_t p = threadIdx.x; p < d.positions; p += kThreads) {
            const float hat = (to_float(x[n * d.xs + p * d.xp + c]) - mean) * rstd;
            const float du = to_float(dy[n * d.ys + p * d.yp + c]) * slope(hat * ga + be, d.act);
            a += du;
            b += du * hat;
        }
        a = block_sum(a, scratch);
        b = block_sum(b, scratch);
        if (threadIdx.x == 0) {
            partial[n * 2 * d.channels + c] = a;
            partial[n * 2 * d.channels + d.channels + c] = b;
        }
        s1 += ga * a;
        s2 += ga * b;
    }
    const float count = static_cast<float>(d.positions) * static_cast<float>(d.per_group);
    s1 /= count;
    s2 /= count;
    for (size_t i = threadIdx.x; i < d.positions * d.per_group; i += kThreads) {
        const size_t p = i / d.per_group;
        const int c = c0 + static_cast<int>(i % d.per_group);
        const float ga = gamma ? gamma[c] : 1.0f, be = beta ? beta[c] : 0.0f;
        const float hat = (to_float(x[n * d.xs + p * d.xp + c]) - mean) * rstd;
        const float du = to_float(dy[n * d.ys + p * d.yp + c]) * slope(hat * ga + be, d.act);
        dx[n * d.xs + p * d.xp + c] = from_float<T>(rstd * (du * ga - s1 - hat * s2));
    }
}

/* One CTA per channel. */
__global__ void __launch_bounds__(kThreads)
norm_parameters(const float *partial, size_t samples, int channels, float *dgamma, float *dbeta) {
    __shared__ float scratch[kThreads / 32];
    float a = 0.0f, b = 0.0f;
    for (size_t n = threadIdx.x; n < samples; n += kThreads) {
        a += partial[n * 2 * channels + blockIdx.x];
        b += partial[n * 2 * channels + channels + blockIdx.x];
    }
    a = block_sum(a, scratch);
    b = block_sum(b, scratch);
    if (threadIdx.x == 0) {
        if (dbeta) dbeta[blockIdx.x] = a;
        if (dgamma) dgamma[blockIdx.x] = b;
    }
}

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

} /* namespace */

extern "C" size_t tb_cuda_group_norm_workspace(const tb_group_norm_desc *desc) {
    NormShape s;
    if (!norm_shape(desc, &s)) return 0;
    return s.samples * 2 * s.channels * sizeof(float);
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
    return with_type(desc->type, [&](auto t) {
        using T = decltype(t);
        norm_forward<T><<<static_cast<unsigned>(s.samples * s.groups), kThreads, 0,
                          static_cast<cudaStream_t>(stream)>>>(s, static_cast<const T *>(x), gamma, beta,
                                                               static_cast<T *>(y), mean, rstd);
        return launched();
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
    return with_type(desc->type, [&](auto t) {
        using T = decltype(t);
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        float *partial = static_cast<float *>(workspace);
        norm_backward<T><<<static_cast<unsigned>(s.samples * s.groups), kThreads, 0, st>>>(
            s, static_cast<const T *>(x), gamma, beta, mean, rstd, static_cast<const T *>(dy), static_cast<T *>(dx),
            partial);
        if (!launched()) return 0;
        if (dgamma || dbeta)
            norm_parameters<<<s.channels, kThreads, 0, st>>>(partial, s.samples, s.channels, dgamma, dbeta);
        return launched();
    });
}
