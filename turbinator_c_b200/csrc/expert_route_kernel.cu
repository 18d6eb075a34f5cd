/*
 * Routing to experts: selection, weights, slot lists and the gradient of the
 * weights (include/turbinator/training/cuda_learner.h).
 */
#include "tb_learner.cuh"

using namespace tb_learn;

namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kTileTokens = 128; /* tokens whose slots one CTA places */
constexpr float kNone = -INFINITY;

struct RouteShape {
    size_t tokens, stride;
    int experts, top_k, groups, top_groups, group_best;
    int score, renormalise;
    float scale;
};

__device__ __forceinline__ float available(float logit) { return logit == logit ? logit : kNone; }

/* The score's expression is the one whose bits the ranking is stated in:
 * expf, one addition, one division. */
__device__ __forceinline__ float sigmoid(float v) { return 1.0f / (1.0f + expf(-v)); }

/* Highest value of the warp's experts and the lowest index that has it;
 * index -1 where every value is -inf. */
__device__ __forceinline__ int warp_best(const float *value, int count, int lane, float *best) {
    float v = kNone;
    int at = -1;
    for (int e = lane; e < count; e += 32)
        if (value[e] > v) {
            v = value[e];
            at = e;
        }
    const float top = warp_max(v);
    int first = v == top && at >= 0 ? at : 0x7fffffff;
    first = __reduce_min_sync(0xffffffffu, first);
    *best = top;
    return first == 0x7fffffff ? -1 : first;
}

/* One warp per token. */
template <class T>
__global__ void __launch_bounds__(kThreads)
route_select(RouteShape d, const T *logits, const float *bias, int32_t *ids, float *weights) {
    extern __shared__ float shared[];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const size_t t = static_cast<size_t>(blockIdx.x) * kWarps + warp;
    float *logit = shared + warp * (2 * d.experts + d.groups), *value = logit + d.experts, *strength = value + d.experts;
    if (t >= d.tokens) return;
    float most = kNone;
    for (int e = lane; e < d.experts; e += 32) {
        logit[e] = available(to_float(logits[t * d.stride + e]));
        most = fmaxf(most, logit[e]);
    }
    most = warp_max(most);
    const bool soft = d.score == TB_SCORE_SOFTMAX;
    float sum = 0.0f;
    for (int e = lane; e < d.experts; e += 32) {
        const float l = logit[e];
        sum += l == kNone ? 0.0f : l == most ? 1.0f : expf(l - most);
    }
    sum = warp_sum(sum);
    const auto score_of = [&](float l) {
        if (l == kNone) return 0.0f;
        return soft ? (l == most ? 1.0f : expf(l - most)) / sum : sigmoid(l);
    };
    const bool by_logit = !bias && (d.groups == 1 || d.group_best == 1);
    for (int e = lane; e < d.experts; e += 32) {
        const float l = logit[e];
        value[e] = l == kNone || by_logit ? l : score_of(l) + (bias ? bias[e] : 0.0f);
    }
    __syncwarp();
    if (d.groups > 1) {
        const int per = d.experts / d.groups;
        for (int g = lane; g < d.groups; g += 32) {
            float a = kNone, b = kNone;
            for (int e = g * per; e < (g + 1) * per; ++e) {
                const float v = value[e];
                if (v > a) {
                    b = a;
                    a = v;
                } else if (v > b) {
                    b = v;
                }
            }
            strength[g] = d.group_best == 2 && b > kNone ? a + b : a;
        }
        __syncwarp();
        for (int r = 0; r < d.top_groups; ++r) {
            float best;
            const int g = warp_best(strength, d.groups, lane, &best);
            if (g < 0) break;
            __syncwarp();
            if (lane == 0) strength[g] = NAN; /* chosen */
            __syncwarp();
        }
        for (int e = lane; e < d.experts; e += 32) {
            const float s = strength[e / per];
            if (s == s) value[e] = kNone;
            else if (!bias && value[e] != kNone) value[e] = logit[e];
        }
        __syncwarp();
    }
    float total = 0.0f, mine = 0.0f; /* lane j keeps slot j */
    int id = -1;
    for (int j = 0; j < d.top_k; ++j) {
        float best;
        const int e = warp_best(value, d.experts, lane, &best);
        if (e < 0) break;
        const float s = score_of(logit[e]);
        total += s;
        if (lane == j) {
            id = e;
            mine = s;
        }
        __syncwarp();
        if (lane == 0) value[e] = kNone;
        __syncwarp();
    }
    if (lane < d.top_k) {
        ids[t * d.top_k + lane] = id;
        const float w = !d.renormalise ? mine : total > 0.0f ? mine / total : 0.0f;
        weights[t * d.top_k + lane] = w * d.scale;
    }
}

/* How many slots of each tile go to each expert: count [tiles, experts]. */
__global__ void __launch_bounds__(kThreads)
route_count(RouteShape d, const int32_t *ids, int32_t *count) {
    __shared__ int hist[TB_ROUTE_MAX_EXPERTS];
    for (int e = threadIdx.x; e < d.experts; e += kThreads) hist[e] = 0;
    __syncthreads();
    const size_t first = static_cast<size_t>(blockIdx.x) * kTileTokens;
    const size_t last = first + kTileTokens < d.tokens ? first + kTileTokens : d.tokens;
    for (size_t i = first * d.top_k + threadIdx.x; i < last * d.top_k; i += kThreads) {
        const int32_t e = ids[i];
        if (e >= 0) atomicAdd(&hist[e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < d.experts; e += kThreads)
        count[static_cast<size_t>(blockIdx.x) * d.experts + e] = hist[e];
}

/* Turns the counts into each tile's first place per expert, and writes the offsets. */
__global__ void __launch_bounds__(1024)
route_offsets(RouteShape d, int tiles, int32_t *count, int32_t *offsets) {
    __shared__ int total[TB_ROUTE_MAX_EXPERTS + 1];
    const int e = threadIdx.x;
    if (e < d.experts) {
        int s = 0;
        for (int b = 0; b < tiles; ++b) s += count[static_cast<size_t>(b) * d.experts + e];
        total[e] = s;
    }
    __syncthreads();
    if (e == 0) {
        int s = 0;
        for (int i = 0; i < d.experts; ++i) {
            const int c = total[i];
            total[i] = s;
            s += c;
        }
        total[d.experts] = s;
    }
    __syncthreads();
    if (e < d.experts) {
        int s = total[e];
        for (int b = 0; b < tiles; ++b) {
            const int c = count[static_cast<size_t>(b) * d.experts + e];
            count[static_cast<size_t>(b) * d.experts + e] = s;
            s += c;
        }
    }
    for (int i = e; i <= d.experts; i += 1024) offsets[i] = total[i];
}

/* One warp per tile, its slots in order. */
__global__ void __launch_bounds__(32)
route_place(RouteShape d, const int32_t *ids, const int32_t *count, const int32_t *offsets, int32_t *order,
            int32_t *position) {
    __shared__ int next[TB_ROUTE_MAX_EXPERTS];
    const int lane = threadIdx.x;
    for (int e = lane; e < d.experts; e += 32) next[e] = count[static_cast<size_t>(blockIdx.x) * d.experts + e];
    __syncwarp();
    const size_t first = static_cast<size_t>(blockIdx.x) * kTileTokens;
    const size_t last = first + kTileTokens < d.tokens ? first + kTileTokens : d.tokens;
    const size_t slots = d.tokens * d.top_k;
    for (size_t base = first * d.top_k; base < last * d.top_k; base += 32) {
        const size_t i = base + lane;
        const int e = i < last * d.top_k ? ids[i] : -1;
        const unsigned peers = __match_any_sync(0xffffffffu, e);
        const int rank = __popc(peers & ((1u << lane) - 1));
        int place = -1;
        if (e >= 0) place = next[e] + rank;
        __syncwarp();
        if (e >= 0 && rank == 0) next[e] += __popc(peers);
        __syncwarp();
        if (e >= 0) order[place] = static_cast<int32_t>(i);
        if (i < last * d.top_k) position[i] = place;
    }
    for (size_t i = offsets[d.experts] + static_cast<size_t>(blockIdx.x) * 32 + lane; i < slots;
         i += static_cast<size_t>(gridDim.x) * 32)
        order[i] = -1;
}

/* One warp per token. */
template <class T>
__global__ void __launch_bounds__(kThreads)
route_backward(RouteShape d, const T *logits, const int32_t *ids, const float *dweights, T *dlogits) {
    extern __shared__ float shared[];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const size_t t = static_cast<size_t>(blockIdx.x) * kWarps + warp;
    float *logit = shared + warp * 2 * d.experts, *dscore = logit + d.experts;
    if (t >= d.tokens) return;
    float most = kNone;
    for (int e = lane; e < d.experts; e += 32) {
        logit[e] = available(to_float(logits[t * d.stride + e]));
        most = fmaxf(most, logit[e]);
        dscore[e] = 0.0f;
    }
    most = warp_max(most);
    const bool soft = d.score == TB_SCORE_SOFTMAX;
    float sum = 0.0f;
    for (int e = lane; e < d.experts; e += 32) {
        const float l = logit[e];
        sum += l == kNone ? 0.0f : l == most ? 1.0f : expf(l - most);
    }
    sum = warp_sum(sum);
    const auto score_of = [&](float l) {
        if (l == kNone) return 0.0f;
        return soft ? (l == most ? 1.0f : expf(l - most)) / sum : sigmoid(l);
    };
    __syncwarp();
    const int id = lane < d.top_k ? ids[t * d.top_k + lane] : -1;
    const bool there = id >= 0 && id < d.experts;
    const float s = there ? score_of(logit[id]) : 0.0f;
    float ds = there ? dweights[t * d.top_k + lane] * d.scale : 0.0f;
    if (d.renormalise) {
        const float total = warp_sum(s);
        const float inner = warp_sum(ds * s);
        ds = there && total > 0.0f ? (ds - inner / total) / total : 0.0f;
    }
    if (there) dscore[id] = ds;
    const float dot = warp_sum(ds * s);
    __syncwarp();
    for (int e = lane; e < d.experts; e += 32) {
        const float p = score_of(logit[e]);
        const float g = soft ? p * (dscore[e] - dot) : dscore[e] * p * (1.0f - p);
        dlogits[t * d.stride + e] = from_float<T>(g);
    }
}

bool route_shape(const tb_expert_route_desc *d, RouteShape *s) {
    if (!d || !d->tokens || !d->experts || d->experts > TB_ROUTE_MAX_EXPERTS || d->top_k < 1 ||
        d->top_k > TB_ROUTE_MAX_TOP_K || static_cast<size_t>(d->top_k) > d->experts || d->groups < 1 ||
        d->experts % d->groups || d->top_groups < 1 || d->top_groups > d->groups || d->group_best < 1 ||
        d->group_best > 2 || !type_known(d->type) ||
        (d->score != TB_SCORE_SOFTMAX && d->score != TB_SCORE_SIGMOID) || !(d->weight_scale == d->weight_scale))
        return false;
    size_t slots, all;
    s->stride = d->logits_stride ? d->logits_stride : d->experts;
    if (!product(d->tokens, d->top_k, 0x7fffffffu, &slots) || s->stride < d->experts ||
        !product(d->tokens, s->stride, SIZE_MAX / 64, &all))
        return false;
    s->tokens = d->tokens;
    s->experts = static_cast<int>(d->experts);
    s->top_k = d->top_k;
    s->groups = d->groups;
    s->top_groups = d->top_groups;
    s->group_best = d->group_best;
    s->score = d->score;
    s->renormalise = d->renormalise;
    s->scale = d->weight_scale;
    return true;
}

int route_tiles(const RouteShape &s) { return static_cast<int>((s.tokens + kTileTokens - 1) / kTileTokens); }

} /* namespace */

extern "C" size_t tb_cuda_route_experts_workspace(const tb_expert_route_desc *desc) {
    RouteShape s;
    if (!route_shape(desc, &s)) return 0;
    return static_cast<size_t>(route_tiles(s)) * s.experts * sizeof(int32_t);
}

extern "C" int tb_cuda_route_experts_device(const tb_expert_route_desc *desc, const void *logits, const float *bias,
                                            int32_t *ids, float *weights, int32_t *offsets, int32_t *order,
                                            int32_t *position, void *workspace, void *stream) {
    RouteShape s;
    if (!route_shape(desc, &s) || !logits || !ids || !weights || !workspace || !offsets != !order ||
        !offsets != !position)
        return 0;
    if (!aligned(logits, type_size(desc->type)) || !aligned(bias, 4) || !aligned(ids, 4) || !aligned(weights, 4) ||
        !aligned(offsets, 4) || !aligned(order, 4) || !aligned(position, 4) || !aligned(workspace, 16))
        return 0;
    cudaGetLastError(); /* report these launches only */
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int ok = with_type(desc->type, [&](auto t) {
        using T = decltype(t);
        route_select<T><<<static_cast<unsigned>((s.tokens + kWarps - 1) / kWarps), kThreads,
                          kWarps * (2 * s.experts + s.groups) * sizeof(float), st>>>(
            s, static_cast<const T *>(logits), bias, ids, weights);
        return launched();
    });
    if (!ok || !offsets) return ok;
    int32_t *count = static_cast<int32_t *>(workspace);
    const int tiles = route_tiles(s);
    route_count<<<tiles, kThreads, 0, st>>>(s, ids, count);
    if (!launched()) return 0;
    route_offsets<<<1, 1024, 0, st>>>(s, tiles, count, offsets);
    if (!launched()) return 0;
    route_place<<<tiles, 32, 0, st>>>(s, ids, count, offsets, order, position);
    return launched();
}

extern "C" int tb_cuda_route_experts_backward_device(const tb_expert_route_desc *desc, const void *logits,
                                                     const int32_t *ids, const float *dweights, void *dlogits,
                                                     void *stream) {
    RouteShape s;
    if (!route_shape(desc, &s) || !logits || !ids || !dweights || !dlogits || logits == dlogits) return 0;
    const size_t size = type_size(desc->type);
    if (!aligned(logits, size) || !aligned(dlogits, size) || !aligned(ids, 4) || !aligned(dweights, 4)) return 0;
    cudaGetLastError(); /* report this launch only */
    return with_type(desc->type, [&](auto t) {
        using T = decltype(t);
        route_backward<T><<<static_cast<unsigned>((s.tokens + kWarps - 1) / kWarps), kThreads,
                            kWarps * 2 * s.experts * sizeof(float), static_cast<cudaStream_t>(stream)>>>(
            s, static_cast<const T *>(logits), ids, dweights, static_cast<T *>(dlogits));
        return launched();
    });
}
