/*
 * Routing to experts: selection, weights, slot lists and the gradient of the
 * weights (include/turbinator/training/cuda_learner.h).
 *
 * Bound: the selection by issue (a few hundred instructions a token), the rest
 * by latency: the logits are read once, the outputs written once.  65,536
 * tokens, the best 8 of 256 experts, bf16: 51 us (selection 33, slot lists 13).
 * The gradient of their weights takes 16 us for 34 MB of dlogits, nearly all of
 * them zeros, 4 MB of ids and weights, and the sectors of the selected logits, 17
 * MB at most: 3.3 TB/s, the zeros' way through shared memory being the rest.
 *
 * Selection, one warp a token, its experts in registers (NV consecutive ones a
 * lane): each lane sorts out its four best keys, then top_k times the best of
 * the lanes' heads is taken and its lane moves on, three instructions of which
 * look at all lanes.  Which of the lane's experts a key belongs to is looked up
 * once at the end.  A lane that gives more than four (a few rows in 100,000 of
 * random logits with top_k 8 of 256) sends the warp to a search of all keys.
 *
 * Slot lists: a CTA on each SM selects for a tile of tokens and counts its
 * slots per expert; a second kernel places each tile's slots behind those of
 * the tiles before it: a rank within the warp (match), the warps before, the
 * tiles before.  No atomics decide an order.  A call of few slots is listed by
 * one CTA.
 */
#include "tb_learner.cuh"

using namespace tb_learn;

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMostTiles = 148;   /* tiles of tokens: one on each SM */
constexpr int kLeastTile = 8;     /* tokens */
constexpr int kPlaceThreads = 512;
constexpr int kPlaceWarps = kPlaceThreads / 32;
constexpr int kHeld = 8;          /* rows of 32 slots that a placing warp keeps in registers */
constexpr int kHeads = 4;         /* best keys that a lane keeps sorted; two: 72 us for 49 */

/* Threads of a selecting CTA: what an SM has registers for. */
constexpr int select_threads(int nv) { return nv <= 8 ? 1024 : nv <= 16 ? 512 : 256; }
constexpr float kNone = -INFINITY;

struct RouteShape {
    size_t tokens, stride;
    int experts, top_k, groups, top_groups, group_best;
    int score, renormalise;
    float scale;
};

__device__ __forceinline__ float available(float logit) { return logit == logit ? logit : kNone; }

/* The sigmoid whose bits the ranking is stated in: expf, one addition, one division. */
__device__ __forceinline__ float sigmoid(float v) { return 1.0f / (1.0f + expf(-v)); }
/* e^(l - most) for l <= most; the highest logits share where they are infinite. */
__device__ __forceinline__ float softened(float l, float most) {
    return l == most ? 1.0f : fast_exp2(kLog2e * (l - most));
}

/* Unsigned keys in the values' order; 0 for what cannot be taken (-inf, NaN). */
__device__ __forceinline__ unsigned key_of(float v) {
    const int b = __float_as_int(v + 0.0f); /* -0 ranks with 0 */
    const unsigned k = static_cast<unsigned>(b ^ (b >> 31 | static_cast<int>(0x80000000u)));
    return k - 0x00800000u <= 0xff800000u - 0x00800000u ? k : 0u; /* from the lowest finite value to +inf */
}

/* The value of a key. */
__device__ __forceinline__ float value_of(unsigned key) {
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

/* Keys of 16-bit logits that rank by themselves: 16 bits in the logits' order,
 * then 65,535 less the expert, so that no two are equal and ties go to the
 * lower expert. */
template <class T> __device__ __forceinline__ unsigned tagged_key(T v, int expert) {
    constexpr unsigned inf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    constexpr unsigned low = (0xffffu - (0x8000u | inf) + 1) << 16, high = (inf | 0x8000u) << 16 | 0xffffu;
    unsigned short h;
    memcpy(&h, &v, 2);
    int b = static_cast<int>(static_cast<unsigned>(h) << 16);
    if (static_cast<unsigned>(b) == 0x80000000u) b = 0; /* -0 ranks with 0 */
    unsigned k = static_cast<unsigned>(b ^ (b >> 31 | static_cast<int>(0x80000000u)));
    k = (k & 0xffff0000u) + (0xffffu - static_cast<unsigned>(expert));
    return k - low <= high - low ? k : 0u; /* from the lowest finite value to +inf */
}
template <class T> __device__ __forceinline__ float tagged_value(unsigned key) {
    const unsigned short h = static_cast<unsigned short>(key & 0x80000000u ? key >> 16 ^ 0x8000u : ~key >> 16);
    T v;
    memcpy(&v, &h, 2);
    return to_float(v);
}

/* NV logits of a token from expert `first` on, as they came: -inf where there is none. */
template <class T, int NV> struct Logits {
    static constexpr int P = NV * sizeof(T) < 16 ? NV : 16 / sizeof(T);
    Pack<T, P> v[NV / P];

    __device__ __forceinline__ void load(const T *row, int first, int experts, bool packs) {
        if (packs && first + NV <= experts) {
#pragma unroll
            for (int i = 0; i < NV / P; ++i) v[i] = *reinterpret_cast<const Pack<T, P> *>(row + first + i * P);
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i / P].v[i % P] = first + i < experts ? row[first + i] : from_float<T>(kNone);
        }
    }
    __device__ __forceinline__ T operator[](int i) const { return v[i / P].v[i % P]; }
};

/* The kHeads largest of NV keys, descending (0 where there are fewer). */
template <int NV> __device__ __forceinline__ void best_keys(const unsigned *key, unsigned (&head)[kHeads]) {
    if constexpr (NV > 4) {
        unsigned other[kHeads];
        best_keys<NV / 2>(key, head);
        best_keys<NV / 2>(key + NV / 2, other);
        /* the larger of each pair of a descending and an ascending run is bitonic */
#pragma unroll
        for (int i = 0; i < 4; ++i) head[i] = max(head[i], other[3 - i]);
#pragma unroll
        for (int o = 2; o > 0; o /= 2)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (!(i & o)) {
                    const unsigned high = max(head[i], head[i + o]);
                    head[i + o] = min(head[i], head[i + o]);
                    head[i] = high;
                }
    } else {
        constexpr int from[5] = {0, 2, 0, 1, 1}, to[5] = {1, 3, 2, 3, 2};
#pragma unroll
        for (int i = 0; i < 4; ++i) head[i] = i < NV ? key[i] : 0u;
#pragma unroll
        for (int i = 0; i < 5; ++i) {
            const unsigned high = max(head[from[i]], head[to[i]]);
            head[to[i]] = min(head[from[i]], head[to[i]]);
            head[from[i]] = high;
        }
    }
}

/* Leaves in value[] what the token's chosen groups hold, kNone elsewhere.  A
 * group is a run of lanes, or else read back from `row`. */
template <int NV>
__device__ __forceinline__ void keep_groups(const RouteShape &d, float (&value)[NV], float *row, int lane) {
    const int per = d.experts / d.groups, first = lane * NV;
    const int run = per / NV; /* lanes of a group */
    if (per % NV == 0 && (run & (run - 1)) == 0) {
        float a = kNone, b = kNone; /* the two best */
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            b = fmaxf(b, fminf(a, value[i]));
            a = fmaxf(a, value[i]);
        }
        for (int o = 1; o < run; o *= 2) {
            const float c = __shfl_xor_sync(0xffffffffu, a, o), e = __shfl_xor_sync(0xffffffffu, b, o);
            b = fmaxf(fminf(a, c), fmaxf(b, e));
            a = fmaxf(a, c);
        }
        const float strength = d.group_best == 2 && b > kNone ? a + b : a;
        const int mine = lane / run;
        int before = 0;
        for (int g = 0; g < d.groups; ++g) {
            const float other = __shfl_sync(0xffffffffu, strength, g * run);
            before += other > strength || (other == strength && g < mine);
        }
        if (before >= d.top_groups || strength == kNone)
#pragma unroll
            for (int i = 0; i < NV; ++i) value[i] = kNone;
        return;
    }
    float *const strength = row + d.experts;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (first + i < d.experts) row[first + i] = value[i];
    __syncwarp();
    for (int g = lane; g < d.groups; g += 32) {
        float a = kNone, b = kNone;
        for (int e = g * per; e < (g + 1) * per; ++e) {
            b = fmaxf(b, fminf(a, row[e]));
            a = fmaxf(a, row[e]);
        }
        strength[g] = d.group_best == 2 && b > kNone ? a + b : a;
    }
    __syncwarp();
    int last = -1;
    bool keep = false;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int g = (first + i) / per;
        if (first + i < d.experts && g != last) {
            last = g;
            const float s = strength[g];
            int before = 0;
            for (int h = 0; h < d.groups; ++h) before += strength[h] > s || (strength[h] == s && h < g);
            keep = before < d.top_groups && s > kNone;
        }
        if (!keep) value[i] = kNone;
    }
}

/* One warp per token.  count: [tiles, experts] where the slots are listed by
 * tiles, or NULL.  TAGGED: 16-bit logits rank by themselves, without groups,
 * and share a key's word with their expert: 48 us for 58. */
template <class T, int NV, bool TAGGED>
__global__ void __launch_bounds__(select_threads(NV), 1)
route_select(RouteShape d, int per_cta, bool packs, const T *logits, const float *bias, int32_t *ids, float *weights,
             int32_t *count) {
    /* a warp's keys [NV][32]; then, where they are needed, rows of experts + groups a warp */
    extern __shared__ __align__(16) unsigned char dynamic[];
    __shared__ int hist[TB_ROUTE_MAX_EXPERTS];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, first = lane * NV, warps = blockDim.x / 32;
    unsigned *const keys = reinterpret_cast<unsigned *>(dynamic) + warp * NV * 32;
    float *const rows = reinterpret_cast<float *>(dynamic) + warps * NV * 32 + warp * (d.experts + d.groups);
    if (count) {
        for (int e = threadIdx.x; e < d.experts; e += blockDim.x) hist[e] = 0;
        __syncthreads();
    }
    const bool soft = d.score == TB_SCORE_SOFTMAX;
    const bool scored = bias || (d.groups > 1 && d.group_best == 2); /* ranked, or grouped, by scores */
    float b[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) b[i] = bias && first + i < d.experts ? bias[first + i] : 0.0f;
    const size_t begin = static_cast<size_t>(blockIdx.x) * per_cta;
    const size_t end = begin + per_cta < d.tokens ? begin + per_cta : d.tokens;
    int lanes = 1; /* that slots take */
    while (lanes < d.top_k) lanes *= 2;
    Logits<T, NV> next;
    if (begin + warp < end) next.load(logits + (begin + warp) * d.stride, first, d.experts, packs);
    for (size_t t = begin + warp; t < end; t += warps) {
        const T *const in = logits + t * d.stride;
        float most = 0.0f, sum = 1.0f;
        unsigned key[NV], head[kHeads];
        const Logits<T, NV> now = next;
        if (t + warps < end) next.load(in + warps * d.stride, first, d.experts, packs);
        if constexpr (TAGGED) {
            if (soft && !d.renormalise) {
                most = kNone;
#pragma unroll
                for (int i = 0; i < NV; ++i) most = fmaxf(most, available(to_float(now[i])));
                most = warp_max(most);
                sum = 0.0f;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const float v = available(to_float(now[i]));
                    sum += v == kNone ? 0.0f : softened(v, most);
                }
                sum = warp_sum(sum);
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) key[i] = tagged_key(now[i], first + i);
        } else {
            float value[NV];
#pragma unroll
            for (int i = 0; i < NV; ++i) value[i] = available(to_float(now[i]));
            if (soft && (scored || !d.renormalise)) { /* else only the selected logits matter */
                most = kNone;
#pragma unroll
                for (int i = 0; i < NV; ++i) most = fmaxf(most, value[i]);
                most = warp_max(most);
                sum = 0.0f;
#pragma unroll
                for (int i = 0; i < NV; ++i) sum += value[i] == kNone ? 0.0f : softened(value[i], most);
                sum = warp_sum(sum);
            }
            if (scored || d.groups > 1) {
                float l[NV];
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    l[i] = value[i];
                    if (scored && l[i] != kNone)
                        value[i] = (soft ? softened(l[i], most) / sum : sigmoid(l[i])) + b[i];
                }
                if (d.groups > 1) {
                    keep_groups<NV>(d, value, rows, lane);
                    if (scored && !bias)
#pragma unroll
                        for (int i = 0; i < NV; ++i) value[i] = value[i] == kNone ? kNone : l[i];
                }
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                key[i] = key_of(value[i]);
                keys[i * 32 + lane] = key[i];
            }
        }
        best_keys<NV>(key, head);
        unsigned mine = 0; /* lane j's: the j-th best key, and its lane */
        int from = 0, given = 0, expert = -1;
        for (int j = 0; j < d.top_k; ++j) {
            const unsigned best = __reduce_max_sync(0xffffffffu, head[0]);
            bool wins = head[0] == best;
            if constexpr (!TAGGED) { /* of equal ones the first lane */
                const int winner = __ffs(__ballot_sync(0xffffffffu, wins)) - 1;
                from = lane == j ? winner : from;
                wins = lane == winner;
            }
            mine = lane == j ? best : mine;
#pragma unroll
            for (int i = 0; i + 1 < kHeads; ++i) head[i] = wins ? head[i + 1] : head[i];
            head[kHeads - 1] = wins ? 0u : head[kHeads - 1];
            given += wins;
        }
        /* a lane that gave all its heads: its fifth may belong (rounds in which
         * no head was left count too, and the search ends at once where nothing is) */
        if (NV > kHeads && __any_sync(0xffffffffu, given >= kHeads)) {
            mine = 0;
            for (int j = 0; j < d.top_k; ++j) {
                unsigned best = 0;
#pragma unroll
                for (int i = 0; i < NV; ++i) best = max(best, key[i]);
                const unsigned all = __reduce_max_sync(0xffffffffu, best);
                if (all == 0) break;
                const int winner = __ffs(__ballot_sync(0xffffffffu, best == all)) - 1;
                int at = NV;
#pragma unroll
                for (int i = NV - 1; i >= 0; --i)
                    if (key[i] == all) at = i;
                at = __shfl_sync(0xffffffffu, at, winner);
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    if (i == at && lane == winner) key[i] = 0;
                if (lane == j) mine = all, expert = winner * NV + at;
            }
        } else if constexpr (TAGGED) {
            if (mine != 0) expert = static_cast<int>(0xffffu - (mine & 0xffffu));
        } else {
            /* equal keys of one lane go to its experts in order */
            __syncwarp();
            const unsigned equal = __match_any_sync(0xffffffffu, mine) & ((1u << lane) - 1);
            int skip = 0;
            if (__any_sync(0xffffffffu, mine != 0 && equal != 0))
                for (int j = 0; j < d.top_k; ++j) {
                    const int other = __shfl_sync(0xffffffffu, from, j);
                    skip += (equal >> j & 1) && other == from;
                }
            if (mine != 0) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    if (keys[i * 32 + from] == mine && skip-- == 0) expert = from * NV + i;
            }
        }
        const bool takes = expert >= 0;
        float l = kNone;
        if (takes) l = TAGGED ? tagged_value<T>(mine) : scored ? to_float(in[expert]) : value_of(mine);
        float score;
        if (soft) {
            if (!scored && d.renormalise) most = __shfl_sync(0xffffffffu, l, 0); /* the best comes first */
            score = takes ? __fdividef(softened(l, most), sum) : 0.0f;
        } else {
            score = takes ? sigmoid(l) : 0.0f;
        }
        if (d.renormalise) {
            float total = score;
            for (int o = lanes / 2; o > 0; o /= 2) total += __shfl_xor_sync(0xffffffffu, total, o);
            score = total > 0.0f ? __fdividef(score, total) : 0.0f;
        }
        if (lane < d.top_k) {
            ids[t * d.top_k + lane] = expert;
            weights[t * d.top_k + lane] = score * d.scale;
        }
        if (count && takes) atomicAdd(&hist[expert], 1);
        __syncwarp();
    }
    if (count) {
        __syncthreads();
        for (int e = threadIdx.x; e < d.experts; e += kThreads) count[static_cast<size_t>(blockIdx.x) * d.experts + e] = hist[e];
    }
}

/* Places the slots of a tile of tokens (ALONE: of all tokens).  Each warp takes
 * consecutive slots; next[warp][expert] is where its next slot of the expert
 * goes. */
template <bool ALONE>
__global__ void __launch_bounds__(kPlaceThreads)
route_place(RouteShape d, int tile_tokens, const int32_t *ids, const int32_t *count, int32_t *offsets, int32_t *order,
            int32_t *position) {
    /* next [kPlaceWarps][experts]; of all tiles and of those before [kPlaceWarps][experts] each; first [experts] */
    extern __shared__ int next[];
    __shared__ int part[kPlaceWarps];
    int *const all_of = next + kPlaceWarps * d.experts, *const before_of = all_of + (ALONE ? 0 : kPlaceWarps * d.experts);
    int *const first = before_of + (ALONE ? 0 : kPlaceWarps * d.experts);
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const size_t slots = d.tokens * d.top_k;
    const size_t own_slots = ALONE ? slots : static_cast<size_t>(tile_tokens) * d.top_k;
    const size_t begin = blockIdx.x * own_slots, end = begin + own_slots < slots ? begin + own_slots : slots;
    const size_t each = (end - begin + kPlaceThreads - 1) / kPlaceThreads * 32; /* of a warp, whole rows of lanes */
    const size_t from = begin + warp * each, to = from + each < end ? from + each : end;
    int *const own = next + warp * d.experts;
    for (int e = lane; e < d.experts; e += 32) own[e] = 0;
    if (!ALONE) { /* every kPlaceWarps-th tile a warp */
        const int tile = static_cast<int>(blockIdx.x), tiles = static_cast<int>(gridDim.x);
        for (int e = lane; e < d.experts; e += 32) {
            int all = 0, before = 0;
#pragma unroll
            for (int i = 0; i < (kMostTiles + kPlaceWarps - 1) / kPlaceWarps; ++i) { /* all under way at once */
                const int b = warp + i * kPlaceWarps;
                const int c = b < tiles ? count[static_cast<size_t>(b) * d.experts + e] : 0;
                all += c;
                before += b < tile ? c : 0;
            }
            all_of[warp * d.experts + e] = all;
            before_of[warp * d.experts + e] = before;
        }
    }
    __syncwarp();
    int held[kHeld]; /* the warp's first rows of slots: most often all */
#pragma unroll
    for (int r = 0; r < kHeld; ++r) held[r] = from + r * 32 + lane < to ? ids[from + r * 32 + lane] : -1;
    const auto expert_at = [&](size_t base) { return base + lane < to ? ids[base + lane] : -1; };
    const auto count_row = [&](int e) {
        const unsigned peers = __match_any_sync(0xffffffffu, e);
        if (e >= 0 && lane == __ffs(peers) - 1) own[e] += __popc(peers);
        __syncwarp();
    };
#pragma unroll
    for (int r = 0; r < kHeld; ++r)
        if (from + r * 32 < to) count_row(held[r]);
    for (size_t base = from + kHeld * 32; base < to; base += 32) count_row(expert_at(base));
    __syncthreads();
    /* totals of the experts, then the experts before each: runs of experts a thread */
    const int run = (d.experts + kPlaceThreads - 1) / kPlaceThreads, mine = threadIdx.x * run;
    int sum = 0;
    for (int i = 0; i < run; ++i) {
        const int e = mine + i;
        if (e >= d.experts) break;
        int c = 0;
#pragma unroll
        for (int w = 0; w < kPlaceWarps; ++w) c += (ALONE ? next : all_of)[w * d.experts + e];
        first[e] = sum;
        sum += c;
    }
    int before = sum; /* inclusive over the threads, then exclusive */
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
    }
    if (lane == 31) part[warp] = before;
    __syncthreads();
    before -= sum;
    int all = 0;
#pragma unroll
    for (int w = 0; w < kPlaceWarps; ++w) {
        if (w == warp) before += all;
        all += part[w];
    }
    for (int i = 0; i < run; ++i) {
        const int e = mine + i;
        if (e >= d.experts) break;
        int at = first[e] + before;
        if (blockIdx.x == 0) offsets[e] = at;
        if (!ALONE)
#pragma unroll
            for (int w = 0; w < kPlaceWarps; ++w) at += before_of[w * d.experts + e];
#pragma unroll
        for (int w = 0; w < kPlaceWarps; ++w) {
            const int c = next[w * d.experts + e];
            next[w * d.experts + e] = at;
            at += c;
        }
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) offsets[d.experts] = all;
    __syncthreads();
    const auto place_row = [&](size_t base, int e) {
        const size_t i = base + lane;
        const unsigned peers = __match_any_sync(0xffffffffu, e);
        const int rank = __popc(peers & ((1u << lane) - 1));
        const int place = e >= 0 ? own[e] + rank : -1;
        __syncwarp();
        if (e >= 0 && rank == 0) own[e] += __popc(peers);
        __syncwarp();
        if (e >= 0) order[place] = static_cast<int32_t>(i);
        if (i < to) position[i] = place;
    };
#pragma unroll
    for (int r = 0; r < kHeld; ++r)
        if (from + r * 32 < to) place_row(from + r * 32, held[r]);
    for (size_t base = from + kHeld * 32; base < to; base += 32) place_row(base, expert_at(base));
    for (size_t i = all + static_cast<size_t>(blockIdx.x) * kPlaceThreads + threadIdx.x; i < slots;
         i += static_cast<size_t>(gridDim.x) * kPlaceThreads)
        order[i] = -1;
}

/* A row of gradients, from the warp's shared memory. */
template <class T>
__device__ __forceinline__ void store_row(T *out, const T *row, int experts, bool packs, int lane) {
    constexpr int P = 16 / sizeof(T);
    if (packs) {
        for (int e = lane * P; e < experts; e += 32 * P)
            *reinterpret_cast<Pack<T, P> *>(out + e) = *reinterpret_cast<const Pack<T, P> *>(row + e);
    } else {
        for (int e = lane; e < experts; e += 32) out[e] = row[e];
    }
}

/* Sigmoid scores, and renormalised softmax scores, where the whole row's sum
 * cancels: dlogit_j = w_j (dw_j - sum dw w).  Only the selected logits have a
 * gradient, and no other is read.  A warp takes 32 / lanes tokens together, a
 * lane a slot, then their rows one after the other. */
template <class T>
__global__ void __launch_bounds__(kThreads)
route_backward_selected(RouteShape d, int lanes, bool packs, const T *logits, const int32_t *ids, const float *dweights,
                        T *dlogits) {
    extern __shared__ __align__(16) unsigned char dynamic[];
    constexpr int P = 16 / sizeof(T);
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int pitch = (d.experts + P - 1) / P * P, tokens = 32 / lanes;
    T *const row = reinterpret_cast<T *>(dynamic) + warp * pitch;
    const size_t base = (static_cast<size_t>(blockIdx.x) * kWarps + warp) * tokens;
    if (base >= d.tokens) return;
    const size_t t = base + lane / lanes;
    const int j = lane % lanes;
    int id = -1;
    float l = kNone, dw = 0.0f;
    if (t < d.tokens && j < d.top_k) {
        id = ids[t * d.top_k + j];
        dw = dweights[t * d.top_k + j] * d.scale;
        if (id >= 0 && id < d.experts) l = available(to_float(logits[t * d.stride + id]));
    }
    for (int e = lane * P; e < pitch; e += 32 * P) *reinterpret_cast<uint4 *>(row + e) = make_uint4(0u, 0u, 0u, 0u);
    const bool there = l > kNone;
    if (!there) dw = 0.0f;
    const auto sum_of = [&](float v) {
        for (int o = lanes / 2; o > 0; o /= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    };
    float gradient; /* of logit `id` */
    if (d.score == TB_SCORE_SOFTMAX) {
        float most = l;
        for (int o = lanes / 2; o > 0; o /= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        float s = there ? softened(l, most) : 0.0f;
        const float total = sum_of(s);
        s = there ? s / total : 0.0f;
        gradient = s * (dw - sum_of(dw * s));
    } else {
        /* 2^24 of the score: not flushed where the forward pass's score is not */
        float s = there ? fast_rcp((1.0f + fast_exp2(-kLog2e * l)) * 0x1p-24f) : 0.0f;
        const float rest = there ? fast_sigmoid(-l) : 0.0f;
        if (d.renormalise) {
            const float total = sum_of(s), inner = sum_of(dw * s), over = total > 0.0f ? fast_rcp(total) : 0.0f;
            s *= over; /* the weight */
            dw = fmaf(-inner, over, dw);
        } else {
            s *= 0x1p-24f;
        }
        gradient = dw * s * rest;
    }
    for (int i = 0; i < tokens && base + i < d.tokens; ++i) {
        const bool mine = there && lane / lanes == i;
        __syncwarp();
        if (mine) row[id] = from_float<T>(gradient);
        __syncwarp();
        store_row(dlogits + (base + i) * d.stride, row, d.experts, packs, lane);
        __syncwarp();
        if (mine) row[id] = from_float<T>(0.0f);
    }
}

/* Softmax scores as they are: every logit of the row has a gradient, p_e (ds_e -
 * sum ds p).  One warp per token. */
template <class T>
__global__ void __launch_bounds__(kThreads)
route_backward_dense(RouteShape d, bool packs, const T *logits, const int32_t *ids, const float *dweights, T *dlogits) {
    extern __shared__ __align__(16) unsigned char dynamic[];
    constexpr int P = 16 / sizeof(T);
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int pitch = (d.experts + P - 1) / P * P;
    T *const row = reinterpret_cast<T *>(dynamic) + warp * pitch;
    const size_t t = static_cast<size_t>(blockIdx.x) * kWarps + warp;
    if (t >= d.tokens) return;
    const T *const in = logits + t * d.stride;
    const int id = lane < d.top_k ? ids[t * d.top_k + lane] : -1;
    const float l = id >= 0 && id < d.experts ? available(to_float(in[id])) : kNone;
    const bool there = l > kNone;
    const float dw = there ? dweights[t * d.top_k + lane] * d.scale : 0.0f;
    float most = kNone, sum = 0.0f;
    for (int e = lane; e < d.experts; e += 32) most = fmaxf(most, available(to_float(in[e])));
    most = warp_max(most);
    for (int e = lane; e < d.experts; e += 32) {
        const float v = available(to_float(in[e]));
        sum += v == kNone ? 0.0f : softened(v, most);
    }
    sum = warp_sum(sum);
    const float over = sum > 0.0f ? 1.0f / sum : 0.0f, s = there ? softened(l, most) * over : 0.0f;
    const float dot = warp_sum(dw * s);
    for (int e = lane; e < d.experts; e += 32) {
        const float v = available(to_float(in[e]));
        row[e] = from_float<T>(v == kNone ? 0.0f : -dot * (softened(v, most) * over));
    }
    __syncwarp();
    if (there) row[id] = from_float<T>(s * (dw - dot));
    __syncwarp();
    store_row(dlogits + t * d.stride, row, d.experts, packs, lane);
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

int tile_tokens(const RouteShape &s) {
    const size_t each = (s.tokens + kMostTiles - 1) / kMostTiles;
    return static_cast<int>(each < kLeastTile ? kLeastTile : each);
}
int route_tiles(const RouteShape &s) {
    const int each = tile_tokens(s);
    return static_cast<int>((s.tokens + each - 1) / each);
}
/* Whether one CTA lists all slots.  Its work grows with the slots, that of
 * tiles with the experts: of 64, 512 slots take 6.1 us alone and 6.9 in tiles,
 * 1,024 7.3 and 6.9; of 256, 800 slots 7.9 and 10.4, 2,400 11.0 and 10.2. */
bool route_alone(const RouteShape &s) { return s.tokens * s.top_k <= 512 + 6 * static_cast<size_t>(s.experts); }

/* Whether rows start on 16 bytes and hold whole packs of them. */
template <class T> bool route_packs(const RouteShape &s, const void *a, const void *b) {
    const size_t bits = reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | s.stride * sizeof(T);
    return (bits | s.experts * sizeof(T)) % 16 == 0;
}

template <class T, int NV>
int launch_select(const RouteShape &s, const T *logits, const float *bias, int32_t *ids, float *weights, int32_t *count,
                  cudaStream_t st) {
    /* tiles: as wide as an SM takes; else one token a warp, on many SMs */
    const int per_cta = count ? tile_tokens(s) : kWarps;
    int threads = count ? select_threads(NV) : kThreads;
    while (threads > kThreads && threads / 32 >= 2 * per_cta) threads /= 2;
    const int warps = threads / 32;
    const size_t shared = (static_cast<size_t>(warps) * NV * 32 + (s.groups > 1 ? warps * (s.experts + s.groups) : 0)) * 4;
    const unsigned grid = static_cast<unsigned>((s.tokens + per_cta - 1) / per_cta);
    const bool packs = route_packs<T>(s, logits, nullptr);
    if constexpr (sizeof(T) == 2)
        if (!bias && s.groups == 1) {
            route_select<T, NV, true><<<grid, threads, 0, st>>>(s, per_cta, packs, logits, bias, ids, weights, count);
            return launched();
        }
    if (!allow_shared<route_select<T, NV, false>>(shared)) return 0;
    route_select<T, NV, false><<<grid, threads, shared, st>>>(s, per_cta, packs, logits, bias, ids, weights, count);
    return launched();
}

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
        !aligned(offsets, 4) || !aligned(order, 4) || !aligned(position, 4) || !aligned(workspace, 16) ||
        collide({ids, weights, offsets, order, position, workspace}, {logits, bias}))
        return 0;
    cudaGetLastError(); /* report these launches only */
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool alone = route_alone(s);
    int32_t *count = static_cast<int32_t *>(workspace);
    int32_t *const to = offsets && !alone ? count : nullptr;
    const int ok = with_type(desc->type, [&](auto t) {
        using T = decltype(t);
        const T *in = static_cast<const T *>(logits);
        if (s.experts <= 32) return launch_select<T, 1>(s, in, bias, ids, weights, to, st);
        if (s.experts <= 64) return launch_select<T, 2>(s, in, bias, ids, weights, to, st);
        if (s.experts <= 128) return launch_select<T, 4>(s, in, bias, ids, weights, to, st);
        if (s.experts <= 256) return launch_select<T, 8>(s, in, bias, ids, weights, to, st);
        if (s.experts <= 512) return launch_select<T, 16>(s, in, bias, ids, weights, to, st);
        return launch_select<T, 32>(s, in, bias, ids, weights, to, st);
    });
    if (!ok || !offsets) return ok;
    const size_t shared = ((alone ? 1 : 3) * kPlaceWarps + 1) * s.experts * sizeof(int);
    if (alone) {
        if (!allow_shared<route_place<true>>(shared)) return 0;
        route_place<true><<<1, kPlaceThreads, shared, st>>>(s, 0, ids, nullptr, offsets, order, position);
    } else {
        if (!allow_shared<route_place<false>>(shared)) return 0;
        route_place<false><<<route_tiles(s), kPlaceThreads, shared, st>>>(s, tile_tokens(s), ids, count, offsets, order,
                                                                         position);
    }
    return launched();
}

extern "C" int tb_cuda_route_experts_backward_device(const tb_expert_route_desc *desc, const void *logits,
                                                     const int32_t *ids, const float *dweights, void *dlogits,
                                                     void *stream) {
    RouteShape s;
    if (!route_shape(desc, &s) || !logits || !ids || !dweights || !dlogits) return 0;
    const size_t size = type_size(desc->type);
    if (!aligned(logits, size) || !aligned(dlogits, size) || !aligned(ids, 4) || !aligned(dweights, 4) ||
        collide({dlogits}, {logits, ids, dweights}))
        return 0;
    cudaGetLastError(); /* report this launch only */
    return with_type(desc->type, [&](auto t) {
        using T = decltype(t);
        const size_t shared = kWarps * align_up(s.experts * sizeof(T), 16);
        const T *in = static_cast<const T *>(logits);
        T *out = static_cast<T *>(dlogits);
        const bool packs = route_packs<T>(s, dlogits, nullptr);
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (s.score == TB_SCORE_SOFTMAX && !s.renormalise) {
            if (!allow_shared<route_backward_dense<T>>(shared)) return 0;
            route_backward_dense<T><<<static_cast<unsigned>((s.tokens + kWarps - 1) / kWarps), kThreads, shared, st>>>(
                s, packs, in, ids, dweights, out);
            return launched();
        }
        int lanes = 1;
        while (lanes < s.top_k) lanes *= 2;
        const size_t per_cta = static_cast<size_t>(kWarps) * (32 / lanes);
        if (!allow_shared<route_backward_selected<T>>(shared)) return 0;
        route_backward_selected<T><<<static_cast<unsigned>((s.tokens + per_cta - 1) / per_cta), kThreads, shared, st>>>(
            s, lanes, packs, in, ids, dweights, out);
        return launched();
    });
}
