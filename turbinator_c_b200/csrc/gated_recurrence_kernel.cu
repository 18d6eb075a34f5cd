/*
 * Gated linear recurrence with resets: forward and backward
 * (include/turbinator/training/cuda_learner.h).
 *
 * h_t = a_t h_(t-1) + b_t is a chain over t for each channel, but steps compose:
 * a span of steps maps the state before it, h, to A h + H, so spans can be
 * taken apart and joined.  A warp takes spans of 16 steps of 32 or 64 channels
 * (a tile); the warps of a CTA take consecutive spans of one tile, join them in
 * shared memory and go on together, the state in registers.  Inputs are staged
 * in shared memory one round ahead, outputs leave through the same slots: by
 * bulk tensor copies that one lane starts (every row on 16 bytes), else by
 * asynchronous copies of 16 or 4 bytes, else element by element.
 *
 * Bound: HBM with the gates' arithmetic close behind it (two sigmoids, a
 * softplus' share, an exponential and a square root a step and channel, on
 * packed pairs).  64 x 1,024 x 1,024 bf16, resets, states saved: forward 128 us
 * (4.3 TB/s), backward 258 us (3.7 TB/s), without resets 124 and 251.  Without
 * bulk copies 145 and 295 us; without the short series of decays that stay near
 * 1, 148 and 290 us.  What keeps both from their bounds is 18 % of the warps
 * that an SM could hold: a span's products stay in registers, 127 or 128 a
 * thread (backward some 150 bytes of them are spilled).
 *
 * Calls of few steps or of very many rows go step by step, a thread a pack of
 * channels (forward).
 *
 * Where tiles alone cannot fill the GPU, the steps are cut into strips and a
 * first kernel finds each strip's map, from which every strip's first state
 * follows: the inputs of the maps are read twice (three of the forward pass's
 * four tensors, two of the backward pass's seven), but nothing waits: three
 * logs of 15,005 to 30,011 x 321 f32 take 270 us, without strips 1,135; 64 x 1,024 x 128
 * bf16 backward 52 us and 81.  (The
 * strips joined in one kernel through published maps, each waiting for those
 * before it, was measured at 372 to 685 us on three logs of 30,011 steps: a
 * CTA that waits publishes its next map late, and so all wait.)
 *
 * The backward pass is the same scan in the other direction over
 * c_t = a_t (dh_t + c_(t+1)), the gradient of the state before step t; the
 * states that it needs are recomputed within 16 steps from the saved ones.
 */
#include <cuda.h> /* tensor maps */

#include "tb_features_internal.h"
#include "tb_learner.cuh"
#include "tb_pipeline.cuh"

using namespace tb_learn;

namespace {

constexpr int kSteps = TB_RECURRENCE_CHECKPOINT; /* steps of a warp's span, forward */
constexpr int kHalf = kSteps / 2;                /* and backward */
constexpr int kWarps = 4;                        /* warps of a CTA at most */
constexpr size_t kMostSteps = 0x7fffff00;        /* so that the last round's steps, of which some lie past the end, are ints */
static_assert(kMostSteps + 2 * kWarps * kSteps <= 0x7fffffff, "a round and the next one");

struct RecurrenceShape {
    size_t sequences, steps, channels;
    size_t is, it, os, ot, gs, gt; /* strides of sequences and steps: inputs, h, gradients */
    float scale;
};

struct ForwardArgs {
    RecurrenceShape d;
    const void *x, *rec, *inp;
    const float *decay, *state_in;
    const uint8_t *reset;
    const int32_t *lengths;
    void *h;
    float *state_out, *checkpoints;
    int in_piece, out_piece; /* bytes of a piece that rows move in */
};

struct BackwardArgs {
    RecurrenceShape d;
    const void *x, *rec, *inp, *dh;
    const float *decay, *checkpoints, *dstate_out;
    const uint8_t *reset;
    const int32_t *lengths;
    void *dx, *drec, *dinp;
    float *partial, *dstate_in; /* partial [spans, sequences, channels] */
    int in_piece, dh_piece, out_piece;
};

/* Who takes what: tiles of channels times strips of rounds (a span for each
 * of the CTA's warps), one unit of work each; unit = strip * tiles + tile. */
struct Split {
    unsigned tiles, tiles_per_sequence, rounds, strips, strip_rounds;
    unsigned magic_tiles, magic_sequence; /* floor((2^32 - 1) / tiles), .. / tiles_per_sequence) */
    float *maps;                          /* [tiles, strips, 2, channels of a tile] where strips > 1 */
    float *first;                         /* [sequences, channels]: the state before the scan, or NULL (keep_first) */
};

/* log(1 + e^l) = max(l, 0) + log(1 + e) with e = e^-|l|, log(1 + e) =
 * 2 artanh(e / (2 + e)), whose argument is at most 1/3: the series' next term
 * is below 2e-8 of it.  The exponent keeps the part that its product rounds
 * off, so that a far negative l has all its digits. */
__device__ __forceinline__ float softplus(float l) {
    const float a = -fabsf(l), n = a < -126.0f ? -126.0f : a, t = n * kLog2e; /* e is 0 from there on */
    float e = fast_exp2(t);
    e = fmaf(e, fmaf(n, kLog2e, -t) * 0.69314718f, e);
    const float r = e * fast_rcp(2.0f + e), q = r * r;
    float f = fmaf(q, 1.0f / 13.0f, 1.0f / 11.0f);
    f = fmaf(f, q, 1.0f / 9.0f);
    f = fmaf(f, q, 1.0f / 7.0f);
    f = fmaf(f, q, 1.0f / 5.0f);
    f = fmaf(f, q, 1.0f / 3.0f);
    f = fmaf(f, q, 1.0f);
    return fmaxf(l, 0.0f) + 2.0f * r * f;
}

/* log a of a fully open gate.  An infinite decay is one of 1e30: a product with
 * an infinite rate would be NaN where the other factor is 0. */
__device__ __forceinline__ float rate_of(float scale, float decay) {
    constexpr float most = 1e30f;
    const float s = softplus(decay), r = -scale * (s > most ? most : s);
    return r < -most ? -most : r;
}

/* Steps of sequence b that count. */
__device__ __forceinline__ int live_of(const RecurrenceShape &d, const int32_t *lengths, size_t b) {
    const int steps = static_cast<int>(d.steps);
    if (!lengths) return steps;
    const int n = lengths[b];
    return n < 0 ? 0 : n < steps ? n : steps;
}
/* Of `live` steps those of the span from step t on. */
__device__ __forceinline__ int of_span(int live, int t, int steps) { return min(max(live - t, 0), steps); }
template <int STEPS = kSteps> __device__ __forceinline__ int of_span(int live, int t) { return of_span(live, t, STEPS); }

/* e^l - 1 from its series, the next term below 5e-8 of it: for -kNear <= l <= 0
 * with five terms, for -kSeries <= l with seven. */
constexpr float kNear = 0.125f, kSeries = 0.35f;
template <bool NEAR> __device__ __forceinline__ F2 expm1_series(F2 l) {
    F2 q = both(1.0f / 120.0f);
    if (!NEAR) q = fma2(fma2(l, both(1.0f / 5040.0f), both(1.0f / 720.0f)), l, q);
    q = fma2(q, l, both(1.0f / 24.0f));
    q = fma2(q, l, both(1.0f / 6.0f));
    q = fma2(q, l, both(0.5f));
    q = fma2(q, l, both(1.0f));
    return mul2(l, q);
}

/* Decays of two steps or channels.  p = e^(log a) - 1 keeps the digits of
 * 1 - a^2 = -p (2 + p) where a is near 1.  NEAR: no log a of the warp can be
 * below -kNear (sigmoid <= 1, so the rates decide), which saves the
 * exponential, the choice and two terms. */
struct Decay {
    F2 a, beta;
};
template <bool NEAR> __device__ __forceinline__ Decay decay_of(F2 rate, F2 open) {
    const F2 l = mul2(rate, open);
    F2 p = expm1_series<NEAR>(l), a = add2(p, both(1.0f));
    if (!NEAR) {
        float l0, l1, p0, p1, a0, a1;
        split(l, l0, l1);
        split(p, p0, p1);
        split(a, a0, a1);
        if (!(l0 >= -kSeries)) {
            a0 = fast_exp2(kLog2e * l0);
            p0 = a0 - 1.0f;
        }
        if (!(l1 >= -kSeries)) {
            a1 = fast_exp2(kLog2e * l1);
            p1 = a1 - 1.0f;
        }
        a = pair(a0, a1);
        p = pair(p0, p1);
    }
    float s0, s1;
    split(mul2(p, fma2(p, both(-1.0f), both(-2.0f))), s0, s1);
    return {a, pair(fast_sqrt(s0), fast_sqrt(s1))};
}

/* ---- rows between global and the warp's shared memory ---- */

__device__ __forceinline__ uint32_t shared_address(const void *p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
template <int BYTES> __device__ __forceinline__ void copy_async(uint32_t to, const void *from, int bytes) {
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

/* N tensors of the same strides, at the same place: from[n] to
 * to + n * STEPS * CT, BYTES at a time. */
template <class T, int CT, int BYTES, int N, bool FULL, int STEPS>
__device__ __forceinline__ void load_pieces(T *to, const T *const (&from)[N], size_t at, size_t stride, int rows,
                                            int columns, int lane) {
    constexpr int kSize = static_cast<int>(sizeof(T));
    constexpr int kPer = CT * kSize / BYTES;          /* pieces of a row */
    constexpr int kRows = kPer < 32 ? 32 / kPer : 1;  /* rows at a time */
    constexpr int kTurns = kPer < 32 ? 1 : kPer / 32; /* pieces of a row a lane */
    const int row = kPer < 32 ? lane / kPer : 0;
    const size_t step = stride * kSize * kRows;
#pragma unroll
    for (int u = 0; u < kTurns; ++u) {
        const int piece = lane % (kPer < 32 ? kPer : 32) + 32 * u;
        const int left = columns * kSize - piece * BYTES;
        if (!FULL && left <= 0) return;
        const int bytes = FULL || left > BYTES ? BYTES : left;
        const size_t first = (at + row * stride) * kSize + piece * BYTES;
        const uint32_t t = shared_address(to + row * CT) + piece * BYTES;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const char *f = reinterpret_cast<const char *>(from[n]) + first;
#pragma unroll
            for (int r = 0; r < STEPS; r += kRows) {
                if (FULL || row + r < rows) copy_async<BYTES>(t + (n * STEPS + r) * CT * kSize, f, bytes);
                f += step;
            }
        }
    }
}

/* Starts copying rows x columns elements of N tensors into [N][STEPS][CT];
 * `piece` bytes at a time (16, 4: asynchronous). */
template <class T, int CT, int N, int STEPS = kSteps>
__device__ __forceinline__ void load_rows(T *to, const T *const (&from)[N], size_t at, size_t stride, int rows, int columns,
                                          int piece, int lane) {
    if (piece == 16) {
        if (rows == STEPS && columns == CT) load_pieces<T, CT, 16, N, true, STEPS>(to, from, at, stride, rows, columns, lane);
        else load_pieces<T, CT, 16, N, false, STEPS>(to, from, at, stride, rows, columns, lane);
    } else if (piece == 4) {
        load_pieces<T, CT, 4, N, false, STEPS>(to, from, at, stride, rows, columns, lane);
    } else {
        for (int n = 0; n < N; ++n)
            for (int c = lane; c < columns; c += 32)
#pragma unroll
                for (int r = 0; r < STEPS; ++r)
                    if (r < rows) to[(n * STEPS + r) * CT + c] = from[n][at + r * stride + c];
    }
}

/* rows x columns elements of from [STEPS][CT] to global memory. */
template <class T, int CT, int STEPS = kSteps>
__device__ __forceinline__ void store_rows(T *to, const T *from, size_t stride, int rows, int columns, int piece, int lane) {
    if (piece == 16) {
        constexpr int kPer = CT * static_cast<int>(sizeof(T)) / 16, kRows = 32 / kPer;
        constexpr int kIn = 16 / static_cast<int>(sizeof(T));
        const int row = lane / kPer, c = lane % kPer * kIn;
        const T *f = from + row * CT + c;
        T *t = to + row * stride + c;
        if (c + kIn <= columns) {
#pragma unroll
            for (int r = 0; r < STEPS; r += kRows)
                if (row + r < rows)
                    *reinterpret_cast<Pack<T, kIn> *>(t + r * stride) =
                        *reinterpret_cast<const Pack<T, kIn> *>(f + r * CT);
        } else {
            for (int r = 0; row + r < rows; r += kRows)
                for (int i = 0; c + i < columns; ++i) t[r * stride + i] = f[r * CT + i];
        }
    } else {
        for (int c = lane; c < columns; c += 32)
#pragma unroll
            for (int r = 0; r < STEPS; ++r)
                if (r < rows) to[r * stride + c] = from[r * CT + c];
    }
}

/* The same by bulk tensor copies: a box of steps x CT channels from one tensor.
 * A box lies on 128 bytes of shared memory.  Where the dynamic part starts
 * depends on the static part before it, so the first slot is moved up to the
 * next such place; calls ask for as much more. */
constexpr int kBoxAlign = 128;
template <class T> __device__ __forceinline__ T *slots_of(unsigned char *dynamic) {
    return reinterpret_cast<T *>(dynamic + (-shared_address(dynamic) & (kBoxAlign - 1)));
}
struct alignas(64) Maps {
    CUtensorMap in[4], out[3]; /* x, rec, inp, dh; h or dx, drec, dinp */
    unsigned *status;
    bool inner[3]; /* x, rec and inp; dh; the outputs: sequences lie within a step */
};
/* What a kernel without them takes in their place. */
struct NoMaps {
    unsigned *status;
};
template <bool BULK> using MapsOf = std::conditional_t<BULK, Maps, NoMaps>;
constexpr unsigned long long kWaitNs = 1000000000ull;

__device__ __forceinline__ void load_box(void *to, const CUtensorMap *map, int c, int t, int b, bool inner, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(shared_address(to)), "l"(map), "r"(c), "r"(inner ? b : t), "r"(inner ? t : b), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void store_box(const CUtensorMap *map, const void *from, int c, int t, int b, bool inner) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map),
                 "r"(shared_address(from)), "r"(c), "r"(inner ? b : t), "r"(inner ? t : b)
                 : "memory");
}
__device__ __forceinline__ void boxes_end() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
/* The lane's stores have read their slots; or are done. */
__device__ __forceinline__ void boxes_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void boxes_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

/* A warp's wait for its boxes, bounded: after a first timeout the stream's
 * status word says so and the kernel goes to its end without waiting again, nor
 * does it ask for boxes: a barrier whose boxes are still under way takes no
 * further arrival. */
struct BoxWait {
    unsigned long long limit = kWaitNs;
    __device__ __forceinline__ bool gave_up() const { return limit == 0; }
    __device__ __forceinline__ void operator()(uint32_t bar, unsigned parity, unsigned *status) {
        if (tb_pipe::mbar_wait(bar, parity, limit)) return;
        atomicOr(status, TB_FEATURE_STATUS_WAIT_TIMEOUT);
        limit = 0;
    }
    /* At the end: the lane's stores are done, and after a timeout boxes that are
     * still under way get another moment before their slots go. */
    __device__ __forceinline__ void finish(uint64_t (&bars)[2], int lane) {
        if (lane != 0) return;
        boxes_done();
        if (limit != 0) return;
        for (int n = 0; n < 2; ++n)
            for (unsigned parity = 0; parity < 2; ++parity)
                tb_pipe::mbar_wait(shared_address(&bars[n]), parity, kWaitNs / 8);
    }
};

/* Whether step t0 + lane starts anew. */
__device__ __forceinline__ unsigned reset_byte(const uint8_t *reset, size_t at, int live, int lane) {
    return reset && lane < live ? reset[at + lane] : 0u;
}

/* ---- the scan over spans ---- */

template <int V> struct Lane {
    float v[V];
};

/* A reset starts anew whatever the state was, an infinite or NaN one too, of
 * which 0 times it is not 0.  So a map of states over a reset has the
 * coefficient -0, which says that it takes nothing from the state before (no
 * other coefficient has this sign). */
constexpr float kAnew = -0.0f;
__device__ __forceinline__ bool starts_anew(float a) { return __float_as_int(a) < 0; }
/* Through the map (a, b): a state; the coefficient of a map before it.  Maps of
 * gradients (STATES false) have no such mark. */
template <bool STATES = true> __device__ __forceinline__ float carried(float a, float state, float b) {
    return STATES && starts_anew(a) ? b : fmaf(a, state, b);
}
template <bool STATES = true> __device__ __forceinline__ float carried(float a, float before) {
    return STATES && starts_anew(a) ? kAnew : a * before;
}
__device__ __forceinline__ bool finite(float v) { return fabsf(v) < INFINITY; }

/* Joins the spans of a CTA's round: each warp brings its span's map of V
 * channels a lane (`order`: its place in the scan) and the state before the
 * round; it leaves with the state before its own span, *state with that after
 * the round.  Every warp folds all spans, so one barrier a round does, given
 * buffers sa, sh that alternate. */
template <bool STATES, int CT, int V>
__device__ __forceinline__ Lane<V> join(const Lane<V> &map_a, const Lane<V> &map_h, Lane<V> *state, float (*sa)[CT],
                                        float (*sh)[CT], int order, int warps, int lane) {
    Lane<V> h = *state, mine = h;
    if (warps == 1) {
#pragma unroll
        for (int v = 0; v < V; ++v) state->v[v] = carried<STATES>(map_a.v[v], h.v[v], map_h.v[v]);
        return mine;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
        sa[order][lane * V + v] = map_a.v[v];
        sh[order][lane * V + v] = map_h.v[v];
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w >= warps) break;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if (w == order) mine.v[v] = h.v[v];
            h.v[v] = carried<STATES>(sa[w][lane * V + v], h.v[v], sh[w][lane * V + v]);
        }
    }
    *state = h;
    return mine;
}

/* Where a CTA works: a round of a strip of a tile. */
struct Place {
    unsigned round, last; /* rounds of the scan's order: this one, the strip's last */
    unsigned unit, b;
    int c0, live; /* first channel, steps of the sequence that count */
};

/* The first round of a unit. */
template <int CT>
__device__ __forceinline__ Place place_of(unsigned unit, const RecurrenceShape &d, const int32_t *lengths, const Split &s) {
    Place at;
    at.unit = unit;
    const unsigned strip = divided(unit, s.tiles, s.magic_tiles), tile = unit - strip * s.tiles;
    at.round = strip * s.strip_rounds;
    at.last = at.round + s.strip_rounds < s.rounds ? at.round + s.strip_rounds - 1 : s.rounds - 1;
    at.b = divided(tile, s.tiles_per_sequence, s.magic_sequence);
    at.c0 = static_cast<int>(tile - at.b * s.tiles_per_sequence) * CT;
    at.live = live_of(d, lengths, at.b);
    return at;
}

/* The round after it, of the next unit of the CTA at the strip's end. */
template <int CT>
__device__ __forceinline__ Place place_after(const Place &at, const RecurrenceShape &d, const int32_t *lengths, const Split &s) {
    Place next = at;
    if (++next.round <= at.last) return next;
    next.unit = at.unit + gridDim.x;
    if (next.unit < s.tiles * s.strips) next = place_of<CT>(next.unit, d, lengths, s);
    return next;
}

/* The state before a strip from `initial`, that before the first one: through
 * the maps of the strips before it, four parts of them at a time, one for each
 * of the warps that there are. */
template <bool STATES, int CT, int V>
__device__ Lane<V> before_strip(const Split &s, unsigned unit, const Lane<V> &initial, float (*sa)[CT], float (*sh)[CT],
                                int warp, int warps, int lane) {
    Lane<V> h = initial;
    const unsigned strip = divided(unit, s.tiles, s.magic_tiles), tile = unit - strip * s.tiles;
    const unsigned each = (strip + warps - 1) / warps, first = warp * each;
    const unsigned last = first + each < strip ? first + each : strip;
    float a[V], b[V];
#pragma unroll
    for (int v = 0; v < V; ++v) a[v] = 1.0f, b[v] = 0.0f;
    const float *m = s.maps + (static_cast<size_t>(tile) * s.strips + first) * 2 * CT + lane * V;
#pragma unroll 8
    for (unsigned i = first; i < last; ++i, m += 2 * CT)
#pragma unroll
        for (int v = 0; v < V; ++v) {
            b[v] = carried<STATES>(m[v], b[v], m[CT + v]);
            a[v] = carried<STATES>(m[v], a[v]);
        }
    __syncthreads(); /* the round before has read sa, sh */
#pragma unroll
    for (int v = 0; v < V; ++v) {
        sa[warp][lane * V + v] = a[v];
        sh[warp][lane * V + v] = b[v];
    }
    __syncthreads();
    for (int w = 0; w < warps; ++w)
#pragma unroll
        for (int v = 0; v < V; ++v) h.v[v] = carried<STATES>(sa[w][lane * V + v], h.v[v], sh[w][lane * V + v]);
    __syncthreads(); /* sa, sh are free again */
    return h;
}

/* Every strip starts from the state before the scan, and the last strip's CTA
 * writes the state after it: nothing orders the two.  Where one buffer holds
 * both, the CTA that finds the first strip's map leaves a copy that the strips
 * start from. */
template <int V>
__device__ __forceinline__ void keep_first(const Split &s, const Place &at, const RecurrenceShape &d, const float *states,
                                           int warp, int lane) {
    if (!s.first || at.round != 0 || warp != 0) return;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const size_t c = at.c0 + lane * V + v;
        if (c < d.channels) s.first[at.b * d.channels + c] = states[at.b * d.channels + c];
    }
}

/* A strip's map from those of its warps' parts, in the order of the scan. */
template <bool STATES, int CT, int V>
__device__ __forceinline__ void leave_map(const Split &s, unsigned unit, const Lane<V> &a, const Lane<V> &b, float (*sa)[CT],
                                          float (*sh)[CT], int order, int warps, int lane) {
    __syncthreads(); /* the unit before has read sa, sh */
#pragma unroll
    for (int v = 0; v < V; ++v) {
        sa[order][lane * V + v] = a.v[v];
        sh[order][lane * V + v] = b.v[v];
    }
    __syncthreads();
    if (order != 0) return;
    const unsigned strip = divided(unit, s.tiles, s.magic_tiles), tile = unit - strip * s.tiles;
    float *m = s.maps + (static_cast<size_t>(tile) * s.strips + strip) * 2 * CT + lane * V;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        float all = 1.0f, h = 0.0f;
        for (int w = 0; w < warps; ++w) {
            all = carried<STATES>(sa[w][lane * V + v], all);
            h = carried<STATES>(sa[w][lane * V + v], h, sh[w][lane * V + v]);
        }
        m[v] = all;
        m[CT + v] = h;
    }
}

/* ---- forward ---- */

/* Lanes of V channels: 64 channels (128 bytes) a row for 16-bit types, 32 for f32. */
template <class T> constexpr int kForwardV = sizeof(T) == 2 ? 2 : 1;

/* Pairs: two channels of a lane (V = 2), or two steps of its channel.  FAST:
 * the rates are NEAR, every step is live and none starts anew. */
template <class T, int V, bool FAST>
__device__ __forceinline__ void forward_span(const T *xs, const T *rs, const T *is, const float *rate, int live,
                                             unsigned anew, float (&prod)[kSteps][V], float (&local)[kSteps][V], int lane) {
    constexpr int CT = 32 * V;
    constexpr int second = V == 2 ? 1 : CT; /* from a pair's first element to its second */
    float a_one = 1.0f, h_one = 0.0f;
    F2 a_all = both(1.0f), h = both(0.0f);
    const F2 rates = pair(rate[0], rate[V - 1]);
#pragma unroll
    for (int j = 0; j < kSteps; j += 3 - V) {
        const int at = j * CT + lane * V;
        const auto two = [&](const T *p) {
            if constexpr (V == 2) {
                const Pack<T, 2> v = *reinterpret_cast<const Pack<T, 2> *>(p + at);
                return pair(to_float(v.v[0]), to_float(v.v[1]));
            } else {
                return pair(to_float(p[at]), to_float(p[at + second]));
            }
        };
        const Decay s = decay_of<FAST>(rates, sigmoid2(two(rs)));
        const F2 u = mul2(sigmoid2(two(is)), two(xs));
        F2 a = s.a, b = mul2(s.beta, u);
        if (!FAST) {
            float a0, a1, b0, b1, u0, u1;
            split(a, a0, a1);
            split(b, b0, b1);
            split(u, u0, u1);
            const int j1 = V == 2 ? j : j + 1;
            if (anew >> j & 1) a0 = 0.0f, b0 = u0;
            if (anew >> j1 & 1) a1 = 0.0f, b1 = u1;
            if (V == 2 && (anew >> j & 1)) a_all = h = both(0.0f); /* nothing before it is carried on */
            if (j >= live) a0 = 1.0f, b0 = 0.0f;
            if (j1 >= live) a1 = 1.0f, b1 = 0.0f;
            a = pair(a0, a1);
            b = pair(b0, b1);
        }
        if constexpr (V == 2) {
            a_all = mul2(a_all, a);
            h = fma2(a, h, b);
            split(a_all, prod[j][0], prod[j][1]);
            split(h, local[j][0], local[j][1]);
        } else {
            float a0, a1, b0, b1;
            split(a, a0, a1);
            split(b, b0, b1);
            if (!FAST && (anew >> j & 1)) a_one = h_one = 0.0f; /* nothing before it is carried on */
            prod[j][0] = a_one *= a0;
            local[j][0] = h_one = fmaf(a0, h_one, b0);
            if (!FAST && (anew >> (j + 1) & 1)) a_one = h_one = 0.0f;
            prod[j + 1][0] = a_one *= a1;
            local[j + 1][0] = h_one = fmaf(a1, h_one, b1);
        }
    }
}

/* BULK: by bulk tensor copies. */
template <class T, bool BULK>
__global__ void __launch_bounds__(32 * kWarps, 16 / kWarps)
recurrence_forward(const ForwardArgs p, const Split s, const __grid_constant__ MapsOf<BULK> maps) {
    constexpr int V = kForwardV<T>, CT = 32 * V;
    extern __shared__ __align__(16) unsigned char dynamic[];
    __shared__ uint64_t bars[kWarps][2]; /* of a stage's boxes */
    __shared__ float sa[2][kWarps][CT], sh[2][kWarps][CT];
    const RecurrenceShape &d = p.d;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32, steps = static_cast<int>(d.steps);
    T *const slots = slots_of<T>(dynamic) + warp * 2 * 3 * kSteps * CT; /* two stages of x, rec, inp */
    static_assert(kSteps * CT * sizeof(T) % kBoxAlign == 0, "a box's place");
    const size_t saved = (d.steps + kSteps - 1) / kSteps;
    const unsigned units = s.tiles * s.strips;

    BoxWait wait;
    const auto step_of = [&](const Place &to) { return static_cast<int>(to.round * warps + warp) * kSteps; };
    const auto start = [&](const Place &to, int stage) {
        const int t = step_of(to), left = static_cast<int>(d.channels) - to.c0;
        if constexpr (BULK) {
            if (lane == 0 && !wait.gave_up()) {
                boxes_read(); /* the slot's outputs of two rounds ago have left */
                const uint32_t bar = shared_address(&bars[warp][stage]);
                const bool any = t < to.live;
                tb_pipe::mbar_arrive_expect_tx(bar, any ? 3 * kSteps * CT * sizeof(T) : 0);
                for (int n = 0; n < 3 && any; ++n)
                    load_box(slots + (stage * 3 + n) * kSteps * CT, &maps.in[n], to.c0, t, static_cast<int>(to.b), maps.inner[0], bar);
            }
            return;
        }
        const T *const from[3] = {static_cast<const T *>(p.x), static_cast<const T *>(p.rec), static_cast<const T *>(p.inp)};
        load_rows<T, CT, 3>(slots + stage * 3 * kSteps * CT, from, to.b * d.is + t * d.it + to.c0, d.it,
                            of_span(to.live, t), left < CT ? left : CT, p.in_piece, lane);
        copies_end();
    };
    /* of the step that is the lane's number */
    const auto reset_at = [&](const Place &to) {
        const int t = step_of(to);
        return reset_byte(p.reset, to.b * d.steps + t, of_span(to.live, t), lane);
    };
    if (BULK && lane == 0) {
        for (int n = 0; n < 2; ++n) tb_pipe::mbar_init(shared_address(&bars[warp][n]), 1);
        tb_pipe::fence_mbar_init();
    }
    __syncwarp();

    Place at = place_of<CT>(blockIdx.x, d, p.lengths, s);
    int stage = 0;
    unsigned parity = 0; /* of both stages' barriers */
    start(at, 0);
    unsigned flag = reset_at(at);
    float rate[V];
    Lane<V> state;
    bool near = false, fresh = true;
    while (at.unit < units) {
        const int t = step_of(at), live = of_span(at.live, t), rows = of_span(steps, t);
        T *const xs = slots + stage * 3 * kSteps * CT;
        const unsigned anew = __ballot_sync(0xffffffffu, flag);
        const Place next = place_after<CT>(at, d, p.lengths, s);
        if (next.unit < units) {
            flag = reset_at(next);
            if (!BULK) start(next, stage ^ 1);
        } else if (!BULK) {
            copies_end();
        }
        if (fresh) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const size_t c = at.c0 + lane * V + v;
                const bool in = c < d.channels;
                rate[v] = in ? rate_of(d.scale, p.decay[c]) : 0.0f;
                state.v[v] = p.state_in && in ? p.state_in[at.b * d.channels + c] : 0.0f;
            }
            near = __all_sync(0xffffffffu, fminf(rate[0], rate[V - 1]) >= -kNear);
            if (at.round > 0) state = before_strip<true, CT, V>(s, at.unit, state, sa[stage], sh[stage], warp, warps, lane);
        }
        if (BULK) wait(shared_address(&bars[warp][stage]), parity, maps.status);
        else copies_wait<1>();
        __syncwarp();
        float prod[kSteps][V], local[kSteps][V];
        Lane<V> map_a, map_h;
        /* past the sequence's length nothing changes the state (three logs of up
         * to 10,000 x 320 bf16: 38 us, with all spans computed 46) */
        if (live == 0) {
#pragma unroll
            for (int v = 0; v < V; ++v) map_a.v[v] = 1.0f, map_h.v[v] = 0.0f;
        } else {
            if (live == kSteps && !anew && near)
                forward_span<T, V, true>(xs, xs + kSteps * CT, xs + 2 * kSteps * CT, rate, live, anew, prod, local, lane);
            else
                forward_span<T, V, false>(xs, xs + kSteps * CT, xs + 2 * kSteps * CT, rate, live, anew, prod, local, lane);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                map_a.v[v] = anew ? kAnew : prod[kSteps - 1][v];
                map_h.v[v] = local[kSteps - 1][v];
            }
        }
        const Lane<V> h0 = join<true, CT, V>(map_a, map_h, &state, sa[stage], sh[stage], warp, warps, lane);
        if (BULK && next.unit < units) start(next, stage ^ 1); /* half a round ahead: the other slot has been read */
        fresh = at.round == at.last;
        const bool ends = at.round + 1 == s.rounds && p.state_out && warp == 0;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const size_t c = at.c0 + lane * V + v;
            if (c >= d.channels) continue;
            if (p.checkpoints && rows > 0) p.checkpoints[(at.b * saved + t / kSteps) * d.channels + c] = h0.v[v];
            if (ends) p.state_out[at.b * d.channels + c] = state.v[v];
        }
        const auto leave = [&](auto cut) {
            Lane<V> from = h0;
#pragma unroll
            for (int j = 0; j < kSteps; j += 3 - V) {
                float o0, o1;
                if (decltype(cut)::value && (anew >> j & 1)) from.v[0] = from.v[V - 1] = 0.0f;
                float second = from.v[V - 1];
                if (decltype(cut)::value && V == 1 && (anew >> (j + 1) & 1)) second = 0.0f;
                split(fma2(pair(prod[j][0], prod[j + 2 - V][V - 1]), pair(from.v[0], second),
                           pair(local[j][0], local[j + 2 - V][V - 1])), o0, o1);
                if (V == 1) from.v[0] = second;
                if constexpr (V == 2) {
                    *reinterpret_cast<Pack<T, 2> *>(xs + j * CT + lane * 2) = {{from_float<T>(o0), from_float<T>(o1)}};
                } else {
                    xs[j * CT + lane] = from_float<T>(o0);
                    xs[(j + 1) * CT + lane] = from_float<T>(o1);
                }
            }
        };
        if (anew) leave(std::true_type{}); /* an infinite or NaN state ends at the first reset */
        else if (live > 0) leave(std::false_type{});
        if (live < kSteps) { /* steps past the sequence's length */
#pragma unroll
            for (int j = 0; j < kSteps; ++j)
                if (j >= live)
                    for (int v = 0; v < V; ++v) xs[j * CT + lane * V + v] = from_float<T>(0.0f);
        }
        if constexpr (BULK) {
            tb_pipe::fence_proxy_async_shared();
            __syncwarp();
            if (lane == 0 && rows > 0) {
                store_box(&maps.out[0], xs, at.c0, t, static_cast<int>(at.b), maps.inner[2]);
                boxes_end();
            }
        } else {
            __syncwarp();
            const int left = static_cast<int>(d.channels) - at.c0;
            store_rows<T, CT>(static_cast<T *>(p.h) + at.b * d.os + t * d.ot + at.c0, xs, d.ot, rows, left < CT ? left : CT,
                              p.out_piece, lane);
            __syncwarp();
        }
        at = next;
        parity ^= stage; /* each stage's barrier turns once in two rounds */
        stage ^= 1;
    }
    if constexpr (BULK) wait.finish(bars[warp], lane);
}

/* The maps of the strips, all but the last: each warp takes consecutive spans. */
template <class T>
__global__ void __launch_bounds__(32 * kWarps, 16 / kWarps) recurrence_forward_maps(const ForwardArgs p, const Split s) {
    constexpr int V = kForwardV<T>, CT = 32 * V;
    extern __shared__ __align__(16) unsigned char dynamic[];
    __shared__ float sa[kWarps][CT], sh[kWarps][CT];
    const RecurrenceShape &d = p.d;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
    T *const slots = reinterpret_cast<T *>(dynamic) + warp * 2 * 3 * kSteps * CT;
    const unsigned units = s.tiles * (s.strips - 1);
    for (unsigned unit = blockIdx.x; unit < units; unit += gridDim.x) {
        const Place at = place_of<CT>(unit, d, p.lengths, s);
        keep_first<V>(s, at, d, p.state_in, warp, lane);
        const int left = static_cast<int>(d.channels) - at.c0, columns = left < CT ? left : CT;
        const int first = static_cast<int>(at.round * warps + warp * s.strip_rounds);
        const int spans = of_span((at.live + kSteps - 1) / kSteps, first, static_cast<int>(s.strip_rounds)); /* that live */
        const auto start = [&](int span, int stage) {
            const int t = (first + span) * kSteps, live = of_span(at.live, t);
            const T *const from[3] = {static_cast<const T *>(p.x), static_cast<const T *>(p.rec), static_cast<const T *>(p.inp)};
            load_rows<T, CT, 3>(slots + stage * 3 * kSteps * CT, from, at.b * d.is + t * d.it + at.c0, d.it, live, columns,
                                p.in_piece, lane);
            return reset_byte(p.reset, at.b * d.steps + t, live, lane);
        };
        unsigned flag = start(0, 0);
        copies_end();
        float rate[V];
        Lane<V> a, b;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const size_t c = at.c0 + lane * V + v;
            rate[v] = c < d.channels ? rate_of(d.scale, p.decay[c]) : 0.0f;
            a.v[v] = 1.0f;
            b.v[v] = 0.0f;
        }
        const bool near = __all_sync(0xffffffffu, fminf(rate[0], rate[V - 1]) >= -kNear);
        for (int i = 0; i < spans; ++i) {
            const int live = of_span(at.live, (first + i) * kSteps);
            const unsigned anew = __ballot_sync(0xffffffffu, flag);
            const T *xs = slots + (i & 1) * 3 * kSteps * CT;
            if (i + 1 < spans) flag = start(i + 1, (i + 1) & 1);
            copies_end();
            copies_wait<1>();
            __syncwarp();
            float prod[kSteps][V], local[kSteps][V];
            if (live == kSteps && !anew && near)
                forward_span<T, V, true>(xs, xs + kSteps * CT, xs + 2 * kSteps * CT, rate, live, anew, prod, local, lane);
            else
                forward_span<T, V, false>(xs, xs + kSteps * CT, xs + 2 * kSteps * CT, rate, live, anew, prod, local, lane);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float through = anew ? kAnew : prod[kSteps - 1][v];
                b.v[v] = carried(through, b.v[v], local[kSteps - 1][v]);
                a.v[v] = carried(through, a.v[v]);
            }
            __syncwarp();
        }
        leave_map<true, CT, V>(s, unit, a, b, sa, sh, warp, warps, lane);
    }
}

/* ---- step by step ---- */

/* Floats of the thread's pack of channels; QUADS: rows of them on 16 bytes. */
template <int PACK, bool QUADS> __device__ __forceinline__ void load_floats(const float *from, float (&to)[PACK]) {
#pragma unroll
    for (int i = 0; i < PACK; i += QUADS ? 4 : 1) {
        if constexpr (QUADS) {
            const float4 v = *reinterpret_cast<const float4 *>(from + i);
            to[i] = v.x, to[i + 1] = v.y, to[i + 2] = v.z, to[i + 3] = v.w;
        } else {
            to[i] = from[i];
        }
    }
}
template <int PACK, bool QUADS> __device__ __forceinline__ void store_floats(float *to, const float (&from)[PACK]) {
#pragma unroll
    for (int i = 0; i < PACK; i += QUADS ? 4 : 1) {
        if constexpr (QUADS)
            *reinterpret_cast<float4 *>(to + i) = make_float4(from[i], from[i + 1], from[i + 2], from[i + 3]);
        else
            to[i] = from[i];
    }
}

/* For few steps, as programs that act take them, and for many rows: a thread
 * takes a pack of channels of every rows-th sequence through its steps, the
 * loads of TOGETHER steps at once, its rates found once.  No step is computed
 * that is not asked for, and no span is joined: one step of 4,096 x 512 bf16
 * takes 9.3 us (2.3 TB/s), by spans 101; of 64 x 512 2.2 and 4.5 us. */
constexpr int kFewSteps = 8, kSerialThreads = 128;
template <class T, int PACK, bool QUADS, int TOGETHER>
__global__ void __launch_bounds__(kSerialThreads)
recurrence_serial(const ForwardArgs p, unsigned packs, unsigned rows) {
    constexpr int N = (PACK + 1) / 2;
    const RecurrenceShape &d = p.d;
    const unsigned thread = blockIdx.x * kSerialThreads + threadIdx.x;
    if (thread >= packs * rows) return;
    const size_t c = static_cast<size_t>(thread % packs) * PACK;
    const int steps = static_cast<int>(d.steps);
    /* one channel: a pair of which the second is idle */
    const auto pairs = [](const float (&f)[PACK], int k) { return pair(f[2 * k], PACK > 1 ? f[PACK > 1 ? 2 * k + 1 : 0] : 0.0f); };
    F2 rate[N];
    {
        float l[PACK];
        load_floats<PACK, QUADS>(p.decay + c, l);
#pragma unroll
        for (int i = 0; i < PACK; ++i) l[i] = rate_of(d.scale, l[i]);
#pragma unroll
        for (int k = 0; k < N; ++k) rate[k] = pairs(l, k);
    }
    for (size_t b = thread / packs; b < d.sequences; b += rows) {
        const int live = live_of(d, p.lengths, b);
        float h[PACK];
#pragma unroll
        for (int i = 0; i < PACK; ++i) h[i] = 0.0f;
        if (p.state_in) load_floats<PACK, QUADS>(p.state_in + b * d.channels + c, h);
        float *saved = p.checkpoints ? p.checkpoints + b * ((d.steps + kSteps - 1) / kSteps) * d.channels + c : nullptr;
        const size_t in = b * d.is + c;
        T *to = static_cast<T *>(p.h) + b * d.os + c;
        for (int t = 0; t < steps; t += TOGETHER) {
            Held<T, PACK> x[TOGETHER], rec[TOGETHER], inp[TOGETHER];
            bool anew[TOGETHER];
            if (saved && t % kSteps == 0) {
                store_floats<PACK, QUADS>(saved, h);
                saved += d.channels;
            }
#pragma unroll
            for (int j = 0; j < TOGETHER; ++j) {
                if (t + j >= live) continue;
                const size_t at = in + (t + j) * d.it;
                x[j] = *reinterpret_cast<const Held<T, PACK> *>(static_cast<const T *>(p.x) + at);
                rec[j] = *reinterpret_cast<const Held<T, PACK> *>(static_cast<const T *>(p.rec) + at);
                inp[j] = *reinterpret_cast<const Held<T, PACK> *>(static_cast<const T *>(p.inp) + at);
                anew[j] = p.reset && p.reset[b * d.steps + t + j];
            }
#pragma unroll
            for (int j = 0; j < TOGETHER; ++j) {
                if (t + j >= steps) break;
                float out[PACK];
#pragma unroll
                for (int i = 0; i < PACK; ++i) out[i] = 0.0f;
                if (t + j < live) {
                    float xs[PACK], rs[PACK], is[PACK];
                    unpack(x[j], xs);
                    unpack(rec[j], rs);
                    unpack(inp[j], is);
#pragma unroll
                    for (int k = 0; k < N; ++k) {
                        const Decay s = decay_of<false>(rate[k], sigmoid2(pairs(rs, k)));
                        const F2 u = mul2(sigmoid2(pairs(is, k)), pairs(xs, k));
                        const F2 next = anew[j] ? u : fma2(s.a, pairs(h, k), mul2(s.beta, u));
                        float h0, h1;
                        split(next, h0, h1);
                        h[2 * k] = out[2 * k] = h0;
                        if (PACK > 1) h[2 * k + 1] = out[2 * k + 1] = h1;
                    }
                }
                *reinterpret_cast<Held<T, PACK> *>(to + (t + j) * d.ot) = packed<T, PACK>(out);
            }
        }
        if (p.state_out) store_floats<PACK, QUADS>(p.state_out + b * d.channels + c, h);
    }
}

/* ---- backward ---- */

/* A span of kHalf steps of two channels a lane.  What the gradients need of a
 * step: a; w = beta gate, so that dx = total w; z = x (1 - gate), so that dinp =
 * dx z; m = 1 - open; and q = open (h_(t-1) - a / beta gate x), so that a total
 * q is dlog a times open.  The span's first state h0 may not be known yet: q =
 * near_q + far_q h0. */
struct BackwardSpan {
    F2 a[kHalf], w[kHalf], z[kHalf], m[kHalf], near_q[kHalf], far_q[kHalf];
};

template <class T, int CT> __device__ __forceinline__ F2 two_of(const T *row, int lane) {
    const Pack<T, 2> v = *reinterpret_cast<const Pack<T, 2> *>(row + lane * 2);
    return pair(to_float(v.v[0]), to_float(v.v[1]));
}

/* map_a, map_h: the span's map of the state. */
template <class T, int CT>
__device__ __forceinline__ void backward_span(const T *xs, const T *rs, const T *is, F2 rate, bool near, int live,
                                              unsigned anew, BackwardSpan &g, F2 *map_a, F2 *map_h, int lane) {
    F2 beta[kHalf], open[kHalf], u[kHalf]; /* u = gate x */
#pragma unroll
    for (int j = 0; j < kHalf; ++j) {
        open[j] = sigmoid2(two_of<T, CT>(rs + j * CT, lane));
        const F2 gate = sigmoid2(two_of<T, CT>(is + j * CT, lane)), x = two_of<T, CT>(xs + j * CT, lane);
        const Decay s = decay_of<true>(rate, open[j]);
        g.a[j] = s.a;
        beta[j] = s.beta;
        u[j] = mul2(gate, x);
        g.z[j] = fma2(u[j], both(-1.0f), x);
        g.w[j] = gate; /* times beta, below */
    }
    if (!near) {
#pragma unroll
        for (int j = 0; j < kHalf; ++j) {
            const Decay s = decay_of<false>(rate, open[j]);
            g.a[j] = s.a;
            beta[j] = s.beta;
        }
    }
    unsigned still = 0; /* steps whose log a has no gradient */
    if (anew | (live < kHalf)) {
        still = anew | ~((1u << live) - 1);
#pragma unroll
        for (int j = 0; j < kHalf; ++j) {
            if (anew >> j & 1) g.a[j] = both(0.0f), beta[j] = both(1.0f);
            if (j >= live) { /* changes no state, and its gradients are zero */
                g.a[j] = both(1.0f);
                beta[j] = u[j] = g.z[j] = g.w[j] = open[j] = both(0.0f);
            }
        }
    }
    F2 prod = both(1.0f), h = both(0.0f);
#pragma unroll
    for (int j = 0; j < kHalf; ++j) {
        float b0, b1;
        split(beta[j], b0, b1);
        g.w[j] = mul2(beta[j], g.w[j]);
        g.m[j] = fma2(open[j], both(-1.0f), both(1.0f));
        /* where beta is 0, open or the rate is, which are factors of both
         * gradients: what stands for 1 / beta there only has to be finite */
        const F2 over = pair(fast_rcp(fmaxf(b0, 1e-18f)), fast_rcp(fmaxf(b1, 1e-18f)));
        g.near_q[j] = mul2(open[j], fma2(mul2(g.a[j], over), mul2(u[j], both(-1.0f)), h));
        g.far_q[j] = mul2(open[j], prod);
        h = fma2(g.a[j], h, mul2(beta[j], u[j]));
        prod = mul2(prod, g.a[j]);
    }
    if (still) {
#pragma unroll
        for (int j = 0; j < kHalf; ++j)
            if (still >> j & 1) g.near_q[j] = g.far_q[j] = both(0.0f);
    }
    *map_a = anew ? both(kAnew) : prod;
    *map_h = h;
}

/* Pairs of warps share 16 steps, so that the second's first state follows from
 * the saved one through the first's map. */
template <class T, bool BULK>
__global__ void __launch_bounds__(32 * kWarps, 16 / kWarps)
recurrence_backward(const BackwardArgs p, const Split s, const __grid_constant__ MapsOf<BULK> maps) {
    constexpr int CT = 64, kSlot = kHalf * CT;
    extern __shared__ __align__(16) unsigned char dynamic[];
    __shared__ uint64_t bars[kWarps][2]; /* of a stage's boxes */
    __shared__ float sa[2][kWarps][CT], sh[2][kWarps][CT], forward_h[2][kWarps][CT], sums[kWarps][CT];
    const RecurrenceShape &d = p.d;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32, steps = static_cast<int>(d.steps);
    T *const slots = slots_of<T>(dynamic) + warp * 2 * 4 * kSlot; /* two stages of x, rec, inp, dh */
    static_assert(kSlot * sizeof(T) % kBoxAlign == 0, "a box's place");
    const size_t saved = (d.steps + kSteps - 1) / kSteps;
    const unsigned units = s.tiles * s.strips;

    BoxWait wait;
    /* rounds in the order of the scan: the last steps first */
    const auto step_of = [&](const Place &to) {
        return static_cast<int>((s.rounds - 1 - to.round) * warps + warp) * kHalf;
    };
    const auto start = [&](const Place &to, int stage) {
        const int t = step_of(to), left = static_cast<int>(d.channels) - to.c0, columns = left < CT ? left : CT;
        const int live = of_span<kHalf>(to.live, t);
        if constexpr (BULK) {
            if (lane == 0 && !wait.gave_up()) {
                boxes_read(); /* the slot's outputs of two rounds ago have left */
                const uint32_t bar = shared_address(&bars[warp][stage]);
                tb_pipe::mbar_arrive_expect_tx(bar, 4 * kSlot * sizeof(T));
                for (int n = 0; n < 4; ++n)
                    load_box(slots + (stage * 4 + n) * kSlot, &maps.in[n], to.c0, t, static_cast<int>(to.b), maps.inner[n / 3], bar);
            }
            return;
        }
        const T *const from[3] = {static_cast<const T *>(p.x), static_cast<const T *>(p.rec), static_cast<const T *>(p.inp)};
        const T *const dh[1] = {static_cast<const T *>(p.dh)};
        load_rows<T, CT, 3, kHalf>(slots + stage * 4 * kSlot, from, to.b * d.is + t * d.it + to.c0, d.it, live, columns,
                                   p.in_piece, lane);
        load_rows<T, CT, 1, kHalf>(slots + stage * 4 * kSlot + 3 * kSlot, dh, to.b * d.os + t * d.ot + to.c0, d.ot, live,
                                   columns, p.dh_piece, lane);
        copies_end();
    };
    /* of the step that is the lane's number */
    const auto reset_at = [&](const Place &to) {
        const int t = step_of(to);
        return reset_byte(p.reset, to.b * d.steps + t, of_span<kHalf>(to.live, t), lane);
    };
    if (BULK && lane == 0) {
        for (int n = 0; n < 2; ++n) tb_pipe::mbar_init(shared_address(&bars[warp][n]), 1);
        tb_pipe::fence_mbar_init();
    }
    __syncwarp();
    /* two floats of the lane's channels, or zero */
    const auto two_floats = [&](const float *row, int c) {
        const int left = static_cast<int>(d.channels) - c;
        return pair(left > 0 ? row[c] : 0.0f, left > 1 ? row[c + 1] : 0.0f);
    };
    /* the saved state of the place's 16 steps: a row that moves with the rounds of a unit */
    const float *row = nullptr;
    const size_t row_step = static_cast<size_t>(warps * kHalf / kSteps) * d.channels;
    const auto saved_state = [&](const Place &to, bool anew) {
        const int t = step_of(to);
        if (anew) row = p.checkpoints + (to.b * saved + t / kSteps) * d.channels;
        else row -= row_step;
        return t < steps ? two_floats(row, to.c0 + lane * 2) : both(0.0f);
    };
    const auto put_floats = [&](float *row, int c, F2 v) {
        float a, b;
        split(v, a, b);
        const int left = static_cast<int>(d.channels) - c;
        if (left > 0) row[c] = a;
        if (left > 1) row[c + 1] = b;
    };

    Place at = place_of<CT>(blockIdx.x, d, p.lengths, s);
    int stage = 0;
    unsigned parity = 0; /* of both stages' barriers */
    start(at, 0);
    unsigned flag = reset_at(at);
    F2 h_next = saved_state(at, true);
    F2 rate = both(0.0f), sum_all = both(0.0f);
    Lane<2> state;
    bool near = false, fresh = true;
    while (at.unit < units) {
        const int t = step_of(at), live = of_span<kHalf>(at.live, t), rows = of_span<kHalf>(steps, t);
        const int c = at.c0 + lane * 2;
        T *const xs = slots + stage * 4 * kSlot;
        const unsigned anew = __ballot_sync(0xffffffffu, flag);
        F2 h0 = h_next;
        const Place next = place_after<CT>(at, d, p.lengths, s);
        if (next.unit < units) {
            flag = reset_at(next);
            h_next = saved_state(next, next.unit != at.unit);
            if (!BULK) start(next, stage ^ 1);
        } else if (!BULK) {
            copies_end();
        }
        if (fresh) {
            float l0, l1;
            split(two_floats(p.decay, c), l0, l1);
            l0 = c < static_cast<int>(d.channels) ? rate_of(d.scale, l0) : 0.0f;
            l1 = c + 1 < static_cast<int>(d.channels) ? rate_of(d.scale, l1) : 0.0f;
            rate = pair(l0, l1);
            near = __all_sync(0xffffffffu, fminf(l0, l1) >= -kNear);
            const F2 last = p.dstate_out ? two_floats(p.dstate_out + at.b * d.channels, c) : both(0.0f);
            split(last, state.v[0], state.v[1]);
            sum_all = both(0.0f);
            if (at.round > 0) state = before_strip<false, CT, 2>(s, at.unit, state, sa[stage], sh[stage], warp, warps, lane);
        }
        if (BULK) wait(shared_address(&bars[warp][stage]), parity, maps.status);
        else copies_wait<1>();
        __syncwarp();
        BackwardSpan g;
        F2 map_a, map_h;
        backward_span<T, CT>(xs, xs + kSlot, xs + 2 * kSlot, rate, near, live, anew, g, &map_a, &map_h, lane);
        F2 grad = both(0.0f); /* the span's map of the gradient, from zero after it */
#pragma unroll
        for (int j = kHalf - 1; j >= 0; --j)
            grad = mul2(g.a[j], add2(j < live ? two_of<T, CT>(xs + 3 * kSlot + j * CT, lane) : both(0.0f), grad));
        Lane<2> all, from_zero;
        split(map_a, all.v[0], all.v[1]);
        split(grad, from_zero.v[0], from_zero.v[1]);
        if (warps > 1) split(map_h, forward_h[stage][warp][lane * 2], forward_h[stage][warp][lane * 2 + 1]);
        const int order = warps - 1 - warp;
        const Lane<2> after = join<false, CT, 2>(all, from_zero, &state, sa[stage], sh[stage], order, warps, lane);
        grad = pair(after.v[0], after.v[1]);
        if (warp & 1) {
            float h_one[2];
            split(h0, h_one[0], h_one[1]);
#pragma unroll
            for (int v = 0; v < 2; ++v)
                h_one[v] = carried(sa[stage][order + 1][lane * 2 + v], h_one[v], forward_h[stage][warp - 1][lane * 2 + v]);
            h0 = pair(h_one[0], h_one[1]);
        }
        if ((anew & 1) | (live == 0)) h0 = both(0.0f); /* no step of the span takes it, whatever it is */
        if (BULK && next.unit < units) start(next, stage ^ 1); /* half a round ahead: the other slot has been read */
        fresh = at.round == at.last;
        if (at.round + 1 == s.rounds && p.dstate_in && warp == 0)
            put_floats(p.dstate_in + at.b * d.channels, c, pair(state.v[0], state.v[1]));
#pragma unroll
        for (int j = kHalf - 1; j >= 0; --j) {
            T *const to = xs + j * CT;
            const F2 total = add2(grad, j < live ? two_of<T, CT>(to + 3 * kSlot, lane) : both(0.0f));
            grad = mul2(g.a[j], total);
            const F2 gx = mul2(total, g.w[j]), dlog = mul2(grad, fma2(g.far_q[j], h0, g.near_q[j]));
            const auto leave = [&](T *row, F2 v) {
                float v0, v1;
                split(v, v0, v1);
                *reinterpret_cast<Pack<T, 2> *>(row + lane * 2) = {{from_float<T>(v0), from_float<T>(v1)}};
            };
            leave(to, gx);
            leave(to + kSlot, mul2(mul2(dlog, rate), g.m[j]));
            leave(to + 2 * kSlot, mul2(gx, g.z[j]));
            sum_all = add2(sum_all, dlog);
        }
        if (live < kHalf) { /* steps past the sequence's length, whatever dstate_out is */
#pragma unroll
            for (int j = 0; j < kHalf; ++j)
                if (j >= live)
                    for (int n = 0; n < 3; ++n)
                        *reinterpret_cast<Pack<T, 2> *>(xs + n * kSlot + j * CT + lane * 2) = {{from_float<T>(0.0f), from_float<T>(0.0f)}};
        }
        if constexpr (BULK) {
            tb_pipe::fence_proxy_async_shared();
            __syncwarp();
            if (lane == 0 && rows > 0) {
                for (int n = 0; n < 3; ++n) store_box(&maps.out[n], xs + n * kSlot, at.c0, t, static_cast<int>(at.b), maps.inner[2]);
                boxes_end();
            }
        } else {
            __syncwarp();
            const size_t to = at.b * d.gs + t * d.gt + at.c0;
            const int left = static_cast<int>(d.channels) - at.c0, columns = left < CT ? left : CT;
            store_rows<T, CT, kHalf>(static_cast<T *>(p.dx) + to, xs, d.gt, rows, columns, p.out_piece, lane);
            store_rows<T, CT, kHalf>(static_cast<T *>(p.drec) + to, xs + kSlot, d.gt, rows, columns, p.out_piece, lane);
            store_rows<T, CT, kHalf>(static_cast<T *>(p.dinp) + to, xs + 2 * kSlot, d.gt, rows, columns, p.out_piece, lane);
            __syncwarp();
        }
        if (fresh && p.partial) {
            split(sum_all, sums[warp][lane * 2], sums[warp][lane * 2 + 1]);
            __syncthreads();
            if (warp == 0) {
                F2 sum = both(0.0f);
                for (int i = 0; i < warps; ++i) sum = add2(sum, pair(sums[i][lane * 2], sums[i][lane * 2 + 1]));
                const size_t strip = divided(at.unit, s.tiles, s.magic_tiles);
                put_floats(p.partial + (strip * d.sequences + at.b) * d.channels, c, sum);
            }
            __syncthreads(); /* sums is free again */
        }
        at = next;
        parity ^= stage; /* each stage's barrier turns once in two rounds */
        stage ^= 1;
    }
    if constexpr (BULK) wait.finish(bars[warp], lane);
}

/* The maps of the strips, all but the last of the scan: of rec and dh alone. */
template <class T>
__global__ void __launch_bounds__(32 * kWarps, 16 / kWarps) recurrence_backward_maps(const BackwardArgs p, const Split s) {
    constexpr int CT = 64, kSlot = kHalf * CT;
    extern __shared__ __align__(16) unsigned char dynamic[];
    __shared__ float sa[kWarps][CT], sh[kWarps][CT];
    const RecurrenceShape &d = p.d;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
    T *const slots = reinterpret_cast<T *>(dynamic) + warp * 2 * 4 * kSlot;
    const unsigned units = s.tiles * (s.strips - 1);
    for (unsigned unit = blockIdx.x; unit < units; unit += gridDim.x) {
        const Place at = place_of<CT>(unit, d, p.lengths, s);
        keep_first<2>(s, at, d, p.dstate_out, warp, lane);
        const int left = static_cast<int>(d.channels) - at.c0, columns = left < CT ? left : CT;
        /* the strip's spans from its last steps on; warp 0 takes the first ones of the scan */
        const int spans = static_cast<int>(s.strip_rounds);
        const int top = static_cast<int>((s.rounds - at.round) * warps) - 1 - warp * spans;
        const auto start = [&](int span, int stage) {
            const int t = (top - span) * kHalf, live = of_span<kHalf>(at.live, t);
            const T *const rec[1] = {static_cast<const T *>(p.rec)}, *const dh[1] = {static_cast<const T *>(p.dh)};
            load_rows<T, CT, 1, kHalf>(slots + stage * 2 * kSlot, rec, at.b * d.is + t * d.it + at.c0, d.it, live, columns,
                                       p.in_piece, lane);
            load_rows<T, CT, 1, kHalf>(slots + stage * 2 * kSlot + kSlot, dh, at.b * d.os + t * d.ot + at.c0, d.ot, live,
                                       columns, p.dh_piece, lane);
            return reset_byte(p.reset, at.b * d.steps + t, live, lane);
        };
        /* those past the sequence's length change nothing */
        const int past = of_span(top + 1, (at.live + kHalf - 1) / kHalf, spans);
        unsigned flag = past < spans ? start(past, past & 1) : 0;
        copies_end();
        const int c = at.c0 + lane * 2;
        const float l0 = left > lane * 2 ? rate_of(d.scale, p.decay[c]) : 0.0f;
        const float l1 = left > lane * 2 + 1 ? rate_of(d.scale, p.decay[c + 1]) : 0.0f;
        F2 all = both(1.0f), grad = both(0.0f);
        for (int i = past; i < spans; ++i) {
            const int live = of_span<kHalf>(at.live, (top - i) * kHalf);
            const unsigned anew = __ballot_sync(0xffffffffu, flag);
            const T *rs = slots + (i & 1) * 2 * kSlot;
            if (i + 1 < spans) flag = start(i + 1, (i + 1) & 1);
            copies_end();
            copies_wait<1>();
            __syncwarp();
#pragma unroll
            for (int j = kHalf - 1; j >= 0; --j) {
                F2 a = decay_of<false>(pair(l0, l1), sigmoid2(two_of<T, CT>(rs + j * CT, lane))).a;
                if (anew >> j & 1) a = both(0.0f);
                if (j < live) {
                    grad = mul2(a, add2(two_of<T, CT>(rs + kSlot + j * CT, lane), grad));
                    all = mul2(all, a);
                }
            }
            __syncwarp();
        }
        Lane<2> map_a, map_h;
        split(all, map_a.v[0], map_a.v[1]);
        split(grad, map_h.v[0], map_h.v[1]);
        leave_map<false, CT, 2>(s, unit, map_a, map_h, sa, sh, warp, warps, lane);
    }
}

/* ddecay from the sums of dlog a / rate over all steps. */
struct DecayGradient {
    const float *decay;
    float scale, *ddecay;
    __device__ void operator()(size_t c, float sum) const { ddecay[c] = -scale / (1.0f + expf(-decay[c])) * sum; }
};

/* ---- host side ---- */

bool recurrence_shape(const tb_gated_recurrence_desc *d, RecurrenceShape *s) {
    if (!d || !d->sequences || !d->steps || !d->channels || !type_known(d->type) || !(d->decay_scale >= 0.0f) ||
        d->steps > kMostSteps)
        return false;
    size_t rows, all, items;
    if (!product(d->sequences, d->channels, 0x7fffffffu, &rows) || !product(rows, d->steps, SIZE_MAX / 64, &all) ||
        !product(d->sequences * ((d->channels + 31) / 32), (d->steps + kHalf - 1) / kHalf, 0x7fffffffu, &items))
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

constexpr unsigned kSms = 148;
constexpr unsigned kLeastRounds = 2; /* of a strip */

/* How a pass is laid out: steps of a span, channels of a tile, warps that an SM
 * has registers and shared memory for. */
struct Pass {
    int span, tile;
    unsigned room;
};
Pass forward_pass(int type) { return {kSteps, type == TB_TYPE_F32 ? 32 : 64, 16}; }
Pass backward_pass(int type) { return {kHalf, 64, type == TB_TYPE_F32 ? 12u : 16u}; }

/* Warps: as many as leave every tile room on the GPU at once (backward in
 * pairs).  Strips: where tiles of four warps take less than a third of the
 * room. */
Split split_of(const RecurrenceShape &d, const Pass &p, int *warps) {
    Split s{};
    s.tiles_per_sequence = static_cast<unsigned>((d.channels + p.tile - 1) / p.tile);
    s.tiles = static_cast<unsigned>(d.sequences * s.tiles_per_sequence);
    const unsigned spans = static_cast<unsigned>((d.steps + p.span - 1) / p.span), fill = p.room * kSms;
    unsigned w = fill / s.tiles;
    w = w < 1 ? 1 : w > kWarps ? kWarps : w;
    w = w > spans ? spans : w;
    if (p.span < kSteps && spans > 1) w = w < 4 ? 2 : 4;
    s.rounds = (spans + w - 1) / w;
    unsigned strips = fill / (s.tiles * w);
    if (strips < 3) strips = 1;
    const unsigned most = s.rounds / kLeastRounds;
    if (strips > most) strips = most < 2 ? 1 : most;
    s.strip_rounds = (s.rounds + strips - 1) / strips;
    s.strips = (s.rounds + s.strip_rounds - 1) / s.strip_rounds;
    s.magic_tiles = static_cast<unsigned>(0xffffffffull / s.tiles);
    s.magic_sequence = static_cast<unsigned>(0xffffffffull / s.tiles_per_sequence);
    *warps = static_cast<int>(w);
    return s;
}
size_t map_bytes(const Split &s, int tile) {
    return s.strips > 1 ? static_cast<size_t>(s.tiles) * s.strips * 2 * tile * sizeof(float) : 0;
}
size_t first_bytes(const RecurrenceShape &d, const Split &s) {
    return s.strips > 1 ? d.sequences * d.channels * sizeof(float) : 0;
}

/* Rows of partial sums for ddecay, and behind them the parts that they are first summed into. */
size_t partial_rows(const RecurrenceShape &d, const Split &s) { return d.sequences * s.strips; }
size_t partial_bytes(const RecurrenceShape &d, const Split &s) {
    const size_t rows = partial_rows(d, s);
    return (rows + column_parts(rows)) * d.channels * sizeof(float);
}

/* Largest piece that every row of a tensor starts and goes on at. */
int piece_of(const void *p, size_t sequence_stride, size_t step_stride, size_t size, int least) {
    const size_t all = reinterpret_cast<uintptr_t>(p) | sequence_stride * size | step_stride * size;
    return all % 16 == 0 ? 16 : all % 4 == 0 && least == 4 ? 4 : 0;
}

/* Tensor maps of [sequences, steps, channels] tensors in boxes of one warp's
 * span and tile; of the two outer dimensions the one of smaller stride comes
 * first (*inner: sequences do), since CUDA's interface wants each stride to be
 * a multiple of the one before.  False where CUDA has no such copies or refuses
 * them, or the larger stride is no such multiple. */
using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encoder() {
    static std::atomic<EncodeTiled> known{nullptr};
    EncodeTiled f = known.load(std::memory_order_relaxed);
    if (!f) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult result;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &result) != cudaSuccess ||
            result != cudaDriverEntryPointSuccess)
            return nullptr;
        f = reinterpret_cast<EncodeTiled>(p);
        known.store(f, std::memory_order_relaxed);
    }
    return f;
}
bool encode(CUtensorMap *map, bool *inner, int type, const void *tensor, const RecurrenceShape &d, size_t sequence_stride,
            size_t step_stride, const Pass &pass) {
    const EncodeTiled f = encoder();
    const size_t size = type_size(type);
    const bool in = d.sequences > 1 && sequence_stride < step_stride; /* sequences lie within a step */
    const size_t first = (in ? sequence_stride : step_stride) * size;
    const size_t second = in ? step_stride * size : d.sequences > 1 ? sequence_stride * size : first;
    *inner = in;
    const cuuint64_t extent[3] = {d.channels, in ? d.sequences : d.steps, in ? d.steps : d.sequences};
    const cuuint64_t stride[2] = {first, second};
    const cuuint32_t span = static_cast<cuuint32_t>(pass.span);
    const cuuint32_t box[3] = {static_cast<cuuint32_t>(pass.tile), in ? 1 : span, in ? span : 1}, one[3] = {1, 1, 1};
    const CUtensorMapDataType kind = type == TB_TYPE_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : type == TB_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                            : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    return f && second < 1ull << 40 && second % first == 0 &&
           f(map, kind, 3, const_cast<void *>(tensor), extent, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
               CUDA_SUCCESS;
}
/* Bulk copies from this many rounds of a unit on: encoding the maps takes the
 * host 1 to 2 us, which short calls wait for; on the GPU short units gain nothing (256 x 64 x 1,024 bf16:
 * 34 us with them and without, of few rounds). */
constexpr unsigned kBulkRounds = 4;

/* Launches a kernel over `work` units: at most as many CTAs as there is room
 * for, each taking every grid-th unit. */
template <auto Kernel, class... Args>
int launch_units(unsigned work, const Pass &pass, int warps, size_t shared, cudaStream_t st, const Args &...args) {
    int dev = 0;
    const int sms = multiprocessors(&dev);
    if (!sms || !allow_shared<Kernel>(shared)) return 0;
    const unsigned most = static_cast<unsigned>(sms) * (pass.room / warps);
    Kernel<<<work < most ? work : most, warps * 32, shared, st>>>(args...);
    return launched();
}

/* The serial kernel's pack: 16 bytes where these fill the GPU (500 x 1,024 f32, one
 * step: 3.6 us, in packs of 4 bytes 5.7), else 4 bytes (64 x 512 bf16: 2.2 us,
 * in packs of 16 bytes 2.6; 8 steps 4.1 and 6.3). */
int serial_pack(const ForwardArgs &p, size_t size) {
    const RecurrenceShape &d = p.d;
    const size_t all = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.rec) |
                       reinterpret_cast<uintptr_t>(p.inp) | reinterpret_cast<uintptr_t>(p.h) |
                       (d.is | d.it | d.os | d.ot | d.channels) * size;
    const int pack = pack_of(all, size);
    const bool full = d.sequences * d.channels / pack >= kSms * 128;
    return pack * size == 16 && !full ? 4 / static_cast<int>(size) : pack;
}
/* Few steps, or threads that are enough: 1,000 x 100 x 321 f32 140 us, by spans
 * 204, 4,096 x 64 x 512 bf16 230 and 264, 600 x 100 x 320 (24,000 threads) 46
 * both; fewer where spans load element by element: 64 x 1,024 x 1,023 bf16 396
 * and 551, 20 x 300 x 1,023 98 and 76. */
bool goes_serial(const RecurrenceShape &d, size_t bytes, size_t threads) {
    return d.steps <= kFewSteps || threads >= kSms * (bytes == 2 ? 256 : 512);
}
template <class T> int launch_serial(const ForwardArgs &p, int pack, cudaStream_t st) {
    const RecurrenceShape &d = p.d;
    const auto bits = [](const void *a) { return reinterpret_cast<uintptr_t>(a); };
    const bool quads = (bits(p.decay) | bits(p.state_in) | bits(p.state_out) | bits(p.checkpoints) | d.channels * 4) % 16 == 0;
    return with_pack<T>(pack, [&](auto n) {
        constexpr int PACK = decltype(n)::value;
        const size_t packs = d.channels / PACK;
        const size_t fill = (kSms * 2048 + packs - 1) / packs, rows = d.sequences < fill ? d.sequences : fill;
        const unsigned grid = static_cast<unsigned>((packs * rows + kSerialThreads - 1) / kSerialThreads);
        const unsigned a = static_cast<unsigned>(packs), b = static_cast<unsigned>(rows);
        const auto launch = [&](auto wide, auto together) {
            recurrence_serial<T, PACK, decltype(wide)::value, decltype(together)::value>
                <<<grid, kSerialThreads, 0, st>>>(p, a, b);
            return launched();
        };
        /* 500 x 16 x 1,023 bf16 33 us by fours, by twos 40; 1,024 x 128 x 1,024
         * 233 and 268; one step 6.0 and 5.7; f32 500 x 100 x 1,024 147 and 131 */
        const auto choose = [&](auto wide) {
            if constexpr (PACK == 1 || sizeof(T) == 2) {
                if (d.steps > (PACK == 1 ? 2 : kSteps)) return launch(wide, std::integral_constant<int, 4>{});
            }
            return launch(wide, std::integral_constant<int, 2>{});
        };
        if constexpr (PACK % 4 == 0) {
            if (quads) return choose(std::true_type{});
        }
        return choose(std::false_type{});
    });
}

} /* namespace */

extern "C" size_t tb_cuda_gated_recurrence_workspace(const tb_gated_recurrence_desc *desc) {
    RecurrenceShape s;
    if (!recurrence_shape(desc, &s)) return 0;
    int warps;
    const Pass forward = forward_pass(desc->type), backward = backward_pass(desc->type);
    const Split a = split_of(s, forward, &warps), b = split_of(s, backward, &warps);
    const size_t f = map_bytes(a, forward.tile) + first_bytes(s, a);
    const size_t back = map_bytes(b, backward.tile) + partial_bytes(s, b) + first_bytes(s, b);
    return f > back ? f : back;
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
        !aligned(checkpoints, 4) || !aligned(workspace, 16) ||
        collide({h, state_out, checkpoints, workspace}, {x, recurrence_gate, input_gate, decay, reset, lengths}) ||
        collide({h, checkpoints, workspace}, {state_in}))
        return 0;
    cudaGetLastError(); /* report these launches only */
    ForwardArgs p{s, x, recurrence_gate, input_gate, decay, state_in, reset, lengths, h, state_out, checkpoints, 0, 0};
    const int serial = serial_pack(p, size);
    if (goes_serial(s, serial * size, s.sequences * s.channels / serial))
        return with_type(desc->type, [&](auto t) {
            return launch_serial<decltype(t)>(p, serial, static_cast<cudaStream_t>(stream));
        });
    const uintptr_t in = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(recurrence_gate) |
                         reinterpret_cast<uintptr_t>(input_gate);
    p.in_piece = piece_of(reinterpret_cast<const void *>(in), s.is, s.it, size, 4);
    p.out_piece = piece_of(h, s.os, s.ot, size, 16);
    int warps;
    const Pass pass = forward_pass(desc->type);
    Split split = split_of(s, pass, &warps);
    split.maps = static_cast<float *>(workspace);
    if (split.strips > 1 && state_in && state_in == state_out)
        split.first = split.maps + map_bytes(split, pass.tile) / sizeof(float);
    const size_t shared = static_cast<size_t>(warps) * 2 * 3 * pass.span * pass.tile * size + kBoxAlign;
    return with_type(desc->type, [&](auto t) {
        using T = decltype(t);
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (split.strips > 1 && !launch_units<recurrence_forward_maps<T>>(split.tiles * (split.strips - 1), pass, warps,
                                                                          shared, st, p, split))
            return 0;
        if (split.first) p.state_in = split.first;
        const unsigned units = split.tiles * split.strips;
        if (split.strip_rounds < kBulkRounds)
            return launch_units<recurrence_forward<T, false>>(units, pass, warps, shared, st, p, split, NoMaps{});
        Maps maps{};
        if (p.in_piece == 16 && p.out_piece == 16 &&
            (maps.status = tb_status_slot(stream)) && encode(&maps.in[0], &maps.inner[0], desc->type, x, s, s.is, s.it, pass) &&
            encode(&maps.in[1], &maps.inner[0], desc->type, recurrence_gate, s, s.is, s.it, pass) &&
            encode(&maps.in[2], &maps.inner[0], desc->type, input_gate, s, s.is, s.it, pass) &&
            encode(&maps.out[0], &maps.inner[2], desc->type, h, s, s.os, s.ot, pass))
            return launch_units<recurrence_forward<T, true>>(units, pass, warps, shared, st, p, split, maps);
        return launch_units<recurrence_forward<T, false>>(units, pass, warps, shared, st, p, split, NoMaps{});
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
        !aligned(ddecay, 4) || !aligned(dstate_in, 4) || !aligned(workspace, 16) ||
        collide({dx, drecurrence_gate, dinput_gate, ddecay, dstate_in, workspace},
                {x, recurrence_gate, input_gate, decay, reset, lengths, checkpoints, dh}) ||
        collide({dx, drecurrence_gate, dinput_gate, ddecay, workspace}, {dstate_out}))
        return 0;
    const void *in[] = {x, recurrence_gate, input_gate, dh}, *out[] = {dx, drecurrence_gate, dinput_gate};
    uintptr_t ins = 0, outs = 0;
    for (int i = 0; i < 3; ++i) {
        ins |= reinterpret_cast<uintptr_t>(in[i]);
        outs |= reinterpret_cast<uintptr_t>(out[i]);
    }
    cudaGetLastError(); /* report these launches only */
    int warps;
    const Pass pass = backward_pass(desc->type);
    Split split = split_of(s, pass, &warps);
    split.maps = static_cast<float *>(workspace);
    float *partial = split.maps + map_bytes(split, pass.tile) / sizeof(float);
    if (split.strips > 1 && dstate_out && dstate_out == dstate_in)
        split.first = partial + partial_bytes(s, split) / sizeof(float);
    BackwardArgs p{s, x, recurrence_gate, input_gate, dh, decay, checkpoints, dstate_out, reset, lengths, dx,
                   drecurrence_gate, dinput_gate, ddecay ? partial : nullptr, dstate_in, 0, 0, 0};
    p.in_piece = piece_of(reinterpret_cast<const void *>(ins), s.is, s.it, size, 4);
    p.dh_piece = piece_of(dh, s.os, s.ot, size, 4);
    p.out_piece = piece_of(reinterpret_cast<const void *>(outs), s.gs, s.gt, size, 16);
    const size_t shared = static_cast<size_t>(warps) * 2 * 4 * pass.span * pass.tile * size + kBoxAlign;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int ok = with_type(desc->type, [&](auto t) {
        using T = decltype(t);
        if (split.strips > 1 && !launch_units<recurrence_backward_maps<T>>(split.tiles * (split.strips - 1), pass, warps,
                                                                           shared, st, p, split))
            return 0;
        if (split.first) p.dstate_out = split.first;
        const unsigned units = split.tiles * split.strips;
        Maps maps{};
        bool bulk = split.strip_rounds >= kBulkRounds && p.in_piece == 16 && p.dh_piece == 16 && p.out_piece == 16 &&
                    (maps.status = tb_status_slot(stream));
        for (int i = 0; i < 4 && bulk; ++i)
            bulk = encode(&maps.in[i], &maps.inner[i / 3], desc->type, in[i], s, i < 3 ? s.is : s.os, i < 3 ? s.it : s.ot, pass);
        for (int i = 0; i < 3 && bulk; ++i) bulk = encode(&maps.out[i], &maps.inner[2], desc->type, out[i], s, s.gs, s.gt, pass);
        return bulk ? launch_units<recurrence_backward<T, true>>(units, pass, warps, shared, st, p, split, maps)
                    : launch_units<recurrence_backward<T, false>>(units, pass, warps, shared, st, p, split, NoMaps{});
    });
    if (!ok || !ddecay) return ok;
    return sum_columns(partial, partial_rows(s, split), s.channels, DecayGradient{decay, s.scale, ddecay}, st);
}
