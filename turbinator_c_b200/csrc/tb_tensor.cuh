/*
 * Products on the fifth-generation tensor cores (tcgen05), fed by bulk tensor
 * copies: what the learner's products share.
 *
 * Every product here is O[n, m] = sum_k B[n, k] A[m, k], m the contiguous
 * dimension of the output: 128 values of m are the tensor core's rows (TMEM
 * lanes), up to 256 of n its columns, so that a warp that reads a column of
 * the accumulator holds 32 neighbours of one row of O and stores them without
 * a transpose.  n may be ragged: a tile issues its instructions for as many
 * columns, to the next 16 (32), as it has (tb_product_columns.h).  Either operand may lie with k
 * contiguous or with m (n) contiguous; the tensor cores take both.
 *
 * One warp of a CTA asks for the copies, one issues the products, eight or
 * sixteen read the accumulators.  A ring of 128-byte-deep stages (64 values of 16 bits,
 * 128 of 8) feeds the products; two accumulators of 256 columns let the
 * storing of one tile run under the products of the next.  Two CTAs on
 * neighbouring SMs share a tile of 256 m where there are as many (PAIR): each
 * brings its 128 rows of A and half of B's, so that a product's 128 x 256 x 64
 * take 32 KB from L2 and not 48 (L2 gives some 45 to 51 bytes a cycle and SM):
 * 131,072 rows x 1,024 x 2,048 bf16 425 us, 519 without pairs, 581 in tiles of
 * 128 x 128.  A library's product of as many equal runs takes 421 us in short
 * runs as this one does.  Over seconds the power cap decides: 508 us here, in 0.53
 * million cycles at 1,050 MHz, 477 there, in 0.66 at 1,387.  Tiles of 256 x 512,
 * whose products run without a pause, took as long at a lower clock.
 * CTAs (pairs) are persistent and take every so-many-th tile of a job.
 *
 * Operands of more than 16 bits come as planes that sum to them, each held
 * 2^kPlaneRise higher than the one in front of it, so that its values are as far
 * from the type's least ones; a stage holds all planes, and the pairs of planes
 * whose product counts are multiplied one after the other, small ones first.  The
 * instruction with which a larger kind of pair begins takes what the smaller ones
 * left 2^kPlaneRise lower.  Their sums are taken out of the tensor
 * cores after every stage and go on in f32 registers: the tensor cores' own
 * additions cut what does not fit, which over thousands of k left errors of 4e-6
 * to 2e-5 in results that f32 arithmetic has to 1e-6.  Every second stage would
 * take 0 to 3 % less time, at errors of 6e-7 for 1e-7 (f32 products) and 1.7e-6 for
 * 1.0e-6 (updates).
 *
 * Where tiles are few and k is long, a tile's k is cut into parts of whole
 * stages: each writes its sums to a workspace, and a second kernel adds them in
 * order.
 *
 * A job says what its tiles are and stores them (struct Job: setup, tiles,
 * tile, store: eight columns of a row of the tensor core's; or, where kStaging
 * is not 0, 32 columns of 32 rows by a warp with so many bytes of its own, into
 * which ask has asked for what it reads for them).
 *
 * Waits are bounded by a second (a tile's sums by 10 us a stage more); one that runs out reports
 * TB_FEATURE_STATUS_WAIT_TIMEOUT through the stream's status word, after which
 * every warp goes to its end: no further copies or products are asked for,
 * those under way are waited for (again with a bound) and the TMEM is freed.
 */
#ifndef TB_TENSOR_CUH
#define TB_TENSOR_CUH

#include <cuda.h>

#include "tb_features_internal.h"
#include "tb_learner.cuh"
#include "tb_pipeline.cuh"
#include "tb_product_columns.h"

namespace tb_tensor {

using tb_pipe::mbar_arrive;
using tb_pipe::mbar_arrive_expect_tx;
using tb_pipe::mbar_init;
using tb_pipe::smem_addr;

constexpr int kRows = 128;                    /* of m in a CTA's part of a tile */
constexpr int kBlockBytes = 128;              /* of k in a stage */
constexpr int kChunk = 64;                    /* 16-bit values of m (n) in a swizzled row, where those are contiguous */
constexpr int kChunkBytes = 64 * kBlockBytes; /* 64 such rows, one for each k of a stage */
constexpr int kColumns = 512; /* of TMEM: two accumulators of 256 */
/* How many powers of two a plane is held higher than the one in front of it.  Two f16: what the rounding of one leaves is
 * 2^-11 of it at most.  Three bf16: 2^-9 of it, or 2^-8 where the largest values are cut; seven, so that nothing passes
 * f32's range that did not before. */
template <int PLANES> constexpr int kPlaneRise = PLANES == 3 ? 7 : PLANES == 2 ? 11 : 0;
constexpr unsigned long long kWaitNs = 1000000000ull;

/* ---- instructions ---- */

/* One lane of a whole warp, the same each time.  The compiler knows that it is
 * one, and issues copies and products without a loop over lanes: with `lane ==
 * 0` in its place four products took 394 cycles to issue. */
__device__ __forceinline__ bool elected() {
    uint32_t yes;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
    return yes != 0;
}

template <bool PAIR> __device__ __forceinline__ void tmem_alloc(uint32_t result, uint32_t columns) {
    if constexpr (PAIR)
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(result), "r"(columns) : "memory");
    else
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(result), "r"(columns) : "memory");
}
template <bool PAIR> __device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t columns) {
    if constexpr (PAIR) {
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns));
    } else {
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns));
    }
}
__device__ __forceinline__ void tensor_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tensor_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
/* `bar` (of both CTAs of a pair) completes a phase when the products issued so far by this thread are done. */
template <bool PAIR> __device__ __forceinline__ void tensor_commit(uint32_t bar) {
    if constexpr (PAIR)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
            "h"(static_cast<uint16_t>(3))
            : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
#define TB_TENSOR_PRODUCT(GROUP, KIND, LOWER, ...)                                                              \
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::" GROUP ".kind::" KIND \
                 " [%0], %1, %2, %3, p" LOWER ";\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(how), "r"(static_cast<uint32_t>(add)), ##__VA_ARGS__ \
                 : "memory")
/* LOWER: what is in d already counts 2^-LOWER of itself. */
template <bool I8, bool PAIR, int LOWER = 0>
__device__ __forceinline__ void tensor_product(uint32_t d, uint64_t a, uint64_t b, uint32_t how, bool add) {
    static_assert(LOWER >= 0 && LOWER <= 15 && (!I8 || LOWER == 0), "what the instruction takes");
    if constexpr (I8 && PAIR) TB_TENSOR_PRODUCT("2", "i8", "");
    else if constexpr (I8) TB_TENSOR_PRODUCT("1", "i8", "");
    else if constexpr (PAIR && LOWER != 0) TB_TENSOR_PRODUCT("2", "f16", ", %5", "n"(LOWER));
    else if constexpr (PAIR) TB_TENSOR_PRODUCT("2", "f16", "");
    else if constexpr (LOWER != 0) TB_TENSOR_PRODUCT("1", "f16", ", %5", "n"(LOWER));
    else TB_TENSOR_PRODUCT("1", "f16", "");
}
#undef TB_TENSOR_PRODUCT
/* 32 columns of this warp's 32 lanes; tensor_wait_load() before the values are used. */
__device__ __forceinline__ void tensor_load(uint32_t tmem, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(tmem));
}
__device__ __forceinline__ void tensor_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

/* `bar` lies in this CTA, or (PAIR) in either of the two. */
template <bool PAIR>
__device__ __forceinline__ void load_box(uint32_t to, const CUtensorMap *map, int x, int y, int z, uint32_t bar) {
    if constexpr (PAIR)
        asm volatile(
            "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
            "[%1, {%2, %3, %4}], [%5];" ::"r"(to), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
            ::"r"(to), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
            : "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

/* ---- the other CTA of a pair ---- */

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
/* Where the first CTA of the pair has what lies at `at` here. */
__device__ __forceinline__ uint32_t in_first(uint32_t at) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(at));
    return r;
}
/* Relaxed: they publish nothing, and a release waits for this thread's stores
 * and copies, a microsecond each. */
__device__ __forceinline__ void remote_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
/* What this warp has written to its shared memory is there for the products. */
__device__ __forceinline__ void remote_arrive_written(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void remote_arrive_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.relaxed.cluster.shared::cluster.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

/* An operand in shared memory, rows of 128 bytes in the 128-byte swizzle.
 * Contiguous in k: a row per m, eight rows 1,024 bytes apart.  Contiguous in m:
 * a row of 64 per k, eight of k 1,024 bytes apart, the next 64 of m a chunk on. */
__device__ __forceinline__ uint64_t operand(uint32_t at, bool outer_contiguous) {
    return static_cast<uint64_t>((at >> 4) & 0x3fff) |
           (static_cast<uint64_t>(outer_contiguous ? kChunkBytes >> 4 : 1) << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
/* How the products are taken: type of the operands (0 f16, 1 bf16; 1 signed 8
 * bits), their orders, rows and columns; 32-bit accumulators. */
__device__ __forceinline__ uint32_t product_form(bool i8, int type, bool a_outer, bool b_outer, int rows, int columns) {
    return (i8 ? 2u : 1u) << 4 | static_cast<uint32_t>(type) << 7 | static_cast<uint32_t>(type) << 10 |
           static_cast<uint32_t>(a_outer) << 15 | static_cast<uint32_t>(b_outer) << 16 |
           static_cast<uint32_t>(columns / 8) << 17 | static_cast<uint32_t>(rows / 16) << 24;
}

/* ---- jobs ---- */

/* Both operands, 3-dimensional: {contiguous, other, z}; z counts planes and, in
 * them, matrices. */
struct Operands {
    CUtensorMap a, b;
    unsigned *status;
    int a_outer, b_outer; /* m (n) contiguous instead of k */
    int type;             /* 0 f16, 1 bf16, 1 signed 8 bits */
    int a_plane, b_plane; /* z of the second plane */
    int parts;            /* of a tile's k */
    uint32_t *sums;       /* of the parts, if there are several: [tile][part][column][m] */
};

/* k in [k0, k0 + depth) of rows m0.. of A's matrix az and n0.. (columns of
 * them) of B's bz. */
struct Tile {
    int m0, n0, columns, k0, depth, az, bz;
    int which; /* the job's own */
};
/* A part of a tile's k: whole stages but for the last. */
__device__ __forceinline__ Tile part_of(Tile t, int part, int parts, int stage) {
    const int per = ((t.depth + stage - 1) / stage + parts - 1) / parts * stage;
    const int first = min(part * per, t.depth);
    t.k0 += first;
    t.depth = min(per, t.depth - first);
    return t;
}

/* ---- the kernel ---- */

template <int NT, int PLANES, bool PAIR, int STAGING = 0> struct Shape {
    static constexpr int kTileM = PAIR ? 2 * kRows : kRows;
    static constexpr int kPart = PAIR ? NT / 2 : NT; /* rows of B that a CTA brings */
    static constexpr int kABytes = kRows * kBlockBytes, kBBytes = kPart * kBlockBytes; /* of a block: 128 bytes of k */
    /* Blocks of k in a stage: two of a single plane, so that a stage's waits and its commit, some 250 cycles to issue,
     * come with eight products of 128 cycles and not four. */
    static constexpr int kBlocks = PLANES == 1 ? 2 : 1;
    static constexpr int kStage = kBlocks * PLANES * (kABytes + kBBytes);
    static constexpr int kStages = 196608 / kStage > 12 ? 12 : 196608 / kStage;
    /* Sums of 256 columns in registers: 128 each of eight warps, which take the registers that the others leave (216 and
     * 72 of 168 each); in sixteen warps of 96 registers the sums spilled and a tile's storing took four times as long. */
    static constexpr bool kWide = PLANES > 1 && NT == 256;
    static constexpr int kShare = kWide ? 128 : NT >= 128 ? 64 : 32; /* columns that a storing warp reads */
    static constexpr int kFirstStore = kWide ? 4 : 2, kStoreWarps = 4 * (NT / kShare);
    static constexpr int kThreads = 32 * (kFirstStore + kStoreWarps);
    static constexpr int kShared = kStages * kStage + kStoreWarps * STAGING + 1024; /* + alignment */
    static constexpr int kLaunchRegisters = 168, kStoreRegisters = 216, kOtherRegisters = 72;
    static_assert(!kWide || kThreads * kLaunchRegisters == 32 * (kStoreWarps * kStoreRegisters + 4 * kOtherRegisters), "a split");
    static_assert(kStages >= 2, "a ring");
    static_assert(NT % 32 == 0 && NT <= kMostColumns, "whole tiles are issued as they are");
};

struct Waits {
    unsigned *status;
    volatile int *gave_up; /* in shared memory */
    /* stages: of work in front of what is waited for, some microseconds each at most. */
    __device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, int stages = 0) const {
        /* the clock is read late: reading it takes longer than most waits */
        unsigned long long t0 = 0;
        for (;;) {
            for (int i = 0; i < 256; ++i)
                if (tb_pipe::mbar_try_wait(bar, parity)) return true;
            if (*gave_up) return false;
            const unsigned long long now = tb_pipe::global_ns();
            if (t0 == 0) t0 = now;
            else if (now - t0 > kWaitNs + stages * 10000ull) break;
        }
        if (!*gave_up) atomicOr(status, TB_FEATURE_STATUS_WAIT_TIMEOUT);
        *gave_up = 1;
        return false;
    }
};

/* A storing warp's own shared memory, which bulk tensor copies fill and empty. */
struct Staging {
    unsigned char *at;
    uint32_t bar, phase;
    int lane;
    const Waits *w;
    bool under_way;
    /* What was put in has been read. */
    __device__ __forceinline__ void free() const {
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
    }
    __device__ __forceinline__ void stored() const {
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    /* Asks for boxes of `bytes` of planes z and z + next. */
    __device__ __forceinline__ void load(const CUtensorMap *map, int x, int y, int z, int next, int bytes) {
        free();
        if (lane == 0) {
            mbar_arrive_expect_tx(bar, 2 * bytes);
            load_box<false>(smem_addr(at), map, x, y, z, bar);
            load_box<false>(smem_addr(at) + bytes, map, x, y, z + next, bar);
        }
        under_way = true;
    }
    /* They are there; false where the wait for them ran out. */
    __device__ __forceinline__ bool loaded() {
        if (!under_way) return true;
        const bool ok = w->wait(bar, phase);
        if (!ok) tb_pipe::mbar_wait(bar, phase, kWaitNs); /* they land all the same */
        phase ^= 1;
        under_way = false;
        return ok;
    }
    /* The same out of shared memory, as this warp has written it. */
    __device__ __forceinline__ void store(const CUtensorMap *map, int x, int y, int z, int next, int bytes) const {
        tb_pipe::fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) {
            for (int p = 0; p < 2; ++p)
                asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map),
                             "r"(x), "r"(y), "r"(z + p * next), "r"(smem_addr(at) + p * bytes)
                             : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
    }
};

/* Rows of k at and past `from` of a block's chunks (m or n contiguous) become
 * zero, up to the next 16; by a warp. */
__device__ __forceinline__ void clear_past(unsigned char *at, int chunks, int from, int lane) {
    const int rows = (from + 15) / 16 * 16 - from, words = rows * 8; /* of 16 bytes */
    for (int c = 0; c < chunks; ++c)
        for (int i = lane; i < words; i += 32)
            *reinterpret_cast<uint4 *>(at + c * kChunkBytes + from * kBlockBytes + i * 16) = uint4{0, 0, 0, 0};
    tb_pipe::fence_proxy_async_shared();
    __syncwarp();
}

template <class Job, int NT, int PLANES, bool I8, bool PAIR>
__global__ void __launch_bounds__(Shape<NT, PLANES, PAIR>::kThreads, 1)
tensor_products(const __grid_constant__ Operands ops, const __grid_constant__ Job job) {
    using S = Shape<NT, PLANES, PAIR, Job::kStaging>;
    constexpr int kBlock = I8 ? 128 : 64, kStep = I8 ? 32 : 16; /* of k: in a block, in an instruction */
    constexpr int kDepth = S::kBlocks * kBlock;                 /* in a stage */
    constexpr int kParts = S::kBlocks * PLANES;
    constexpr bool kSums = PLANES > 1;                          /* of stages, in registers */
    constexpr int kRise = kPlaneRise<PLANES>;
    constexpr int kCtas = PAIR ? 2 : 1;
    constexpr int kBChunks = (S::kPart + kChunk - 1) / kChunk;
    extern __shared__ unsigned char raw[];
    __shared__ uint64_t full[S::kStages], empty[S::kStages], done[2], freed[2], tail[S::kStages];
    __shared__ uint32_t tmem_at;
    __shared__ int gave_up;
    __shared__ uint64_t staged[S::kStoreWarps];
    __shared__ typename Job::Shared shared;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    const uint32_t rank = PAIR ? cluster_rank() : 0;
    const bool first = rank == 0; /* the CTA whose warp issues the products */
    unsigned char *stages = raw + ((1024 - (smem_addr(raw) & 1023)) & 1023);
    if (threadIdx.x == 0) {
        prefetch_map(&ops.a);
        prefetch_map(&ops.b);
        for (int i = 0; i < S::kStages; ++i) {
            mbar_init(smem_addr(&full[i]), kCtas);
            mbar_init(smem_addr(&empty[i]), 1);
            mbar_init(smem_addr(&tail[i]), 1);
        }
        for (int i = 0; i < 2; ++i) mbar_init(smem_addr(&done[i]), 1), mbar_init(smem_addr(&freed[i]), kCtas * S::kStoreWarps);
        if (Job::kStaging)
            for (int i = 0; i < S::kStoreWarps; ++i) mbar_init(smem_addr(&staged[i]), 1);
        gave_up = 0;
        tb_pipe::fence_mbar_init();
    }
    if (warp == 1) tmem_alloc<PAIR>(smem_addr(&tmem_at), kColumns);
    tensor_fence_before();
    tb_learn::later_may_start();
    tb_learn::after_earlier();
    job.setup(shared);
    __syncwarp();
    if constexpr (PAIR) cluster_sync();
    else __syncthreads();
    tensor_fence_after();
    const uint32_t tmem = tmem_at;
    const Waits w{ops.status, &gave_up};
    const int tiles = job.tiles(shared) * ops.parts, start = blockIdx.x / kCtas, stride = gridDim.x / kCtas;
    const auto tile_at = [&](int t) {
        if (ops.parts == 1) return job.tile(shared, t);
        return part_of(job.tile(shared, t / ops.parts), t % ops.parts, ops.parts, kDepth);
    };
    /* Whether a stage's last rows of k belong to another matrix. */
    const auto ends_inside = [&](int left) { return Job::kRagged && left < kDepth && left % kStep != 0; };
    /* Those rows, in the block that they lie in; by a warp. */
    const auto clear_end = [&](unsigned char *at, int left) {
        static_assert(S::kBlocks == 1 || PLANES == 1, "blocks of one plane, or planes of one block");
        const int block = S::kBlocks > 1 ? left / kBlock : 0, from = left - block * kBlock, n = kParts / S::kBlocks;
        clear_past(at + block * S::kABytes, n * (kRows / kChunk), from, lane);
        clear_past(at + kParts * S::kABytes + block * S::kBBytes, n * kBChunks, from, lane);
    };
    if (warp < S::kFirstStore) {
        if constexpr (S::kWide) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kOtherRegisters));
        if (warp == 0) {
            uint32_t n = 0; /* stages asked for */
            bool ok = true;
            for (int t = start; ok && t < tiles; t += stride) {
                const Tile tile = tile_at(t);
                const int m0 = tile.m0 + static_cast<int>(rank) * kRows;
                const int n0 = tile.n0 + static_cast<int>(rank) * second_half(I8, tile.columns);
                for (int k = 0; k < tile.depth; k += kDepth, ++n) {
                    const int s = n % S::kStages;
                    if (n >= S::kStages && !(ok = w.wait(smem_addr(&empty[s]), (n / S::kStages - 1) & 1))) break;
                    if (elected()) {
                        uint32_t bar = smem_addr(&full[s]), at = smem_addr(stages + s * S::kStage);
                        if (PAIR && !first) {
                            if (ends_inside(tile.depth - k)) { /* this CTA clears its own rows, and then says so */
                                bar = smem_addr(&tail[s]);
                                mbar_arrive_expect_tx(bar, S::kStage);
                            } else {
                                bar = in_first(bar);
                                remote_arrive_expect_tx(bar, S::kStage);
                            }
                        } else {
                            mbar_arrive_expect_tx(bar, S::kStage);
                        }
#pragma unroll
                        for (int p = 0; p < kParts; ++p, at += S::kABytes) {
                            const int z = tile.az + (p % PLANES) * ops.a_plane, at_k = tile.k0 + k + p / PLANES * kBlock;
                            if (ops.a_outer) {
                                load_box<PAIR>(at, &ops.a, m0, at_k, z, bar);
                                load_box<PAIR>(at + kChunkBytes, &ops.a, m0 + kChunk, at_k, z, bar);
                            } else {
                                load_box<PAIR>(at, &ops.a, at_k, m0, z, bar);
                            }
                        }
#pragma unroll
                        for (int p = 0; p < kParts; ++p, at += S::kBBytes) {
                            const int z = tile.bz + (p % PLANES) * ops.b_plane, at_k = tile.k0 + k + p / PLANES * kBlock;
                            if (ops.b_outer) {
#pragma unroll
                                for (int c = 0; c < kBChunks; ++c)
                                    load_box<PAIR>(at + c * kChunkBytes, &ops.b, n0 + c * kChunk, at_k, z, bar);
                            } else {
                                load_box<PAIR>(at, &ops.b, at_k, n0, z, bar);
                            }
                        }
                    }
                    __syncwarp();
                }
            }
            /* copies land before the CTA leaves, also where the products gave up on them (a pair's
             * are all counted by its first CTA, and both leave together) */
            if (first)
                for (uint32_t i = n > S::kStages ? n - S::kStages : 0; i < n; ++i)
                    tb_pipe::mbar_wait(smem_addr(&full[i % S::kStages]), (i / S::kStages) & 1, kWaitNs);
        } else if (warp == 1 && first) {
            uint32_t n = 0, number = 0; /* stages taken, accumulators begun */
            bool ok = true;
            for (int t = start; ok && t < tiles; t += stride) {
                const Tile tile = tile_at(t);
                const uint32_t how = product_form(I8, ops.type, ops.a_outer, ops.b_outer, S::kTileM, issued_columns(I8, PAIR, tile.columns));
                uint32_t d = 0;
                for (int k = 0; ok && (k < tile.depth || k == 0); k += kDepth) {
                    if (k == 0 || kSums) { /* the next accumulator */
                        const uint32_t buffer = number & 1;
                        d = tmem + buffer * 256;
                        if (number >= 2 && !(ok = w.wait(smem_addr(&freed[buffer]), (number / 2 - 1) & 1))) break;
                        tensor_fence_after();
                        ++number;
                    }
                    const int s = n % S::kStages, left = tile.depth - k;
                    if (left > 0) {
                        if (!(ok = w.wait(smem_addr(&full[s]), (n / S::kStages) & 1))) break;
                        unsigned char *at = stages + s * S::kStage;
                        if (ends_inside(left)) clear_end(at, left);
                        tensor_fence_after();
                        if (elected()) {
                            const uint32_t ia = (ops.a_outer ? kStep * kBlockBytes : 32) >> 4, ib = (ops.b_outer ? kStep * kBlockBytes : 32) >> 4;
                            bool add = !kSums && k > 0;
                            const auto multiply = [&](int pa, int pb, int steps, auto lower) {
                                uint64_t a = operand(smem_addr(at + pa * S::kABytes), ops.a_outer);
                                uint64_t b = operand(smem_addr(at + kParts * S::kABytes + pb * S::kBBytes), ops.b_outer);
                                if (steps <= 0) return;
                                tensor_product<I8, PAIR, decltype(lower)::value>(d, a, b, how, add);
                                add = true;
                                if (steps >= kBlock / kStep) {
#pragma unroll
                                    for (int i = 1; i < kBlock / kStep; ++i) tensor_product<I8, PAIR>(d, a + i * ia, b + i * ib, how, true);
                                } else {
                                    for (int i = 1; i < steps; ++i) tensor_product<I8, PAIR>(d, a + i * ia, b + i * ib, how, true);
                                }
                            };
                            constexpr std::integral_constant<int, 0> kAsItIs{};
                            constexpr std::integral_constant<int, kRise> kLower{};
                            const int steps = (left + kStep - 1) / kStep;
                            if constexpr (PLANES == 1) {
#pragma unroll
                                for (int j = 0; j < S::kBlocks; ++j) multiply(j, j, steps - j * (kBlock / kStep), kAsItIs);
                            } else { /* planes i and j count while i + j < PLANES: the small products first */
#pragma unroll
                                for (int small = PLANES - 1; small >= 0; --small) {
                                    if (small == PLANES - 1) multiply(0, small, steps, kAsItIs);
                                    else multiply(0, small, steps, kLower);
#pragma unroll
                                    for (int p = 1; p <= small; ++p) multiply(p, small - p, steps, kAsItIs);
                                }
                            }
                            tensor_commit<PAIR>(smem_addr(&empty[s]));
                        }
                        __syncwarp();
                        ++n;
                    }
                    if (left <= kDepth || kSums) {
                        if (elected()) tensor_commit<PAIR>(smem_addr(&done[(number - 1) & 1]));
                        __syncwarp();
                    }
                }
            }
            /* products end before the TMEM is freed, also where the storing warps gave up on them */
            if (n > 0) tb_pipe::mbar_wait(smem_addr(&empty[(n - 1) % S::kStages]), ((n - 1) / S::kStages) & 1, kWaitNs);
        } else if (warp == 1) {
            if (Job::kRagged) { /* the second CTA's rows past a matrix's end, stage by stage as the first takes them */
                uint32_t n = 0, phases = 0; /* a bit for each stage */
                bool ok = true;
                for (int t = start; ok && t < tiles; t += stride) {
                    const Tile tile = tile_at(t);
                    for (int k = 0; k < tile.depth; k += kDepth, ++n) {
                        if (!ends_inside(tile.depth - k)) continue;
                        const int s = n % S::kStages;
                        if (!(ok = w.wait(smem_addr(&tail[s]), phases >> s & 1))) { /* the copies land all the same */
                            tb_pipe::mbar_wait(smem_addr(&tail[s]), phases >> s & 1, kWaitNs);
                            break;
                        }
                        phases ^= 1u << s;
                        unsigned char *at = stages + s * S::kStage;
                        clear_end(at, tile.depth - k);
                        if (lane == 0) remote_arrive_written(in_first(smem_addr(&full[s])));
                        __syncwarp();
                    }
                }
            }
        }
    } else {
        if constexpr (S::kWide) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kStoreRegisters));
        const int part = warp % 4, share = (warp - S::kFirstStore) / 4; /* the lanes of TMEM that this warp may read; its columns */
        const uint32_t lanes = static_cast<uint32_t>(part) << 21;
        uint32_t number = 0;
        bool ok = true;
        Staging staging{stages + S::kStages * S::kStage + (warp - S::kFirstStore) * Job::kStaging,
                        smem_addr(&staged[warp - S::kFirstStore]), 0, lane, &w, false};
        const auto free = [&](uint32_t buffer) {
            tensor_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR) remote_arrive(in_first(smem_addr(&freed[buffer])));
                else mbar_arrive(smem_addr(&freed[buffer]));
            }
        };
        for (int t = start; ok && t < tiles; t += stride) {
            const Tile tile = tile_at(t);
            const int m = tile.m0 + static_cast<int>(rank) * kRows + part * 32 + lane;
            [[maybe_unused]] const auto store = [&](int c, const uint32_t (&r)[8]) {
                if constexpr (Job::kStaging == 0) {
                    if (ops.parts == 1) {
                        job.store(shared, tile, m, c, r);
                    } else {
                        uint32_t *to = ops.sums + (static_cast<size_t>(t) * NT + c) * S::kTileM + (m - tile.m0);
#pragma unroll
                        for (int i = 0; i < 8; ++i) to[i * S::kTileM] = r[i];
                    }
                }
            };
            const int c0 = share * S::kShare, columns = min(tile.columns - c0, S::kShare);
            if constexpr (kSums) {
                float sum[S::kShare];
#pragma unroll
                for (int i = 0; i < S::kShare; ++i) sum[i] = 0.0f;
                if constexpr (Job::kStaging != 0)
                    if (columns > 0 && ops.parts == 1) job.ask(tile, m, c0, staging);
                for (int k = 0; ok && (k < tile.depth || k == 0); k += kDepth, ++number) {
                    const uint32_t buffer = number & 1;
                    if (!(ok = w.wait(smem_addr(&done[buffer]), (number / 2) & 1))) break;
                    tensor_fence_after();
                    if (tile.depth > 0) {
#pragma unroll
                        for (int c = 0; c < S::kShare; c += 32) { /* columns past the tile's are read too, and not stored */
                            uint32_t r[32];
                            tensor_load(tmem + buffer * 256 + lanes + c0 + c, r);
                            tensor_wait_load();
#pragma unroll
                            for (int i = 0; i < 32; ++i) sum[c + i] += __uint_as_float(r[i]);
                        }
                    }
                    free(buffer);
                }
                if (!ok) break;
                if constexpr (Job::kStaging != 0) {
#pragma unroll
                    for (int c = 0; c < S::kShare; c += 32)
                        if (ok && c < columns) {
                            float v[32];
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = sum[c + i];
                            if (ops.parts == 1) {
                                ok = job.store(tile, m, c0 + c, v, staging);
                                if (ok && c + 32 < columns) job.ask(tile, m, c0 + c + 32, staging);
                            } else {
                                uint32_t *to = ops.sums + (static_cast<size_t>(t) * NT + c0 + c) * S::kTileM + (m - tile.m0);
#pragma unroll
                                for (int i = 0; i < 32; ++i) to[i * S::kTileM] = __float_as_uint(v[i]);
                            }
                        }
                } else {
#pragma unroll
                    for (int c = 0; c < S::kShare; c += 8)
                        if (c < columns) {
                            uint32_t r[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(sum[c + i]);
                            store(c0 + c, r);
                            asm volatile("" ::: "memory"); /* the next eight's loads stay behind: they would take registers that the sums need */
                        }
                }
            } else {
                const uint32_t buffer = number & 1;
                if (!(ok = w.wait(smem_addr(&done[buffer]), (number / 2) & 1, tile.depth / kDepth))) break;
                tensor_fence_after();
                for (int c = 0; c < columns; c += 32) {
                    uint32_t r[32];
                    if (tile.depth > 0) {
                        tensor_load(tmem + buffer * 256 + lanes + c0 + c, r);
                        tensor_wait_load();
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) r[i] = 0;
                    }
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        uint32_t eight[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) eight[j] = r[i + j];
                        if (c + i < columns) store(c0 + c + i, eight);
                    }
                }
                free(buffer);
                ++number;
            }
        }
        if constexpr (Job::kStaging != 0) {
            staging.loaded();
            staging.stored();
        }
    }
    __syncwarp();
    tensor_fence_before();
    if constexpr (PAIR) cluster_sync();
    else __syncthreads();
    tensor_fence_after();
    if (warp == 1) tmem_free<PAIR>(tmem, kColumns);
}

/* The parts' sums, in order, and from there to where the job puts them: a CTA
 * eight columns of a tile, a thread an m. */
template <class Job, int NT, int TM, bool I8>
__global__ void __launch_bounds__(TM) join_parts(const __grid_constant__ Job job, int parts, const uint32_t *sums) {
    __shared__ typename Job::Shared shared;
    tb_learn::after_earlier();
    job.setup(shared);
    __syncthreads();
    const int t = blockIdx.x;
    if (t >= job.tiles(shared)) return;
    const Tile tile = job.tile(shared, t);
    const int c = blockIdx.y * 8;
    if (c >= tile.columns) return;
    const uint32_t *from = sums + (static_cast<size_t>(t) * parts * NT + c) * TM + threadIdx.x;
    constexpr int kAhead = 4; /* parts under way at once */
    uint32_t r[8] = {};
    for (int p = 0; p < parts; p += kAhead) {
        uint32_t v[kAhead][8];
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
            if (p + a < parts) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[a][i] = from[(static_cast<size_t>(p + a) * NT + i) * TM];
            }
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
            if (p + a < parts) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if constexpr (I8) r[i] += v[a][i];
                    else r[i] = __float_as_uint(__uint_as_float(r[i]) + __uint_as_float(v[a][i]));
                }
            }
    }
    if constexpr (Job::kStaging == 0) job.store(shared, tile, tile.m0 + threadIdx.x, c, r);
    else job.store_joined(tile, tile.m0 + threadIdx.x, c, r);
}

/* ---- host side ---- */

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeTiled encoder() {
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

/* A stack of `count` matrices [rows, width] of 16-bit values (or bytes), strides
 * in elements. */
struct Matrices {
    const void *at;
    size_t width, rows, count, row_stride, matrix_stride;
    size_t size; /* of an element: 1 or 2 */
    /* Whether bulk tensor copies may read it as it lies. */
    bool straight() const {
        return (reinterpret_cast<uintptr_t>(at) | row_stride * size | (count > 1 ? matrix_stride * size : 0)) % 16 == 0 &&
               row_stride * size < 1ull << 40 && (count == 1 || matrix_stride * size < 1ull << 40);
    }
};

/* Boxes of 128 bytes by `box_rows`, swizzled; or plain ones of box_width elements. */
inline bool encode(CUtensorMap *map, const Matrices &m, int box_rows, int box_width = 0) {
    const EncodeTiled f = encoder();
    const cuuint64_t extent[3] = {m.width, m.rows, m.count};
    const cuuint64_t stride[2] = {m.row_stride * m.size, (m.count > 1 ? m.matrix_stride : m.row_stride) * m.size};
    const cuuint32_t box[3] = {static_cast<cuuint32_t>(box_width ? box_width : kBlockBytes / m.size), static_cast<cuuint32_t>(box_rows), 1};
    const cuuint32_t one[3] = {1, 1, 1};
    return f && f(map, m.size == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 3,
                  const_cast<void *>(m.at), extent, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  box_width ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
/* Both operands' maps for tiles of NT columns (64 at least a CTA where n is contiguous in b). */
template <int NT, bool PAIR> bool encode(Operands *ops, const Matrices &a, bool a_outer, const Matrices &b, bool b_outer) {
    constexpr int kPart = PAIR ? NT / 2 : NT;
    ops->a_outer = a_outer;
    ops->b_outer = b_outer;
    return (!b_outer || kPart >= kChunk) && encode(&ops->a, a, a_outer ? kChunk : kRows) &&
           encode(&ops->b, b, b_outer ? kChunk : kPart);
}

/* ---- which tiles ---- */

struct Fit {
    int columns;
    bool pair;
    int parts;
    size_t tiles; /* at most, for the room of the parts' sums */
    size_t room() const { return parts > 1 ? tiles * parts * columns * (pair ? 2 * kRows : kRows) * sizeof(uint32_t) : 0; }
};
constexpr int kSms = 148; /* the fit is a shape's, whatever the device: a workspace is asked for without one */
constexpr size_t kMostRoom = 64u << 20;

/* The tiles, and parts of their k, that should be done first, in cycles: as many
 * as there are go round the SMs in so many turns; a block of k takes as long as
 * its products (two cycles a column, times the pairs of planes) or its copies
 * (some 46 bytes a cycle and SM); every turn some 2,000 for what is not hidden
 * of its beginning and end, 90 more for each of a storing warp's columns where
 * their sums leave no room for the next tile's, and parts a second kernel and their sums' way
 * through L2.  count(columns, m) says how many tiles of so many columns by m
 * there are likely to be, `average` how many columns one has of them, most(columns, m) how
 * many there may be; least: 64 where n is contiguous in b.
 * An update of 2 x 1,792 x 242 f32 takes 222 us in one part, 172 in several; one
 * of 2,501 x 1,537 the same either way. */
template <class Count, class Most>
Fit best_fit(int planes, int least, size_t average, size_t blocks, bool may_part, Count &&count, Most &&most) {
    Fit best{0, false, 1, 0};
    double lowest = 0.0;
    const auto consider = [&](int columns, bool pair) {
        const int m = pair ? 2 * kRows : kRows;
        const double units = pair ? kSms / 2 : kSms, tiles = static_cast<double>(count(columns, m));
        const double taken = average < static_cast<size_t>(columns) ? static_cast<double>(average) : columns;
        const double products = 2.0 * taken * (planes * (planes + 1) / 2);
        const double copies = planes * kBlockBytes * (kRows + columns / (pair ? 2.0 : 1.0)) / 46.0;
        const double block = products > copies ? products : copies;
        const double ends = 2000.0 + (planes > 1 ? 90.0 * (columns == 256 ? 128 : columns == 128 ? 64 : 32) : 0.0);
        for (int parts = 1; parts <= 64 && (parts == 1 || may_part); parts += parts < 4 ? 1 : parts / 2) {
            const size_t per = (blocks + parts - 1) / parts;
            if (parts > 1 && per < 4) break;
            const double turns = static_cast<double>(static_cast<size_t>((tiles * parts + units - 1) / units));
            double cost = turns * (per * block + ends);
            Fit fit{columns, pair, parts, most(columns, m)};
            if (parts > 1) cost += (planes > 1 ? 12000.0 : 8000.0) + tiles * parts * taken * m * 8.0 / (kSms * 20.0);
            if (fit.room() > kMostRoom) break;
            if (best.columns == 0 || cost < lowest) {
                lowest = cost;
                best = fit;
            }
        }
    };
    consider(256, true);
    if (planes == 1) consider(256, false);
    for (int columns = 128; columns >= least; columns /= 2) consider(columns, false);
    return best;
}
/* Calls f with the fit's columns and whether two CTAs share a tile, as constants. */
template <int PLANES, class F> int with_fit(Fit fit, F &&f) {
    if (fit.pair) return f(std::integral_constant<int, 256>{}, std::true_type{});
    if constexpr (PLANES == 1)
        if (fit.columns == 256) return f(std::integral_constant<int, 256>{}, std::false_type{});
    if (fit.columns == 128) return f(std::integral_constant<int, 128>{}, std::false_type{});
    if (fit.columns == 64) return f(std::integral_constant<int, 64>{}, std::false_type{});
    return f(std::integral_constant<int, 32>{}, std::false_type{});
}

/* tiles: at most. */
template <int NT, int PLANES, bool I8, bool PAIR, class Job>
int launch_products(const Operands &ops, const Job &job, size_t tiles, int sms, cudaStream_t st) {
    constexpr auto kernel = tensor_products<Job, NT, PLANES, I8, PAIR>;
    constexpr int kCtas = PAIR ? 2 : 1, kShared = Shape<NT, PLANES, PAIR, Job::kStaging>::kShared;
    if (!tb_learn::allow_shared<tensor_products<Job, NT, PLANES, I8, PAIR>>(kShared)) return 0;
    if constexpr (Shape<NT, PLANES, PAIR>::kWide) { /* warps that ask for more than the launch gave would wait forever */
        static std::atomic<int> registers{0};
        int n = registers.load(std::memory_order_relaxed);
        if (n == 0) {
            cudaFuncAttributes a;
            if (cudaFuncGetAttributes(&a, kernel) != cudaSuccess) return 0;
            registers.store(n = a.numRegs, std::memory_order_relaxed);
        }
        if (n < Shape<NT, PLANES, PAIR>::kLaunchRegisters) return 0;
    }
    const size_t most = static_cast<size_t>(sms) / kCtas, all = tiles * ops.parts;
    const unsigned grid = static_cast<unsigned>(all < most ? all : most) * kCtas;
    if (!tb_learn::launch_early(kernel, grid, Shape<NT, PLANES, PAIR>::kThreads, kShared, kCtas, st, ops, job)) return 0;
    if (ops.parts > 1) {
        constexpr int TM = Shape<NT, PLANES, PAIR>::kTileM;
        return tb_learn::launch_early(join_parts<Job, NT, TM, I8>, dim3(static_cast<unsigned>(tiles), NT / 8), TM, 0, 1, st, job,
                                      ops.parts, static_cast<const uint32_t *>(ops.sums));
    }
    return 1;
}

} /* namespace tb_tensor */

#endif
