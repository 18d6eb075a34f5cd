/*
 * Products on the fifth-generation tensor cores (tcgen05), fed by bulk tensor
 * copies: what the learner's products share.
 *
 * Every product here is O[n, m] = sum_k B[n, k] A[m, k], m the contiguous
 * dimension of the output: 128 values of m are the tensor core's rows (TMEM
 * lanes), up to 256 of n its columns, so that a warp that reads a column of
 * the accumulator holds 32 neighbours of one row of O and stores them without
 * a transpose.  n may be ragged: a tile issues its instructions for as many
 * columns, to the next 16, as it has.  Either operand may lie with k
 * contiguous or with m (n) contiguous; the tensor cores take both.
 *
 * A CTA of six warps: one asks for the copies, one issues the products, four
 * read the accumulators.  A ring of 128-byte-deep stages (64 values of 16 bits,
 * 128 of 8) feeds the products; two accumulators of 256 columns let the
 * storing of one tile run under the products of the next.  CTAs are persistent
 * and take every gridDim-th tile of a job.
 *
 * A job says what its tiles are and stores them (struct Job: setup, tiles,
 * tile, store); operands of more than 16 bits come as planes that sum to them,
 * and a job lists the pairs of planes to multiply.
 *
 * Waits are bounded by a second; one that runs out reports
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

namespace tb_tensor {

using tb_pipe::mbar_arrive;
using tb_pipe::mbar_arrive_expect_tx;
using tb_pipe::mbar_init;
using tb_pipe::smem_addr;

constexpr int kTileM = 128;
constexpr int kBlockBytes = 128;             /* of k in a stage */
constexpr int kChunk = 64;                   /* 16-bit values of m (n) in a swizzled row, where those are contiguous */
constexpr int kChunkBytes = 64 * kBlockBytes; /* 64 such rows, one for each k of a stage */
constexpr int kThreads = 192;
constexpr int kStoreWarps = 4, kStoreThreads = 32 * kStoreWarps;
constexpr int kMaxPairs = 6;
constexpr int kColumns = 512; /* of TMEM: two accumulators of 256 */
constexpr unsigned long long kWaitNs = 1000000000ull;

/* ---- instructions ---- */

__device__ __forceinline__ void tmem_alloc(uint32_t result, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(result), "r"(columns) : "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t columns) {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns));
}
__device__ __forceinline__ void tensor_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tensor_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
/* `bar` completes a phase when the products issued so far by this thread are done. */
__device__ __forceinline__ void tensor_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
template <bool I8> __device__ __forceinline__ void tensor_product(uint32_t d, uint64_t a, uint64_t b, uint32_t how, bool add) {
    if constexpr (I8)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(how),
            "r"(static_cast<uint32_t>(add))
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(how),
            "r"(static_cast<uint32_t>(add))
            : "memory");
}
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

__device__ __forceinline__ void load_box(uint32_t to, const CUtensorMap *map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(to), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
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
 * bits), their orders, columns; 128 rows, 32-bit accumulators. */
__device__ __forceinline__ uint32_t product_form(bool i8, int type, bool a_outer, bool b_outer, int columns) {
    return (i8 ? 2u : 1u) << 4 | static_cast<uint32_t>(type) << 7 | static_cast<uint32_t>(type) << 10 |
           static_cast<uint32_t>(a_outer) << 15 | static_cast<uint32_t>(b_outer) << 16 |
           static_cast<uint32_t>(columns / 8) << 17 | static_cast<uint32_t>(kTileM / 16) << 24;
}

/* ---- jobs ---- */

/* Both operands, 3-dimensional: {contiguous, other, z}; z counts planes and, in
 * them, matrices. */
struct Operands {
    CUtensorMap a, b;
    unsigned *status;
    int a_outer, b_outer;   /* m (n) contiguous instead of k */
    int type;               /* 0 f16, 1 bf16, 1 signed 8 bits */
    int pairs;              /* of planes, in the order of their sum */
    int a_plane[kMaxPairs], b_plane[kMaxPairs]; /* z of each pair's planes, to be added to a tile's */
};

/* k in [k0, k0 + depth) of rows m0.. of A's matrix az and n0.. (columns of
 * them) of B's bz. */
struct Tile {
    int m0, n0, columns, k0, depth, az, bz;
    int which; /* the job's own */
};

/* ---- the kernel ---- */

template <int NT> struct Shape {
    static constexpr int kABytes = kTileM * kBlockBytes, kBBytes = NT * kBlockBytes, kStage = kABytes + kBBytes;
    static constexpr int kStages = 196608 / kStage > 12 ? 12 : 196608 / kStage;
    static constexpr int kShared = kStages * kStage + 1024; /* + alignment */
};

struct Waits {
    unsigned *status;
    volatile int *gave_up; /* in shared memory */
    __device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity) const {
        if (tb_pipe::mbar_try_wait(bar, parity)) return true;
        const unsigned long long t0 = tb_pipe::global_ns();
        for (;;) {
            for (int i = 0; i < 32; ++i)
                if (tb_pipe::mbar_try_wait(bar, parity)) return true;
            if (*gave_up) return false;
            if (tb_pipe::global_ns() - t0 > kWaitNs) break;
        }
        if (!*gave_up) atomicOr(status, TB_FEATURE_STATUS_WAIT_TIMEOUT);
        *gave_up = 1;
        return false;
    }
};

/* Rows of k at and past `from` of a stage's operand of `chunks` chunks (m or n
 * contiguous) become zero, up to the next 16; by a warp. */
__device__ __forceinline__ void clear_past(unsigned char *at, int chunks, int from, int lane) {
    const int rows = (from + 15) / 16 * 16 - from, words = rows * 8; /* of 16 bytes */
    for (int c = 0; c < chunks; ++c)
        for (int i = lane; i < words; i += 32)
            *reinterpret_cast<uint4 *>(at + c * kChunkBytes + from * kBlockBytes + i * 16) = uint4{0, 0, 0, 0};
}

template <class Job, int NT, bool I8>
__global__ void __launch_bounds__(kThreads, 1)
tensor_products(const __grid_constant__ Operands ops, const __grid_constant__ Job job) {
    using S = Shape<NT>;
    constexpr int kDepth = I8 ? 128 : 64, kStep = I8 ? 32 : 16; /* of k: in a stage, in an instruction */
    extern __shared__ unsigned char raw[];
    __shared__ uint64_t full[S::kStages], empty[S::kStages], done[2], freed[2];
    __shared__ uint32_t tmem_at;
    __shared__ int gave_up;
    __shared__ typename Job::Shared shared;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    unsigned char *stages = raw + ((1024 - (smem_addr(raw) & 1023)) & 1023);
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kStages; ++i) mbar_init(smem_addr(&full[i]), 1), mbar_init(smem_addr(&empty[i]), 1);
        for (int i = 0; i < 2; ++i) mbar_init(smem_addr(&done[i]), 1), mbar_init(smem_addr(&freed[i]), kStoreWarps);
        gave_up = 0;
        tb_pipe::fence_mbar_init();
    }
    if (warp == 1) tmem_alloc(smem_addr(&tmem_at), kColumns);
    tensor_fence_before();
    job.setup(shared);
    __syncthreads();
    tensor_fence_after();
    const uint32_t tmem = tmem_at;
    const Waits w{ops.status, &gave_up};
    const int tiles = job.tiles(shared);
    if (warp == 0) {
        if (lane == 0) {
            uint32_t n = 0; /* stages asked for */
            bool ok = true;
            for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
                const Tile tile = job.tile(shared, t);
                for (int p = 0; ok && p < ops.pairs; ++p) {
                    const int az = tile.az + ops.a_plane[p], bz = tile.bz + ops.b_plane[p];
                    for (int k = 0; k < tile.depth; k += kDepth, ++n) {
                        const int s = n % S::kStages;
                        if (n >= S::kStages && !(ok = w.wait(smem_addr(&empty[s]), (n / S::kStages - 1) & 1))) break;
                        const uint32_t bar = smem_addr(&full[s]), at = smem_addr(stages + s * S::kStage);
                        mbar_arrive_expect_tx(bar, S::kStage);
                        if (ops.a_outer) {
                            load_box(at, &ops.a, tile.m0, tile.k0 + k, az, bar);
                            load_box(at + kChunkBytes, &ops.a, tile.m0 + kChunk, tile.k0 + k, az, bar);
                        } else {
                            load_box(at, &ops.a, tile.k0 + k, tile.m0, az, bar);
                        }
                        if (ops.b_outer) {
#pragma unroll
                            for (int c = 0; c < (NT + kChunk - 1) / kChunk; ++c)
                                load_box(at + S::kABytes + c * kChunkBytes, &ops.b, tile.n0 + c * kChunk, tile.k0 + k, bz, bar);
                        } else {
                            load_box(at + S::kABytes, &ops.b, tile.k0 + k, tile.n0, bz, bar);
                        }
                    }
                }
            }
            /* copies land before the CTA leaves, also where the products gave up on them */
            for (uint32_t i = n > S::kStages ? n - S::kStages : 0; i < n; ++i)
                tb_pipe::mbar_wait(smem_addr(&full[i % S::kStages]), (i / S::kStages) & 1, kWaitNs);
        }
    } else if (warp == 1) {
        uint32_t n = 0, number = 0; /* stages taken, tiles */
        bool ok = true;
        for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x, ++number) {
            const Tile tile = job.tile(shared, t);
            const uint32_t buffer = number & 1, d = tmem + buffer * 256;
            if (number >= 2 && !(ok = w.wait(smem_addr(&freed[buffer]), (number / 2 - 1) & 1))) break;
            tensor_fence_after();
            const uint32_t how = product_form(I8, ops.type, ops.a_outer, ops.b_outer, (tile.columns + 15) / 16 * 16);
            for (int p = 0; ok && p < ops.pairs; ++p)
                for (int k = 0; k < tile.depth; k += kDepth, ++n) {
                    const int s = n % S::kStages, left = tile.depth - k;
                    if (!(ok = w.wait(smem_addr(&full[s]), (n / S::kStages) & 1))) break;
                    unsigned char *at = stages + s * S::kStage;
                    if (Job::kRagged && left < kDepth && left % kStep) { /* what follows belongs to another matrix */
                        clear_past(at, kTileM / kChunk, left, lane);
                        clear_past(at + S::kABytes, (NT + kChunk - 1) / kChunk, left, lane);
                        tb_pipe::fence_proxy_async_shared();
                        __syncwarp();
                    }
                    tensor_fence_after();
                    if (lane == 0) {
                        const uint64_t a = operand(smem_addr(at), ops.a_outer), b = operand(smem_addr(at + S::kABytes), ops.b_outer);
                        const int steps = min(kDepth, left + kStep - 1) / kStep;
                        const uint32_t ia = (ops.a_outer ? kStep * kBlockBytes : 32) >> 4, ib = (ops.b_outer ? kStep * kBlockBytes : 32) >> 4;
#pragma unroll
                        for (int i = 0; i < kDepth / kStep; ++i)
                            if (i < steps) tensor_product<I8>(d, a + i * ia, b + i * ib, how, p > 0 || k > 0 || i > 0);
                        tensor_commit(smem_addr(&empty[s]));
                    }
                    __syncwarp();
                }
            if (lane == 0) tensor_commit(smem_addr(&done[buffer]));
            __syncwarp();
        }
        /* products end before the TMEM is freed, also where the storing warps gave up on them */
        if (n > 0) tb_pipe::mbar_wait(smem_addr(&empty[(n - 1) % S::kStages]), ((n - 1) / S::kStages) & 1, kWaitNs);
    } else {
        const int part = warp % 4; /* the lanes of TMEM that this warp may read */
        uint32_t number = 0;
        for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++number) {
            const Tile tile = job.tile(shared, t);
            const uint32_t buffer = number & 1;
            if (!w.wait(smem_addr(&done[buffer]), (number / 2) & 1)) break;
            tensor_fence_after();
            const int m = tile.m0 + part * 32 + lane;
            for (int c = 0; c < tile.columns; c += 32) {
                uint32_t r[32];
                if (tile.depth > 0) {
                    tensor_load(tmem + buffer * 256 + (static_cast<uint32_t>(part) << 21) + c, r);
                    tensor_wait_load();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) r[i] = 0;
                }
                job.store(shared, tile, m, c, r);
            }
            tensor_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_addr(&freed[buffer]));
        }
    }
    __syncwarp();
    tensor_fence_before();
    __syncthreads();
    tensor_fence_after();
    if (warp == 1) tmem_free(tmem, kColumns);
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

/* Boxes of 128 bytes by `box_rows`. */
inline bool encode(CUtensorMap *map, const Matrices &m, int box_rows) {
    const EncodeTiled f = encoder();
    const cuuint64_t extent[3] = {m.width, m.rows, m.count};
    const cuuint64_t stride[2] = {m.row_stride * m.size, (m.count > 1 ? m.matrix_stride : m.row_stride) * m.size};
    const cuuint32_t box[3] = {static_cast<cuuint32_t>(kBlockBytes / m.size), static_cast<cuuint32_t>(box_rows), 1};
    const cuuint32_t one[3] = {1, 1, 1};
    return f && f(map, m.size == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 3,
                  const_cast<void *>(m.at), extent, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
/* Both operands' maps for tiles of `columns` of n (64 at least where n is contiguous in b). */
inline bool encode(Operands *ops, const Matrices &a, bool a_outer, const Matrices &b, bool b_outer, int columns) {
    ops->a_outer = a_outer;
    ops->b_outer = b_outer;
    if (b_outer && columns < kChunk) return false;
    return encode(&ops->a, a, a_outer ? kChunk : kTileM) && encode(&ops->b, b, b_outer ? kChunk : columns);
}

template <class Job, int NT, bool I8>
int launch_products(const Operands &ops, const Job &job, size_t most_tiles, int sms, cudaStream_t st) {
    if (!tb_learn::allow_shared<tensor_products<Job, NT, I8>>(Shape<NT>::kShared)) return 0;
    const unsigned grid = static_cast<unsigned>(most_tiles < static_cast<size_t>(sms) ? most_tiles : sms);
    tensor_products<Job, NT, I8><<<grid, kThreads, Shape<NT>::kShared, st>>>(ops, job);
    return tb_learn::launched();
}

} /* namespace tb_tensor */

#endif
