/*
 * Shared by the learner kernels: element types, packs of elements that move in
 * one load or store, warp reductions, and the host-side checks of arguments.
 */
#ifndef TB_LEARNER_CUH
#define TB_LEARNER_CUH

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>
#include <string.h>

#include <atomic>
#include <type_traits>

#include "tb_shared_limit.h"
#include "turbinator/training/cuda_learner.h"

namespace tb_learn {

/* ---- element types ---- */

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

/* N consecutive elements moved by one load or store (N * sizeof(T) <= 16). */
template <class T, int N> struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

/* A pack as the words it came in, taken apart where it is used. */
template <class T, int N> struct alignas(sizeof(T) * N) Held {
    uint32_t w[N * sizeof(T) / 4];
};
template <> struct Held<__nv_bfloat16, 1> {
    uint16_t w[1];
};
template <> struct Held<__half, 1> {
    uint16_t w[1];
};
template <class T, int N> __device__ __forceinline__ void unpack(const Held<T, N> &h, float (&f)[N]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = __uint_as_float(h.w[i]);
    } else if constexpr (N == 1) {
        T v;
        memcpy(&v, h.w, 2);
        f[0] = to_float(v);
    } else {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            if constexpr (std::is_same<T, __half>::value) {
                const float2 t = __half22float2(*reinterpret_cast<const __half2 *>(&h.w[i]));
                f[2 * i] = t.x;
                f[2 * i + 1] = t.y;
            } else {
                f[2 * i] = __uint_as_float(h.w[i] << 16);
                f[2 * i + 1] = __uint_as_float(h.w[i] & 0xffff0000u);
            }
        }
    }
}
template <class T, int N> __device__ __forceinline__ Held<T, N> packed(const float (&f)[N]) {
    Held<T, N> h;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; ++i) h.w[i] = __float_as_uint(f[i]);
    } else if constexpr (N == 1) {
        const T v = from_float<T>(f[0]);
        memcpy(h.w, &v, 2);
    } else {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            if constexpr (std::is_same<T, __half>::value) {
                const __half2 t = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
                memcpy(&h.w[i], &t, 4);
            } else {
                const __nv_bfloat162 t = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
                memcpy(&h.w[i], &t, 4);
            }
        }
    }
    return h;
}

/* The same to and from global memory for what is used once: first to leave L2. */
template <class T, int N> __device__ __forceinline__ Held<T, N> load_once(const T *p) {
    Held<T, N> h;
    if constexpr (sizeof(h) == 16) {
        const uint4 v = __ldcs(reinterpret_cast<const uint4 *>(p));
        memcpy(&h, &v, 16);
    } else {
        h = *reinterpret_cast<const Held<T, N> *>(p);
    }
    return h;
}
template <class T, int N> __device__ __forceinline__ void store_once(T *p, const Held<T, N> &h) {
    if constexpr (sizeof(h) == 16) {
        uint4 v;
        memcpy(&v, &h, 16);
        __stcs(reinterpret_cast<uint4 *>(p), v);
    } else {
        *reinterpret_cast<Held<T, N> *>(p) = h;
    }
}

/* ---- warp reductions (every lane receives the result) ---- */

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

/* ---- functions of the special unit, subnormal results flushed ---- */

__device__ __forceinline__ float fast_exp2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float fast_rcp(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float fast_sqrt(float v) {
    float r;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
constexpr float kLog2e = 1.44269504f;
/* 1 / (1 + e^-v): a few units in the last place (2 from each function, one
 * from the argument's product for |v| < 8, where it matters). */
__device__ __forceinline__ float fast_sigmoid(float v) { return fast_rcp(1.0f + fast_exp2(-kLog2e * v)); }

/* v / by for v < 2^31, from floor((2^32 - 1) / by). */
__device__ __forceinline__ unsigned divided(unsigned v, unsigned by, unsigned magic) {
    unsigned q = __umulhi(v, magic); /* at most 2 below */
    unsigned r = v - q * by;
    if (r >= by) ++q, r -= by;
    if (r >= by) ++q;
    return q;
}

/* ---- two f32 values in one register pair, each operation on both ---- */

struct F2 {
    unsigned long long v;
};
__device__ __forceinline__ F2 pair(float a, float b) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void split(F2 p, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p.v)); }
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ F2 both(float v) { return pair(v, v); }
/* fast_sigmoid of both. */
__device__ __forceinline__ F2 sigmoid2(F2 v) {
    float a, b;
    split(mul2(v, both(-kLog2e)), a, b);
    split(add2(pair(fast_exp2(a), fast_exp2(b)), both(1.0f)), a, b);
    return pair(fast_rcp(a), fast_rcp(b));
}

/* The same operations on one value and on a pair, for code that takes either. */
__device__ __forceinline__ float vadd(float a, float b) { return a + b; }
__device__ __forceinline__ float vmul(float a, float b) { return a * b; }
__device__ __forceinline__ float vfma(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ F2 vadd(F2 a, F2 b) { return add2(a, b); }
__device__ __forceinline__ F2 vmul(F2 a, F2 b) { return mul2(a, b); }
__device__ __forceinline__ F2 vfma(F2 a, F2 b, F2 c) { return fma2(a, b, c); }
__device__ __forceinline__ float vsigmoid(float v) { return fast_sigmoid(v); }
__device__ __forceinline__ F2 vsigmoid(F2 v) { return sigmoid2(v); }
template <class V> __device__ __forceinline__ V vall(float v);
template <> __device__ __forceinline__ float vall<float>(float v) { return v; }
template <> __device__ __forceinline__ F2 vall<F2>(float v) { return both(v); }
/* f of each value. */
template <class F> __device__ __forceinline__ float veach(float v, F &&f) { return f(v); }
template <class F> __device__ __forceinline__ F2 veach(F2 v, F &&f) {
    float a, b;
    split(v, a, b);
    return pair(f(a), f(b));
}
/* N values as pairs, or the one value. */
template <int N> struct Values {
    using V = std::conditional_t<N == 1, float, F2>;
    static constexpr int kCount = N == 1 ? 1 : N / 2;
};
template <int N> using Array = typename Values<N>::V[Values<N>::kCount];
template <class V> __device__ __forceinline__ V vload(const float *f) {
    if constexpr (std::is_same<V, F2>::value) return pair(f[0], f[1]);
    else return f[0];
}
__device__ __forceinline__ void vstore(float *f, float v) { f[0] = v; }
__device__ __forceinline__ void vstore(float *f, F2 v) { split(v, f[0], f[1]); }

/* ---- sums over the rows of partial [rows, columns] in f32 ---- */

constexpr int kColumnThreads = 512;      /* 32 columns x 16 rows at a time */
constexpr size_t kColumnRows = 256;      /* rows that one launch of one CTA a strip of columns sums */
constexpr size_t kColumnPartRows = 128;  /* rows of a part where there are more */
constexpr size_t kColumnParts = 128;     /* parts of the rows at most */

/* Part blockIdx.y of the rows of 32 columns; out [gridDim.y, columns], or
 * last(column, sum) where the rows are one part. */
template <class Last>
__global__ void __launch_bounds__(kColumnThreads)
column_sums(const float *partial, size_t rows, size_t columns, float *out, Last last) {
    __shared__ float sums[16][33];
    const int lane = threadIdx.x % 32, row = threadIdx.x / 32;
    const size_t c = static_cast<size_t>(blockIdx.x) * 32 + lane;
    const size_t per = (rows + gridDim.y - 1) / gridDim.y, first = per * blockIdx.y;
    const size_t end = first + per < rows ? first + per : rows;
    float s[8] = {};
    if (c < columns) {
        for (size_t r = first + row; r < end; r += 128)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (r + 16 * i < end) s[i] += partial[(r + 16 * i) * columns + c];
    }
    sums[row][lane] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    __syncthreads();
    if (row == 0 && c < columns) {
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) t += sums[i][lane];
        if (gridDim.y == 1) last(c, t);
        else out[blockIdx.y * columns + c] = t;
    }
}

/* Room behind the partial sums, in rows. */
inline size_t column_parts(size_t rows) {
    if (rows <= kColumnRows) return 1;
    const size_t p = (rows + kColumnPartRows - 1) / kColumnPartRows;
    return p < kColumnParts ? p : kColumnParts;
}

inline int launched() { return cudaGetLastError() == cudaSuccess; }

/* Sums the columns of partial [rows, columns], last(column, sum) for each; the
 * parts' sums go behind it. */
template <class Last>
int sum_columns(float *partial, size_t rows, size_t columns, Last last, cudaStream_t st) {
    const unsigned wide = static_cast<unsigned>((columns + 31) / 32);
    const size_t parts = column_parts(rows);
    if (parts > 1) {
        float *sums = partial + rows * columns;
        column_sums<<<dim3(wide, static_cast<unsigned>(parts)), kColumnThreads, 0, st>>>(partial, rows, columns, sums, last);
        if (!launched()) return 0;
        partial = sums;
        rows = parts;
    }
    column_sums<<<dim3(wide, 1), kColumnThreads, 0, st>>>(partial, rows, columns, static_cast<float *>(nullptr), last);
    return launched();
}

/* ---- host side ---- */

inline size_t type_size(int type) { return type == TB_TYPE_F32 ? 4 : 2; }
inline bool type_known(int type) { return type == TB_TYPE_F32 || type == TB_TYPE_BF16 || type == TB_TYPE_F16; }
inline bool aligned(const void *p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
inline size_t align_up(size_t v, size_t to) { return (v + to - 1) / to * to; }

/* Whether an output lies at the address of an input or of another output (NULL
 * lies nowhere). */
template <size_t OUTS, size_t INS>
inline bool collide(const void *const (&outs)[OUTS], const void *const (&ins)[INS]) {
    for (size_t i = 0; i < OUTS; ++i) {
        if (!outs[i]) continue;
        for (const void *in : ins)
            if (outs[i] == in) return true;
        for (size_t j = 0; j < i; ++j)
            if (outs[i] == outs[j]) return true;
    }
    return false;
}

/* a * b, or false where it passes `most`. */
inline bool product(size_t a, size_t b, size_t most, size_t *out) {
    if (a != 0 && b > most / a) return false;
    *out = a * b;
    return true;
}

/* Calls f with a value of the element type that `type` names. */
template <class F> inline int with_type(int type, F &&f) {
    if (type == TB_TYPE_F32) return f(float{});
    if (type == TB_TYPE_BF16) return f(__nv_bfloat16{});
    return f(__half{});
}

/* Multiprocessors of the current device, 0 if there is none; asked once per device. */
constexpr int kMaxDevices = 64;
inline int multiprocessors(int *device) {
    static std::atomic<int> known[kMaxDevices];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 0;
    *device = dev;
    n = known[dev].load(std::memory_order_relaxed);
    if (n == 0 && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess)
        known[dev].store(n, std::memory_order_relaxed);
    return n;
}

/* Lets a kernel have `shared` bytes of dynamic shared memory; set once per
 * kernel and device, and again only where more is asked for. */
template <auto Kernel> bool allow_shared(size_t shared) {
    static SharedLimit limits[kMaxDevices];
    if (shared <= 32 * 1024) return true; /* 48 KB are allowed anyway, static shared memory included */
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return false;
    return limits[dev].raise(shared, [](size_t bytes) {
        return cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)) == cudaSuccess;
    });
}

/* A pack is 16 bytes, 4 bytes or an element: the widest one that divides all of
 * `bits` (addresses, strides and widths in bytes, or-ed). */
inline int pack_of(size_t bits, size_t size) {
    if (bits % 16 == 0) return static_cast<int>(16 / size);
    return bits % 4 == 0 ? static_cast<int>(4 / size) : 1;
}

/* Calls f with the pack as a constant. */
template <class T, class F> inline int with_pack(int pack, F &&f) {
    if (pack == 16 / static_cast<int>(sizeof(T))) return f(std::integral_constant<int, 16 / static_cast<int>(sizeof(T))>{});
    if constexpr (sizeof(T) == 2)
        if (pack == 2) return f(std::integral_constant<int, 2>{});
    return f(std::integral_constant<int, 1>{});
}

} /* namespace tb_learn */

#endif
