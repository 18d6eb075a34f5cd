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

/* ---- host side ---- */

inline size_t type_size(int type) { return type == TB_TYPE_F32 ? 4 : 2; }
inline bool type_known(int type) { return type == TB_TYPE_F32 || type == TB_TYPE_BF16 || type == TB_TYPE_F16; }
inline bool aligned(const void *p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
inline size_t align_up(size_t v, size_t to) { return (v + to - 1) / to * to; }

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

inline int launched() { return cudaGetLastError() == cudaSuccess; }

} /* namespace tb_learn */

#endif
