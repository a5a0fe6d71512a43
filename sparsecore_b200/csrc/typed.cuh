// 32- and 16-bit floating element types and their vector loads and stores,
// for the kernels of the training step's dense part.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace slb {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N elements moved as one unit of up to 16 bytes (as several where they are
// more): the address is a multiple of that unit.
template <typename T, int N>
struct alignas(sizeof(T) * N >= 16 ? 16 : sizeof(T) * N) Pack {
    T v[N];
};

template <typename T, int N>
__device__ __forceinline__ void load_f(const T* src, float (&out)[N]) {
    const Pack<T, N> q = *reinterpret_cast<const Pack<T, N>*>(src);
#pragma unroll
    for (int k = 0; k < N; ++k) out[k] = to_f(q.v[k]);
}
template <typename T, int N>
__device__ __forceinline__ void store_f(T* dst, const float (&in)[N]) {
    Pack<T, N> q;
#pragma unroll
    for (int k = 0; k < N; ++k) q.v[k] = from_f<T>(in[k]);
    *reinterpret_cast<Pack<T, N>*>(dst) = q;
}

inline int64_t dtype_bytes(int dtype) { return dtype == SL_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) { return dtype == SL_F32 || dtype == SL_BF16 || dtype == SL_F16; }
inline bool off_by(const void* q, int64_t a) { return (reinterpret_cast<uintptr_t>(q) & (a - 1)) != 0; }

}  // namespace slb
