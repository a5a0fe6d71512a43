// 32- and 16-bit floating element types and their vector loads and stores,
// for the kernels of the training step's dense part.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

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

// Packs and their values in 32 bits; 16-bit types two at a time.
template <typename T, int N>
__device__ __forceinline__ void unpack(const Pack<T, N>& q, float (&out)[N]) {
    if constexpr (sizeof(T) == 2 && N % 2 == 0) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(&q);
#pragma unroll
        for (int k = 0; k < N / 2; ++k) {
            if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                out[2 * k] = __uint_as_float(w[k] << 16);
                out[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
            } else {
                const float2 f = __half22float2(reinterpret_cast<const __half2&>(w[k]));
                out[2 * k] = f.x;
                out[2 * k + 1] = f.y;
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) out[k] = to_f(q.v[k]);
    }
}
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> pack(const float (&in)[N]) {
    Pack<T, N> q;
    if constexpr (sizeof(T) == 2 && N % 2 == 0) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&q);
#pragma unroll
        for (int k = 0; k < N / 2; ++k) {
            if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(in[2 * k], in[2 * k + 1]);
                w[k] = reinterpret_cast<const uint32_t&>(h);
            } else {
                const __half2 h = __floats2half2_rn(in[2 * k], in[2 * k + 1]);
                w[k] = reinterpret_cast<const uint32_t&>(h);
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) q.v[k] = from_f<T>(in[k]);
    }
    return q;
}

template <typename T, int N>
__device__ __forceinline__ void load_f(const T* src, float (&out)[N]) {
    unpack(*reinterpret_cast<const Pack<T, N>*>(src), out);
}
template <typename T, int N>
__device__ __forceinline__ void store_f(T* dst, const float (&in)[N]) {
    *reinterpret_cast<Pack<T, N>*>(dst) = pack<T, N>(in);
}

inline int64_t dtype_bytes(int dtype) { return dtype == SL_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) { return dtype == SL_F32 || dtype == SL_BF16 || dtype == SL_F16; }
inline bool off_by(const void* q, int64_t a) { return (reinterpret_cast<uintptr_t>(q) & (a - 1)) != 0; }

}  // namespace slb
