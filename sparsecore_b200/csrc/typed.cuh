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
    // a copy first: taken apart where they lie, 16-bit values come in words of 4 bytes
    const Pack<T, N> q = *reinterpret_cast<const Pack<T, N>*>(src);
    unpack(q, out);
}
template <typename T, int N>
__device__ __forceinline__ void store_f(T* dst, const float (&in)[N]) {
    *reinterpret_cast<Pack<T, N>*>(dst) = pack<T, N>(in);
}

// Arithmetic on arrays, two 32-bit numbers an instruction (f32x2, sm_100):
// kernels with little memory traffic an element are bound by the number of
// their instructions.  Odd counts go one by one.  An operand is an array, or
// one number for all.
using F2 = unsigned long long;
__device__ __forceinline__ F2 f2(float a, float b) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void f2_split(F2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
template <int N> __device__ __forceinline__ float at1(const float (&v)[N], int k) { return v[k]; }
__device__ __forceinline__ float at1(float v, int) { return v; }
template <int N> __device__ __forceinline__ F2 at2(const float (&v)[N], int k) { return f2(v[k], v[k + 1]); }
__device__ __forceinline__ F2 at2(float v, int) { return f2(v, v); }

// d = a b + c
template <int N, typename A, typename B, typename C>
__device__ __forceinline__ void vfma(float (&d)[N], const A& a, const B& b, const C& c) {
    if constexpr (N % 2 == 0) {
#pragma unroll
        for (int k = 0; k < N; k += 2) f2_split(fma2(at2(a, k), at2(b, k), at2(c, k)), d[k], d[k + 1]);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) d[k] = fmaf(at1(a, k), at1(b, k), at1(c, k));
    }
}
// d = a b
template <int N, typename A, typename B>
__device__ __forceinline__ void vmul(float (&d)[N], const A& a, const B& b) {
    if constexpr (N % 2 == 0) {
#pragma unroll
        for (int k = 0; k < N; k += 2) f2_split(mul2(at2(a, k), at2(b, k)), d[k], d[k + 1]);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) d[k] = at1(a, k) * at1(b, k);
    }
}
// d = a + b
template <int N, typename A, typename B>
__device__ __forceinline__ void vadd(float (&d)[N], const A& a, const B& b) {
    if constexpr (N % 2 == 0) {
#pragma unroll
        for (int k = 0; k < N; k += 2) f2_split(add2(at2(a, k), at2(b, k)), d[k], d[k + 1]);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) d[k] = at1(a, k) + at1(b, k);
    }
}
// A sum that takes its terms in pairs.
struct Sum {
    F2 v = 0;
    template <int N, typename A, typename B>
    __device__ __forceinline__ void fma(const A& a, const B& b) {
        if constexpr (N % 2 == 0) {
#pragma unroll
            for (int k = 0; k < N; k += 2) v = fma2(at2(a, k), at2(b, k), v);
        } else {
#pragma unroll
            for (int k = 0; k < N; ++k) v = fma2(f2(at1(a, k), 0.f), f2(at1(b, k), 0.f), v);
        }
    }
    template <int N>
    __device__ __forceinline__ void add(const float (&a)[N]) {
        if constexpr (N % 2 == 0) {
#pragma unroll
            for (int k = 0; k < N; k += 2) v = add2(at2(a, k), v);
        } else {
#pragma unroll
            for (int k = 0; k < N; ++k) v = add2(f2(a[k], 0.f), v);
        }
    }
    __device__ __forceinline__ float total() const {
        float a, b;
        f2_split(v, a, b);
        return a + b;
    }
};

inline int64_t dtype_bytes(int dtype) { return dtype == SL_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) { return dtype == SL_F32 || dtype == SL_BF16 || dtype == SL_F16; }
inline bool off_by(const void* q, int64_t a) { return (reinterpret_cast<uintptr_t>(q) & (a - 1)) != 0; }

}  // namespace slb
