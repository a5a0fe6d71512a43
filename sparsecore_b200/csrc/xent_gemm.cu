// The matrix products of the linear cross entropy and their epilogues:
// plain tiles of 64 x 64 on the 32-bit units.
#include <algorithm>

#include "xent.cuh"

namespace slb {
namespace xent {
namespace {

constexpr int kT = 64, kK = 16, kThreads = 256;

// Element (i, k) of an operand lies at i * si + k * sk of each plane.
struct View {
    const void* base;
    int64_t n, si, sk, plane;
};

struct Args {
    Problem p;
    View a, b;
    int64_t M, N, K;
    int mode;  // 0: partial maxima and sums, 1: gradient planes, 2: output
    int64_t v0;
    void* g;
    int64_t g_stride, g_plane;
    Output o;
};

template <typename T>
__device__ __forceinline__ float get(const View& v, int64_t i, int64_t k, bool two) {
    if (i >= v.n) return 0.f;
    const T* q = static_cast<const T*>(v.base) + i * v.si + k * v.sk;
    return two ? to_f(q[0]) + to_f(q[v.plane]) : to_f(q[0]);
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
gemm_kernel(Args a) {
    __shared__ float As[kK][kT + 1], Bs[kK][kT + 1], C[kT][kT + 1];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int64_t m0 = static_cast<int64_t>(blockIdx.x) * kT, n0 = static_cast<int64_t>(blockIdx.y) * kT;
    const bool two = a.p.f32;
    float acc[4][4] = {};
    for (int64_t k0 = 0; k0 < a.K; k0 += kK) {
        for (int i = threadIdx.x; i < kT * kK; i += kThreads) {
            const int r = i / kK, k = i % kK;
            const bool in = k0 + k < a.K;
            As[k][r] = in ? get<T>(a.a, m0 + r, k0 + k, two) : 0.f;
            Bs[k][r] = in ? get<T>(a.b, n0 + r, k0 + k, two) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kK; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(As[k][ty * 4 + i], Bs[k][tx * 4 + j], acc[i][j]);
        __syncthreads();
    }
    float ux = 1.f, uw = 1.f;
    if (two) {
        ux = exp2f(-static_cast<float>(plane_exponent(a.p.head->max_x)));
        uw = exp2f(-static_cast<float>(plane_exponent(a.p.head->max_w)));
    }
    if (a.mode == 2) {
        const float gs = a.p.bf16 ? 1.f : 1.f / kGradScale, u = a.o.by_x ? ux : uw, g = a.p.head->g;
        for (int i = 0; i < 4; ++i)
            for (int j = 0; j < 4; ++j) {
                const int64_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
                if (m >= a.M || n >= a.N) continue;
                float v = acc[i][j];
                if (a.o.acc) {
                    if (!a.o.first) v += a.o.acc[m * a.N + n];
                    a.o.acc[m * a.N + n] = v;
                }
                if (!a.o.last) continue;
                v = v * gs * u * g;
                if (a.o.dtype == SL_F32) static_cast<float*>(a.o.dst)[m * a.N + n] = v;
                else if (a.o.dtype == SL_BF16) static_cast<__nv_bfloat16*>(a.o.dst)[m * a.N + n] = __float2bfloat16_rn(v);
                else static_cast<__half*>(a.o.dst)[m * a.N + n] = __float2half_rn(v);
            }
        return;
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) C[ty * 4 + i][tx * 4 + j] = acc[i][j] * ux * uw;
    __syncthreads();
    if (a.mode == 0) {
        // one partial for each row of the tile
        if (threadIdx.x < kT && m0 + threadIdx.x < a.M) {
            const int64_t t = m0 + threadIdx.x;
            const int n = static_cast<int>(min(static_cast<int64_t>(kT), a.N - n0));
            float m = -INFINITY, s = 0.f;
            for (int j = 0; j < n; ++j) m = fmaxf(m, C[threadIdx.x][j]);
            for (int j = 0; j < n; ++j) s += expf(C[threadIdx.x][j] - m);
            a.p.part[blockIdx.y * a.M + t] = make_float2(m, s);
            const int64_t at = a.p.tgt[t] - n0;
            if (a.p.tgt[t] >= 0 && at >= 0 && at < n) a.p.zt[t] = C[threadIdx.x][at];
        }
        return;
    }
    for (int i = threadIdx.x; i < kT * kT; i += kThreads) {
        const int r = i / kT, c = i % kT;
        const int64_t t = m0 + r, n = n0 + c;
        if (t >= a.M || n >= a.g_stride) continue;
        const int tg = a.p.tgt[t];
        float v = 0.f;
        if (n < a.N && tg != kIgnored) {
            v = expf(C[r][c] - a.p.row_max[t]) * a.p.row_inv[t] - (a.v0 + n == tg ? 1.f : 0.f);
            if (a.p.g_rows) v = a.p.head->g > 0.f ? v * (a.p.g_rows[t] / a.p.head->g) : 0.f;
        }
        if (a.p.bf16) {
            static_cast<__nv_bfloat16*>(a.g)[t * a.g_stride + n] = __float2bfloat16_rn(v);
        } else {
            v *= kGradScale;
            const __half hi = __float2half_rn(v);
            static_cast<__half*>(a.g)[t * a.g_stride + n] = hi;
            if (two) static_cast<__half*>(a.g)[a.g_plane + t * a.g_stride + n] = __float2half_rn(v - __half2float(hi));
        }
    }
}

int launch(const Args& a, int64_t cols, cudaStream_t s) {
    const dim3 grid(static_cast<unsigned>((a.M + kT - 1) / kT), static_cast<unsigned>((cols + kT - 1) / kT));
    if (a.p.bf16) gemm_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(a);
    else gemm_kernel<__half><<<grid, kThreads, 0, s>>>(a);
    SL_RETURN_IF_LAUNCH_FAILED("sl_xent");
    return SL_OK;
}

View rows(const Operand& o, int64_t from, int64_t n) {
    return {static_cast<const char*>(o.base) + 2 * from * o.stride, n, o.stride, 1, o.plane};
}
View columns(const Operand& o, int64_t n) { return {o.base, n, 1, o.stride, o.plane}; }

}  // namespace

int gemm_stats(const Problem& p, const Operand& x, const Operand& w, cudaStream_t s) {
    Args a{p, rows(x, 0, p.T), rows(w, 0, p.V), p.T, p.V, p.D, 0};
    return launch(a, p.V, s);
}

int gemm_grad(const Problem& p, const Operand& x, const Operand& w, int64_t v0, int64_t cols, const Operand& g,
              cudaStream_t s) {
    Args a{p, rows(x, 0, p.T), rows(w, v0, cols), p.T, cols, p.D, 1, v0, const_cast<void*>(g.base), g.stride, g.plane};
    return launch(a, g.stride, s);
}

int gemm_dx(const Problem& p, const Operand& g, int64_t cols, const Operand& w, int64_t v0, const Output& o, cudaStream_t s) {
    View b = columns(w, p.D);
    b.base = static_cast<const char*>(b.base) + 2 * v0 * w.stride;
    Args a{p, rows(g, 0, p.T), b, p.T, p.D, cols, 2};
    a.o = o;
    return launch(a, p.D, s);
}

int gemm_dw(const Problem& p, const Operand& g, int64_t cols, const Operand& x, const Output& o, cudaStream_t s) {
    Args a{p, columns(g, cols), columns(x, p.D), cols, p.D, p.T, 2};
    a.o = o;
    return launch(a, p.D, s);
}

}  // namespace xent
}  // namespace slb
