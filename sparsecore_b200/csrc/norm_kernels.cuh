// The norms around a block, its gate and residual scale, and the residual
// add, in one pass over the rows (forward) and one back (backward).
//
//   u   = N(y; pw, pb) or y          the norm after the block, if there is one
//   out = r + s * gate * u           rounded to the residual's type
//   h   = N(out; w, b)               the norm before the next block
//
// N is LayerNorm, n = (v - mean) / sqrt(var + eps), or RMSNorm,
// n = v / sqrt(mean(v^2) + eps), times its weight, plus its bias.  The
// gradient through N with dn = d * w is (dn - n mean(dn n) [- mean(dn)]) /
// sqrt(...).  The variance is the mean square of the centred values (a
// second sum over registers): no cancellation where the mean is large.
//
// A row belongs to one CTA, which keeps it in registers between its loads
// and its stores, so every operand crosses HBM once: that is the bound.
#pragma once

#include <algorithm>
#include <type_traits>

#include "norm_plan.cuh"

namespace slb {

namespace norm {
namespace {

template <typename TY, typename TR>
struct Args {
    const TY* y;
    const TR* r;
    const void *w, *b, *gate, *pw, *pb;
    TR* out;
    TY* h;
    float4* stats;  // [T]: 1/deviation and -mean/deviation of out's norm; of y's
    const float* scale_dev;
    float scale, eps, post_eps;
    int64_t T, D, gate_rows;  // gate_rows: rows of x that share a row of the gate
    int layer, vec_f32, gate_f32;
    // backward
    const TR* dout;
    const TY* dh;
    TR* dr;
    TY* dy;
    void* dgate;
    float* part;    // [5][ctas][D]: dw, db, dpw, dpb, dgate
    float* part_s;  // [ctas]
    int64_t rows_per_cta, ctas, seg;
    int need_dy, need_gate, need_scale, gate_direct;
};

// VE values of a vector operand (weights, gate), held in 32 bits or in TY.
template <typename TY, int VE>
__device__ __forceinline__ void load_v(const void* base, int f32, int64_t i, float (&o)[VE]) {
    if (f32) load_f<float, VE>(static_cast<const float*>(base) + i, o);
    else load_f<TY, VE>(static_cast<const TY*>(base) + i, o);
}

// A row's elements in one thread: NV vectors of VE, 32 * warps vectors apart.
// They stay packed as they were loaded until they are used.
template <typename T, int VE, int NV>
struct Row {
    Pack<T, VE> v[NV];
    __device__ __forceinline__ void load(const T* src, int col, int step, int cols) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (col + j * step < cols) v[j] = *reinterpret_cast<const Pack<T, VE>*>(src + col + j * step);
    }
    __device__ __forceinline__ void get(int j, float (&o)[VE]) const { unpack(v[j], o); }
};

// Sum of one value over the row's warps, the same in every thread.  `ws`
// holds two buffers that alternate, so one barrier a call is enough.
__device__ __forceinline__ float row_sum(float a, int warps, float2* ws, int& flip) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    if (warps == 1) return a;
    float2* w = ws + flip * 32;
    flip ^= 1;
    const int lane = threadIdx.x & 31;
    if (lane == 0) w[threadIdx.x >> 5].x = a;
    __syncthreads();
    a = lane < warps ? w[lane].x : 0.f;
    for (int o = 1; o < warps; o <<= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    return __shfl_sync(0xffffffffu, a, 0);
}

// Sums of two values.  Lanes 0-15 go on with the first and 16-31 with the
// second after one exchange: half the shuffles of two sums.
__device__ __forceinline__ void row_sum2(float& a, float& b, int warps, float2* ws, int& flip) {
    const int lane = threadIdx.x & 31;
    const bool up = lane >= 16;
    float v = (up ? b : a) + __shfl_xor_sync(0xffffffffu, up ? a : b, 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (warps > 1) {
        float2* w = ws + flip * 32;
        flip ^= 1;
        if (lane == 0) w[threadIdx.x >> 5].x = v;
        if (lane == 16) w[threadIdx.x >> 5].y = v;
        __syncthreads();
        float2 q = lane < warps ? w[lane] : make_float2(0.f, 0.f);  // up to 32 warps
        v = (up ? q.y : q.x) + __shfl_xor_sync(0xffffffffu, up ? q.x : q.y, 16);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    a = __shfl_sync(0xffffffffu, v, 0);
    b = __shfl_sync(0xffffffffu, v, 16);
}

// 1/deviation and mean (0 for RMSNorm) of a row; the variance is a second sum
// over the centred values.
template <int VE, int NV>
__device__ __forceinline__ void row_stats(const float (&v)[NV][VE], int col, int step, int cols, int layer, float inv_d,
                                          float eps, int warps, float2* ws, int& flip, float& rstd, float& mean) {
    Sum a;
    mean = 0.f;
    if (layer) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (col + j * step < cols) a.add(v[j]);
        mean = row_sum(a.total(), warps, ws, flip) * inv_d;
        a = Sum();
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (col + j * step >= cols) continue;
            float c[VE];
            vadd(c, v[j], -mean);
            a.template fma<VE>(c, c);
        }
    } else {
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (col + j * step < cols) a.template fma<VE>(v[j], v[j]);
    }
    rstd = 1.f / sqrtf(fmaf(row_sum(a.total(), warps, ws, flip), inv_d, eps));
}

// First element of the gate of row t (32-bit division: rows fit an int).
template <typename A>
__device__ __forceinline__ int64_t gate_offset(const A& a, int64_t t) {
    return a.gate_rows == 1 ? t * a.D : static_cast<int64_t>(static_cast<uint32_t>(t) / static_cast<uint32_t>(a.gate_rows)) * a.D;
}

// blockDim = (32 * warps a row, rows): one row a warp up to 32 elements a
// lane, without a barrier; more warps a row beyond.  A CTA takes row after
// row; as many CTAs as an SM holds.  TV: type of the vectors (asked for at run
// time it cost 10 of 73 us on 8191 x 4096 bf16 rows with a norm on both sides,
// 57 us now, of 41 for 268 MB: 34 instructions an element, issued in 61 % of the
// clocks; one barrier a norm instead of two changed nothing).  16384 x 768
// fp32: 33 us of 31 for 201 MB, bound by memory.
template <typename TY, typename TR, typename TV, int VE, int NV, bool POST>
__global__ void __launch_bounds__(kMaxThreads, VE * NV <= 16 ? 2 : 1)
norm_fwd_kernel(Args<TY, TR> a) {
    __shared__ float2 ws[64];
    int flip = 0;
    const int warps = blockDim.x >> 5, cols = static_cast<int>(a.D);
    const int col = threadIdx.x * VE, step = blockDim.x * VE;
    const float inv_d = 1.f / static_cast<float>(cols);
    const float scale = a.scale_dev ? *a.scale_dev : a.scale;
    Row<TY, VE, NV> yr;
    Row<TR, VE, NV> rr;
    int64_t t = blockIdx.x * static_cast<int64_t>(blockDim.y) + threadIdx.y;
    if (t < a.T) {
        yr.load(a.y + t * a.D, col, step, cols);
        rr.load(a.r + t * a.D, col, step, cols);
    }
    for (; t < a.T; t += static_cast<int64_t>(gridDim.x) * blockDim.y) {
        float4 st = make_float4(0.f, 0.f, 1.f, 0.f);
        float r[NV][VE];
        if (POST) {
#pragma unroll
            for (int j = 0; j < NV; ++j) yr.get(j, r[j]);
            row_stats<VE, NV>(r, col, step, cols, a.layer, inv_d, a.post_eps, warps, ws, flip, st.z, st.w);
        }
        const int64_t gate_row = a.gate ? gate_offset(a, t) : 0;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = col + j * step;
            if (c >= cols) continue;
            float y[VE], q[VE];
            yr.get(j, y);
            if (POST) {
                load_f<TV, VE>(static_cast<const TV*>(a.pw) + c, q);
                vadd(y, y, -st.w);
                vmul(y, y, st.z);
                if (a.pb) {
                    float b[VE];
                    load_f<TV, VE>(static_cast<const TV*>(a.pb) + c, b);
                    vfma(y, y, q, b);
                } else {
                    vmul(y, y, q);
                }
            }
            if (a.gate) {
                load_v<TY, VE>(a.gate, a.gate_f32, gate_row + c, q);
                vmul(y, y, q);
            }
            // the stream is held in its own type, and the norm reads what it holds
            rr.get(j, q);
            vfma(y, y, scale, q);
            rr.v[j] = pack<TR, VE>(y);
            rr.get(j, r[j]);
            *reinterpret_cast<Pack<TR, VE>*>(a.out + t * a.D + c) = rr.v[j];
        }
        // the next row's operands are on their way over the rest of this one
        const int64_t next = t + static_cast<int64_t>(gridDim.x) * blockDim.y;
        if (next < a.T) {
            yr.load(a.y + next * a.D, col, step, cols);
            rr.load(a.r + next * a.D, col, step, cols);
        }
        row_stats<VE, NV>(r, col, step, cols, a.layer, inv_d, a.eps, warps, ws, flip, st.x, st.y);
        if (a.stats && threadIdx.x == 0) a.stats[t] = make_float4(st.x, -st.y * st.x, st.z, -st.w * st.z);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = col + j * step;
            if (c >= cols) continue;
            float w[VE], o[VE];
            load_f<TV, VE>(static_cast<const TV*>(a.w) + c, w);
            vadd(o, r[j], -st.y);
            vmul(o, o, st.x);
            if (a.b) {
                float b[VE];
                load_f<TV, VE>(static_cast<const TV*>(a.b) + c, b);
                vfma(o, o, w, b);
            } else {
                vmul(o, o, w);
            }
            store_f<TY, VE>(a.h + t * a.D + c, o);
        }
    }
}

// Rows [t0, t1) of CTA `cta`.  With gates shared by whole runs of rows (seg
// CTAs to a run) no CTA crosses a run's end.
template <typename A>
__device__ __forceinline__ void my_rows(const A& a, int64_t cta, int64_t& t0, int64_t& t1) {
    if (a.seg > 0) {
        const int64_t run = cta / a.seg, part = cta % a.seg;
        t0 = run * a.gate_rows + part * a.rows_per_cta;
        t1 = min(t0 + a.rows_per_cta, min((run + 1) * a.gate_rows, a.T));
    } else {
        t0 = cta * a.rows_per_cta;
        t1 = min(t0 + a.rows_per_cta, a.T);
    }
}

// Backward of out = r + scale * y, h = N(out): dr = dout + N'(dh), dy = scale
// dr.  A row belongs to blockDim.x threads; blockDim.y rows are taken at a
// time.  The vectors' gradients of a thread's columns stay in registers over
// all its rows; they are written once per CTA and summed over the CTAs in
// order by norm_reduce_kernel, so they do not depend on timing.
template <typename TY, typename TR, int VE, int NV>
__global__ void __launch_bounds__(256)
norm_bwd_kernel(Args<TY, TR> a) {
    __shared__ float2 ws[64];
    extern __shared__ float join[];  // [2][D], where a CTA takes several rows
    int flip = 0;
    const int warps = blockDim.x >> 5, cols = static_cast<int>(a.D);
    const int col = threadIdx.x * VE, step = blockDim.x * VE;
    const float inv_d = 1.f / static_cast<float>(cols);
    const float scale = a.scale_dev ? *a.scale_dev : a.scale;
    float aw[NV][VE] = {}, ab[NV][VE] = {};
    int64_t t0, t1;
    my_rows(a, blockIdx.x, t0, t1);
    for (int64_t t = t0 + threadIdx.y; t < t1; t += blockDim.y) {
        const int64_t row = t * a.D;
        Row<TR, VE, NV> xr, dr;
        Row<TY, VE, NV> nr;
        xr.load(a.out + row, col, step, cols);
        nr.load(a.dh + row, col, step, cols);
        dr.load(a.dout + row, col, step, cols);
        const float4 st = a.stats[t];
        Sum s1, s2;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = col + j * step;
            if (c >= cols) continue;
            float w[VE], x[VE], d[VE];
            load_v<TY, VE>(a.w, a.vec_f32, c, w);
            xr.get(j, x);
            nr.get(j, d);
            vfma(x, x, st.x, st.y);
            vfma(aw[j], d, x, aw[j]);
            vadd(ab[j], ab[j], d);
            vmul(d, d, w);
            s1.add(d);
            s2.template fma<VE>(d, x);
        }
        float c1 = s1.total(), c2 = s2.total();
        row_sum2(c1, c2, warps, ws, flip);
        c1 = a.layer ? c1 * inv_d : 0.f;
        c2 *= inv_d;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = col + j * step;
            if (c >= cols) continue;
            float w[VE], d[VE], x[VE], g[VE];
            load_v<TY, VE>(a.w, a.vec_f32, c, w);
            xr.get(j, x);
            nr.get(j, g);
            dr.get(j, d);
            vfma(x, x, st.x, st.y);
            vfma(x, x, -c2, -c1);
            vfma(g, g, w, x);
            vfma(d, g, st.x, d);
            store_f<TR, VE>(a.dr + row + c, d);
            if (a.need_dy) {
                vmul(d, d, scale);
                store_f<TY, VE>(a.dy + row + c, d);
            }
        }
    }
    // The CTA's rows of threads add up in their order.
    for (int y = 1; y < blockDim.y; ++y) {
        if (threadIdx.y == y) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (col + j * step < cols) {
                    store_f<float, VE>(join + col + j * step, aw[j]);
                    store_f<float, VE>(join + cols + col + j * step, ab[j]);
                }
        }
        __syncthreads();
        if (threadIdx.y == 0) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (col + j * step < cols) {
                    float q[VE];
                    load_f<float, VE>(join + col + j * step, q);
#pragma unroll
                    for (int k = 0; k < VE; ++k) aw[j][k] += q[k];
                    load_f<float, VE>(join + cols + col + j * step, q);
#pragma unroll
                    for (int k = 0; k < VE; ++k) ab[j][k] += q[k];
                }
        }
        __syncthreads();
    }
    if (threadIdx.y) return;
    const int64_t plane = a.ctas * a.D;
#pragma unroll
    for (int j = 0; j < NV; ++j)
        if (col + j * step < cols) {
            float* q = a.part + blockIdx.x * a.D + col + j * step;
            store_f<float, VE>(q, aw[j]);
            if (a.b) store_f<float, VE>(q + plane, ab[j]);
        }
}

// Sums of four or eight values over a row's warps in two steps with a barrier
// of the caller's between them, as row_sum2.
__device__ __forceinline__ float fold4(const float4& q) {  // lanes 0, 8, 16 and 24 end with the sums of x, y, z and w
    const int lane = threadIdx.x & 31;
    const bool up = lane & 16, high = lane & 8;
    const float a = (up ? q.z : q.x) + __shfl_xor_sync(0xffffffffu, up ? q.x : q.z, 16);
    const float b = (up ? q.w : q.y) + __shfl_xor_sync(0xffffffffu, up ? q.y : q.w, 16);
    float v = (high ? b : a) + __shfl_xor_sync(0xffffffffu, high ? a : b, 8);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <int Q>
__device__ __forceinline__ void sums_put(const float (&s)[4 * Q], float4 (*w)[32]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const float v = fold4(make_float4(s[4 * q], s[4 * q + 1], s[4 * q + 2], s[4 * q + 3]));
        if ((lane & 7) == 0) reinterpret_cast<float*>(&w[q][threadIdx.x >> 5])[lane >> 3] = v;
    }
}
template <int Q>
__device__ __forceinline__ void sums_get(float (&s)[4 * Q], int warps, float4 (*w)[32]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const float v = fold4(lane < warps ? w[q][lane] : make_float4(0.f, 0.f, 0.f, 0.f));
#pragma unroll
        for (int k = 0; k < 4; ++k) s[4 * q + k] = __shfl_sync(0xffffffffu, v, 8 * k);
    }
}

__device__ __forceinline__ void copy16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the last `n` groups of this thread's copies have landed (n = 1 or 2).
__device__ __forceinline__ void copies_wait(int n) {
    if (n == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 2;" ::: "memory");
}

// Where a thread finds its part of a row's operands and of the vectors: in
// 16-byte granules of shared memory that it fills itself (RING), so that no
// barrier guards them, or in global memory.
enum Operand : int { kX, kDn, kD, kY, kG };
template <typename TY, typename TR, int VE, int NV>
struct Ring {
    static constexpr int kT = VE * sizeof(TY) / 16, kR = VE * sizeof(TR) / 16;  // granules of a vector
    static constexpr int kVec = NV * VE / 4;
    // 32-bit rows leave no room for the vectors (read from L1 instead, as no
    // type has to be changed) nor for a gate a row.
    static constexpr bool kVectors = sizeof(TY) == 2, kGates = sizeof(TY) == 2;
    __host__ __device__ static constexpr int first(int op) {
        return op == kX ? 0 : op == kDn ? NV * kR : op == kD ? NV * (kR + kT) : op == kY ? NV * (2 * kR + kT) : NV * (2 * kR + 2 * kT);
    }
    __host__ __device__ static constexpr int granules(bool gate) { return NV * (2 * kR + (gate ? 3 : 2) * kT); }
};

// Backward with a norm, a gate or a learned scale after the block (and of
// very wide rows): a row a CTA at a time.
//
// With dn = dh w, d = dout + rstd (dn - c1 - x c2) and, behind the block's norm,
// dy = prstd (q - e1 - y e2), q = scale gate pw d, the means e1 and e2 are linear
// in c1 and c2, so the row's sums are all taken at once:
//   e2 D = sum(qy (dout + rstd dn)) - c1 sum(qy rstd) - c2 sum(qy rstd x),
// qy = scale gate pw y, and e1 alike with scale gate pw: one barrier a row, and
// nothing but the packed operands is needed on its other side.  Those wait in
// shared memory, copied there rows ahead; the gradients of the vectors (two
// to five a column) stay in registers, which leave room for one CTA an SM.
// Between two barriers a warp has the sums of the next row and the results
// of this one to work on, which hide each other's latencies.
//
// 8191 x 4096 bf16 with both norms and a gate a channel (which has a kernel of
// its own below): 100 us of 62 for its 403 MB; 220 us with two barriers a row
// and no ring, 121 us before the next row's sums were taken beside this row's
// results.  Bound by the latency of
// sixteen warps with one row under way (the scheduler issues in half of the
// clocks).  L: LayerNorm, or a bias.
template <typename TY, typename TR, int VE, int NV, bool POST, bool L, bool RING>
__global__ void __launch_bounds__(kMaxThreads)
norm_bwd_full_kernel(Args<TY, TR> a, int stages) {
    constexpr int Q = L && POST ? 2 : 1;
    __shared__ float4 ws[2][Q][32];
    extern __shared__ __align__(16) char mem[];
    using R = Ring<TY, TR, VE, NV>;
    constexpr bool KEEP = RING && R::kVectors;
    const int warps = blockDim.x >> 5, cols = static_cast<int>(a.D);
    const int col = threadIdx.x * VE, step = blockDim.x * VE;
    const float inv_d = 1.f / static_cast<float>(cols);
    const float scale = a.scale_dev ? *a.scale_dev : a.scale;
    const bool each = a.gate && a.gate_rows == 1, ring_gate = RING && R::kGates && each && !a.gate_f32;
    float aw[NV][VE] = {}, ag[NV][VE] = {}, apw[POST ? NV : 1][VE] = {};
    float ab[L ? NV : 1][VE] = {}, apb[L && POST ? NV : 1][VE] = {};
    float as = 0.f;
    int64_t t0, t1;
    my_rows(a, blockIdx.x, t0, t1);

    const int lap = blockDim.x * 16;  // bytes from a thread's granule to its next
    char* const mine = mem + threadIdx.x * 16;
    const int stage_bytes = R::granules(ring_gate) * lap;
    char* const vectors = mine + stages * stage_bytes;
    auto vector_slot = [&](int which, int j, int q) {
        return reinterpret_cast<float4*>(vectors + (which * R::kVec + j * (VE / 4) + q) * lap);
    };
    auto fetch = [&](int64_t t, int stage) {
        char* const to = mine + stage * stage_bytes;
        if (t < t1) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = col + j * step;
                if (c >= cols) continue;
                const int64_t i = t * a.D + c;
                auto put = [&](int op, const void* src, int size) {
#pragma unroll
                    for (int q = 0; q < size; ++q) copy16(to + (R::first(op) + j * size + q) * lap, static_cast<const char*>(src) + 16 * q);
                };
                put(kX, a.out + i, R::kR);
                put(kDn, a.dh + i, R::kT);
                put(kD, a.dout + i, R::kR);
                put(kY, a.y + i, R::kT);
                if (ring_gate) put(kG, static_cast<const TY*>(a.gate) + i, R::kT);
            }
        }
        copies_commit();
    };
    // Vector j of an operand of row t.
    auto get = [&](auto type, int op, const auto* base, int64_t t, const char* from, int j, float (&o)[VE]) {
        using T = decltype(type);
        if constexpr (RING) {
            constexpr int size = VE * sizeof(T) / 16;
            Pack<T, VE> p;
#pragma unroll
            for (int q = 0; q < size; ++q) reinterpret_cast<uint4*>(&p)[q] = *reinterpret_cast<const uint4*>(from + (R::first(op) + j * size + q) * lap);
            unpack(p, o);
        } else {
            load_f<T, VE>(reinterpret_cast<const T*>(base) + t * a.D + col + j * step, o);
        }
    };
    // 0: weight, 1: the block's norm's, 2: its bias, 3: a gate that all rows of this CTA share
    const void* const vec_src[4] = {a.w, a.pw, a.pb, each ? nullptr : a.gate};
    const int vec_f32[4] = {a.vec_f32, a.vec_f32, a.vec_f32, a.gate_f32};
    auto vec_read = [&](int which, int64_t from, int j, float (&o)[VE]) { load_v<TY, VE>(vec_src[which], vec_f32[which], from + col + j * step, o); };
    auto vec_keep = [&](int which, int64_t from) {
        if constexpr (KEEP) {
            if (vec_src[which] == nullptr) return;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                if (col + j * step >= cols) continue;
                float o[VE];
                vec_read(which, from, j, o);
#pragma unroll
                for (int q = 0; q < VE / 4; ++q) *vector_slot(which, j, q) = make_float4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
            }
        }
    };
    auto vector = [&](int which, int64_t from, int j, float (&o)[VE]) {
        if constexpr (KEEP) {
#pragma unroll
            for (int q = 0; q < VE / 4; ++q) {
                const float4 f = *vector_slot(which, j, q);
                o[4 * q] = f.x; o[4 * q + 1] = f.y; o[4 * q + 2] = f.z; o[4 * q + 3] = f.w;
            }
        } else {
            vec_read(which, from, j, o);
        }
    };
    auto gate = [&](int64_t t, int64_t from, const char* held, int j, float (&o)[VE]) {
        if (!each) vector(3, from, j, o);
        else if (ring_gate) get(TY{}, kG, static_cast<const TY*>(a.gate), t, held, j, o);
        else load_v<TY, VE>(a.gate, a.gate_f32, t * a.D + col + j * step, o);
    };
    // The rows' sums; gates shared by a run of rows are those of `from`.
    const bool sums_dy = POST && a.need_dy;
    auto sums = [&](int64_t t, int64_t from, const float4& st, const char* held, float4 (*to)[32]) {
        Sum p[4 * Q];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (col + j * step >= cols) continue;
            float x[VE], g[VE], w[VE];
            get(TR{}, kX, a.out, t, held, j, x);
            get(TY{}, kDn, a.dh, t, held, j, g);
            vector(0, 0, j, w);
            vfma(x, x, st.x, st.y);
            vmul(g, g, w);
            p[0].template fma<VE>(g, x);
            if (L) p[1].add(g);
            if (sums_dy) {
                float q[VE], y[VE], d[VE];
                vector(1, 0, j, q);
                if (a.gate) {
                    gate(t, from, held, j, d);
                    vmul(q, q, d);
                }
                get(TR{}, kD, a.dout, t, held, j, d);
                get(TY{}, kY, a.y, t, held, j, y);
                vfma(y, y, st.z, st.w);
                vmul(y, y, q);
                vfma(d, g, st.x, d);
                p[2].template fma<VE>(y, d);
                p[3].template fma<VE>(y, x);
                if constexpr (Q == 2) {
                    p[4].add(y);
                    p[5].template fma<VE>(q, d);
                    p[6].template fma<VE>(q, x);
                    p[7].add(q);
                }
            }
        }
        float s[4 * Q];
#pragma unroll
        for (int k = 0; k < 4 * Q; ++k) s[k] = p[k].total();
        sums_put<Q>(s, to);
    };
    auto statistics = [&](int64_t t) { return a.stats[min(t, t1 - 1)]; };
    auto run_of = [&](int64_t t) { return a.gate && !each ? static_cast<int64_t>(static_cast<uint32_t>(t) / static_cast<uint32_t>(a.gate_rows)) : 0; };

    if (t0 < t1) {
        if constexpr (RING)
            for (int k = 0; k < stages - 1; ++k) fetch(t0 + k, k);
        for (int k = 0; k < 3; ++k) vec_keep(k, 0);
        int64_t run = run_of(t0), gate_row = run * a.D, run_end = (run + 1) * a.gate_rows;
        vec_keep(3, gate_row);
        if constexpr (RING) copies_wait(stages - 2);
        float4 st = statistics(t0);
        int stage = 0, flip = 0;
        sums(t0, gate_row, st, mine, ws[0]);
        for (int64_t t = t0; t < t1; ++t) {
            const char* const held = mine + stage * stage_bytes;
            const int after = stage + 1 == stages ? 0 : stage + 1;
            if constexpr (RING) {
                fetch(t + stages - 1, stage == 0 ? stages - 1 : stage - 1);
                copies_wait(stages - 2);  // row t + 1 is here
            }
            const float4 next = statistics(t + 1);
            if (warps > 1) __syncthreads();
            else __syncwarp();
            float s[4 * Q];
            sums_get<Q>(s, warps, ws[flip]);
            flip ^= 1;
            // A run's last row is finished before the next run's gate takes its place.
            const bool turn = a.gate && !each && t + 1 == run_end;
            if (t + 1 < t1 && !turn) sums(t + 1, gate_row, next, mine + after * stage_bytes, ws[flip]);
            const float c2 = s[0] * inv_d, c1 = L && a.layer ? s[1] * inv_d : 0.f;
            float e1 = 0.f, e2 = 0.f;
            if (POST) {
                e2 = s[2] - st.x * c2 * s[3];
                if constexpr (Q == 2) {
                    e2 -= st.x * c1 * s[4];
                    e1 = a.layer ? (s[5] - st.x * (c2 * s[6] + c1 * s[7])) * (scale * inv_d) : 0.f;
                }
                e2 *= scale * inv_d;
            }
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = col + j * step;
                if (c >= cols) continue;
                const int64_t at = t * a.D + c;
                float x[VE], g[VE], d[VE], w[VE], y[VE];
                get(TR{}, kX, a.out, t, held, j, x);
                get(TY{}, kDn, a.dh, t, held, j, g);
                get(TR{}, kD, a.dout, t, held, j, d);
                vector(0, 0, j, w);
                vfma(x, x, st.x, st.y);
                vfma(aw[j], g, x, aw[j]);
                if (L) vadd(ab[j], ab[j], g);
                if (L) vfma(x, x, -c2, -c1);
                else vmul(x, x, -c2);
                vfma(g, g, w, x);
                vfma(d, g, st.x, d);
                store_f<TR, VE>(a.dr + at, d);
                get(TY{}, kY, a.y, t, held, j, y);
                float u[VE], pw[VE];
                if (POST) {
                    vector(1, 0, j, pw);
                    vfma(y, y, st.z, st.w);
                    if (L && a.pb) {
                        vector(2, 0, j, x);
                        vfma(u, y, pw, x);
                    } else {
                        vmul(u, y, pw);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < VE; ++k) u[k] = y[k];
                }
                if (a.gate) gate(t, gate_row, held, j, x);
                if (a.need_scale) {
#pragma unroll
                    for (int k = 0; k < VE; ++k) as = fmaf(d[k], a.gate ? x[k] * u[k] : u[k], as);
                }
                vmul(d, d, scale);
                if (each) {
                    vmul(u, u, d);
                    vmul(d, d, x);
                    if (a.need_gate) {
                        if (a.gate_f32) store_f<float, VE>(static_cast<float*>(a.dgate) + at, u);
                        else store_f<TY, VE>(static_cast<TY*>(a.dgate) + at, u);
                    }
                } else if (a.gate) {
                    vfma(ag[j], d, u, ag[j]);
                    vmul(d, d, x);
                }
                if (POST) {
                    vfma(apw[j], d, y, apw[j]);
                    if (L) vadd(apb[j], apb[j], d);
                    if (L) vfma(y, y, -e2, -e1);
                    else vmul(y, y, -e2);
                    vfma(d, d, pw, y);
                    vmul(d, d, st.z);
                }
                if (a.need_dy) store_f<TY, VE>(a.dy + at, d);
                if (a.gate_direct && (t + 1 == t1 || t + 1 == run_end)) {  // a run of rows ends
                    if (a.gate_f32) store_f<float, VE>(static_cast<float*>(a.dgate) + gate_row + c, ag[j]);
                    else store_f<TY, VE>(static_cast<TY*>(a.dgate) + gate_row + c, ag[j]);
#pragma unroll
                    for (int k = 0; k < VE; ++k) ag[j][k] = 0.f;
                }
            }
            if (turn && t + 1 < t1) {
                gate_row += a.D;
                run_end += a.gate_rows;
                vec_keep(3, gate_row);
                sums(t + 1, gate_row, next, mine + after * stage_bytes, ws[flip]);
            }
            st = next;
            stage = after;
        }
    }
    const int64_t plane = a.ctas * a.D;
#pragma unroll
    for (int j = 0; j < NV; ++j)
        if (col + j * step < cols) {
            float* q = a.part + blockIdx.x * a.D + col + j * step;
            store_f<float, VE>(q, aw[j]);
            if constexpr (L) store_f<float, VE>(q + plane, ab[j]);
            if constexpr (POST) store_f<float, VE>(q + 2 * plane, apw[j]);
            if constexpr (POST && L) store_f<float, VE>(q + 3 * plane, apb[j]);
            if (a.need_gate && a.seg > 0) store_f<float, VE>(q + 4 * plane, ag[j]);
        }
    if (a.need_scale) {
        float z[4 * Q] = {as};
        __syncthreads();
        sums_put<Q>(z, ws[0]);
        __syncthreads();
        sums_get<Q>(z, warps, ws[0]);
        if (threadIdx.x == 0) a.part_s[blockIdx.x] = z[0];
    }
}

// The same where all rows of a CTA share their gate (or have none), as almost
// always.  What lies behind the stream is then one vector, q = scale gate pw,
// and every gradient of the vectors follows from two sums a column over the
// rows, d yhat and d, multiplied out once at the end:
//   dpw = scale gate S1, dpb = scale gate S0, dgate = scale (pw S1 + pb S0),
//   dscale = sum of gate (pw S1 + pb S0).
// yhat = y where there is no norm behind the block.  Fewer sums, vectors and
// operations a row (46 instructions an element instead of 53): 8191 x 4096
// bf16 with both norms and a gate a channel take 92 us instead of 100.
template <typename TY, typename TR, int VE, int NV, bool POST, bool L>
__global__ void __launch_bounds__(kMaxThreads)
norm_bwd_shared_kernel(Args<TY, TR> a, int stages) {
    constexpr int Q = L && POST ? 2 : 1;
    constexpr int kT = VE * sizeof(TY) / 16, kR = VE * sizeof(TR) / 16;  // granules of a vector
    constexpr int kVec = NV * VE / 4;
    constexpr int oX = 0, oN = NV * kR, oD = NV * (kR + kT), oY = NV * (2 * kR + kT), kGranules = NV * 2 * (kR + kT);
    __shared__ float4 ws[2][Q][32];
    extern __shared__ __align__(16) char mem[];
    const int warps = blockDim.x >> 5, cols = static_cast<int>(a.D);
    const int col = threadIdx.x * VE, step = blockDim.x * VE;
    const float inv_d = 1.f / static_cast<float>(cols);
    const float scale = a.scale_dev ? *a.scale_dev : a.scale;
    float aw[NV][VE] = {}, s1[NV][VE] = {}, ab[L ? NV : 1][VE] = {}, s0[L ? NV : 1][VE] = {};
    int64_t t0, t1;
    my_rows(a, blockIdx.x, t0, t1);
    const int64_t gate_row = a.seg > 0 ? blockIdx.x / a.seg * a.D : 0;

    const int lap = blockDim.x * 16;
    char* const mine = mem + threadIdx.x * 16;
    const int stage_bytes = kGranules * lap;
    char* const vectors = mine + stages * stage_bytes;
    auto keep = [&](int which, int j, const float (&o)[VE]) {
#pragma unroll
        for (int q = 0; q < VE / 4; ++q)
            *reinterpret_cast<float4*>(vectors + (which * kVec + j * (VE / 4) + q) * lap) = make_float4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
    };
    auto kept = [&](int which, int j, float (&o)[VE]) {
#pragma unroll
        for (int q = 0; q < VE / 4; ++q) {
            const float4 f = *reinterpret_cast<const float4*>(vectors + (which * kVec + j * (VE / 4) + q) * lap);
            o[4 * q] = f.x; o[4 * q + 1] = f.y; o[4 * q + 2] = f.z; o[4 * q + 3] = f.w;
        }
    };
    auto fetch = [&](int64_t t, int stage) {
        char* const to = mine + stage * stage_bytes;
        if (t < t1) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = col + j * step;
                if (c >= cols) continue;
                const int64_t i = t * a.D + c;
                auto put = [&](int at, const void* src, int size) {
#pragma unroll
                    for (int q = 0; q < size; ++q) copy16(to + (at + j * size + q) * lap, static_cast<const char*>(src) + 16 * q);
                };
                put(oX, a.out + i, kR);
                put(oN, a.dh + i, kT);
                put(oD, a.dout + i, kR);
                put(oY, a.y + i, kT);
            }
        }
        copies_commit();
    };
    auto get = [&](auto type, int at, const char* held, int j, float (&o)[VE]) {
        using T = decltype(type);
        constexpr int size = VE * sizeof(T) / 16;
        Pack<T, VE> p;
#pragma unroll
        for (int q = 0; q < size; ++q) reinterpret_cast<uint4*>(&p)[q] = *reinterpret_cast<const uint4*>(held + (at + j * size + q) * lap);
        unpack(p, o);
    };
    const bool sums_dy = POST && a.need_dy;
    auto sums = [&](const float4& st, const char* held, float4 (*to)[32]) {
        Sum p[4 * Q];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (col + j * step >= cols) continue;
            float x[VE], g[VE], w[VE];
            get(TR{}, oX, held, j, x);
            get(TY{}, oN, held, j, g);
            kept(0, j, w);
            vfma(x, x, st.x, st.y);
            vmul(g, g, w);
            p[0].template fma<VE>(g, x);
            if (L) p[1].add(g);
            if (sums_dy) {
                float q[VE], y[VE], d[VE];
                kept(1, j, q);
                get(TR{}, oD, held, j, d);
                get(TY{}, oY, held, j, y);
                vfma(y, y, st.z, st.w);
                vmul(y, y, q);
                vfma(d, g, st.x, d);
                p[2].template fma<VE>(y, d);
                p[3].template fma<VE>(y, x);
                if constexpr (Q == 2) {
                    p[4].add(y);
                    p[5].template fma<VE>(q, d);
                    p[6].template fma<VE>(q, x);
                    p[7].add(q);
                }
            }
        }
        float s[4 * Q];
#pragma unroll
        for (int k = 0; k < 4 * Q; ++k) s[k] = p[k].total();
        sums_put<Q>(s, to);
    };

    if (t0 < t1) {
        for (int k = 0; k < stages - 1; ++k) fetch(t0 + k, k);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = col + j * step;
            if (c >= cols) continue;
            float o[VE], g[VE];
            load_v<TY, VE>(a.w, a.vec_f32, c, o);
            keep(0, j, o);
#pragma unroll
            for (int k = 0; k < VE; ++k) o[k] = scale;
            if (POST) {
                load_v<TY, VE>(a.pw, a.vec_f32, c, g);
                vmul(o, o, g);
            }
            if (a.gate) {
                load_v<TY, VE>(a.gate, a.gate_f32, gate_row + c, g);
                vmul(o, o, g);
            }
            keep(1, j, o);
        }
        copies_wait(stages - 2);
        float4 st = a.stats[t0];
        int stage = 0, flip = 0;
        sums(st, mine, ws[0]);
        for (int64_t t = t0; t < t1; ++t) {
            const char* const held = mine + stage * stage_bytes;
            const int after = stage + 1 == stages ? 0 : stage + 1;
            fetch(t + stages - 1, stage == 0 ? stages - 1 : stage - 1);
            copies_wait(stages - 2);  // row t + 1 is here
            const float4 next = a.stats[min(t + 1, t1 - 1)];
            if (warps > 1) __syncthreads();
            else __syncwarp();
            float s[4 * Q];
            sums_get<Q>(s, warps, ws[flip]);
            flip ^= 1;
            if (t + 1 < t1) sums(next, mine + after * stage_bytes, ws[flip]);
            const float c2 = s[0] * inv_d, c1 = L && a.layer ? s[1] * inv_d : 0.f;
            float e1 = 0.f, e2 = 0.f;
            if (POST) {
                e2 = s[2] - st.x * c2 * s[3];
                if constexpr (Q == 2) {
                    e2 -= st.x * c1 * s[4];
                    e1 = a.layer ? (s[5] - st.x * (c2 * s[6] + c1 * s[7])) * inv_d : 0.f;
                }
                e2 *= inv_d;
            }
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = col + j * step;
                if (c >= cols) continue;
                const int64_t at = t * a.D + c;
                float x[VE], g[VE], d[VE], w[VE], y[VE];
                get(TR{}, oX, held, j, x);
                get(TY{}, oN, held, j, g);
                get(TR{}, oD, held, j, d);
                kept(0, j, w);
                vfma(x, x, st.x, st.y);
                vfma(aw[j], g, x, aw[j]);
                if (L) vadd(ab[j], ab[j], g);
                if (L) vfma(x, x, -c2, -c1);
                else vmul(x, x, -c2);
                vfma(g, g, w, x);
                vfma(d, g, st.x, d);
                store_f<TR, VE>(a.dr + at, d);
                get(TY{}, oY, held, j, y);
                if (POST) vfma(y, y, st.z, st.w);
                vfma(s1[j], d, y, s1[j]);
                if (L) vadd(s0[j], s0[j], d);
                if (a.need_dy) {
                    kept(1, j, w);
                    if (POST) {
                        if (L) vfma(y, y, -e2, -e1);
                        else vmul(y, y, -e2);
                        vfma(d, d, w, y);
                        vmul(d, d, st.z);
                    } else {
                        vmul(d, d, w);
                    }
                    store_f<TY, VE>(a.dy + at, d);
                }
            }
            st = next;
            stage = after;
        }
    }
    const int64_t plane = a.ctas * a.D;
    float as = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = col + j * step;
        if (c >= cols) continue;
        float* part = a.part + blockIdx.x * a.D + c;
        store_f<float, VE>(part, aw[j]);
        if constexpr (L) store_f<float, VE>(part + plane, ab[j]);
        float g[VE], u[VE], o[VE];
#pragma unroll
        for (int k = 0; k < VE; ++k) g[k] = 1.f;
        if (a.gate) load_v<TY, VE>(a.gate, a.gate_f32, gate_row + c, g);
        if constexpr (POST) {
            vmul(o, g, s1[j]);
            vmul(o, o, scale);
            store_f<float, VE>(part + 2 * plane, o);
            if constexpr (L) {
                vmul(o, g, s0[j]);
                vmul(o, o, scale);
                store_f<float, VE>(part + 3 * plane, o);
            }
            load_v<TY, VE>(a.pw, a.vec_f32, c, o);
            vmul(u, o, s1[j]);
            if constexpr (L) {
                if (a.pb) {
                    load_v<TY, VE>(a.pb, a.vec_f32, c, o);
                    vfma(u, o, s0[j], u);
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < VE; ++k) u[k] = s1[j][k];
        }
#pragma unroll
        for (int k = 0; k < VE; ++k) as = fmaf(g[k], u[k], as);
        if (a.need_gate) {
            vmul(u, u, scale);
            store_f<float, VE>(part + 4 * plane, u);
        }
    }
    if (a.need_scale) {
        float z[4 * Q] = {as};
        __syncthreads();
        sums_put<Q>(z, ws[0]);
        __syncthreads();
        sums_get<Q>(z, warps, ws[0]);
        if (threadIdx.x == 0) a.part_s[blockIdx.x] = z[0];
    }
}

// dst[g][c] = sum over the CTAs of run g of part[cta][c]: 32 columns a CTA,
// 32 rows of threads striding over the CTAs, joined in a fixed order.
struct Reduce {
    const float* src;
    void* dst;
    int64_t n, seg, groups;
    int f32;
};
struct ReduceList {
    Reduce r[6];
};
template <typename TY>
__global__ void __launch_bounds__(1024)
norm_reduce_kernel(ReduceList list) {
    __shared__ float s[32][33];
    const Reduce q = list.r[blockIdx.z];
    if (q.dst == nullptr) return;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x;
    for (int64_t g = blockIdx.y; g < q.groups; g += gridDim.y) {
        float a = 0.f;
        if (c < q.n)
#pragma unroll 8
            for (int k = threadIdx.y; k < q.seg; k += 32) a += q.src[(g * q.seg + k) * q.n + c];
        __syncthreads();
        s[threadIdx.y][threadIdx.x] = a;
        __syncthreads();
        a = s[threadIdx.x][threadIdx.y];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
        const int64_t cc = static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.y;
        if (threadIdx.x == 0 && cc < q.n) {
            if (q.f32) static_cast<float*>(q.dst)[g * q.n + cc] = a;
            else static_cast<TY*>(q.dst)[g * q.n + cc] = from_f<TY>(a);
        }
    }
}

template <typename TY, typename TR>
bool wide_ok(const sl_norm_args& n) {
    constexpr int64_t ve = 16 / sizeof(TY);
    if (n.cols % ve) return false;
    for (const void* q : {n.y, n.residual, n.weight, n.bias, n.gate, n.post_weight, n.post_bias, n.dout, n.dh,
                          static_cast<const void*>(n.out), static_cast<const void*>(n.h), static_cast<const void*>(n.dresidual),
                          static_cast<const void*>(n.dy), static_cast<const void*>(n.dgate)})
        if (off_by(q, 16)) return false;
    return true;
}

template <typename TY, typename TR>
Args<TY, TR> make_args(const sl_norm_args& n) {
    Args<TY, TR> a{};
    a.y = static_cast<const TY*>(n.y);
    a.r = static_cast<const TR*>(n.residual);
    a.w = n.weight; a.b = n.bias; a.gate = n.gate; a.pw = n.post_weight; a.pb = n.post_bias;
    a.out = static_cast<TR*>(n.out);
    a.h = static_cast<TY*>(n.h);
    a.stats = reinterpret_cast<float4*>(n.stats);
    a.scale_dev = n.scale_dev;
    a.scale = n.scale; a.eps = n.eps; a.post_eps = n.post_eps;
    a.T = n.rows; a.D = n.cols; a.gate_rows = n.gate ? n.rows / n.gate_groups : 1;
    a.layer = n.kind == SL_NORM_LAYER; a.vec_f32 = n.weight_dtype == SL_F32; a.gate_f32 = n.gate_dtype == SL_F32;
    a.dout = static_cast<const TR*>(n.dout);
    a.dh = static_cast<const TY*>(n.dh);
    a.dr = static_cast<TR*>(n.dresidual);
    a.dy = static_cast<TY*>(n.dy);
    a.dgate = n.dgate;
    a.need_dy = n.dy != nullptr; a.need_gate = n.dgate != nullptr; a.need_scale = n.dscale != nullptr;
    return a;
}

// f(vector width, vectors a thread) as constants.
template <typename TY, typename F>
int with_plan(const Plan& p, F f) {
    constexpr int W = 16 / sizeof(TY);
    using std::integral_constant;
#define SL_NORM_CASE(VE, NV) \
    if (p.ve == VE && p.nv <= NV) return f(integral_constant<int, VE>{}, integral_constant<int, NV>{});
    SL_NORM_CASE(W, 1)
    SL_NORM_CASE(W, 2)
    SL_NORM_CASE(W, 4)
    if constexpr (W == 4) {
        SL_NORM_CASE(W, 6)
        SL_NORM_CASE(W, 8)
    }
    SL_NORM_CASE(1, 4)
    SL_NORM_CASE(1, 32)
#undef SL_NORM_CASE
    return fail(SL_ERR_UNSUPPORTED, "sl_norm: no kernel for this width");
}
// f(vector width, vectors a thread, whether rows wait in shared memory).
template <typename TY, typename F>
int with_full_plan(const Plan& p, F f) {
    constexpr int W = 16 / sizeof(TY);
    using std::integral_constant;
    if (p.ve == W && p.ve * p.nv <= 8) return f(integral_constant<int, W>{}, integral_constant<int, 8 / W>{}, std::true_type{});
    if (p.ve == W) return f(integral_constant<int, W>{}, integral_constant<int, 32 / W>{}, std::false_type{});
    if (p.nv <= 4) return f(integral_constant<int, 1>{}, integral_constant<int, 4>{}, std::false_type{});
    return f(integral_constant<int, 1>{}, integral_constant<int, 32>{}, std::false_type{});
}

template <typename TY, typename TR>
int forward(const sl_norm_args& n, cudaStream_t s) {
    const Args<TY, TR> a = make_args<TY, TR>(n);
    const Plan p = forward_plan(n.cols, wide_ok<TY, TR>(n), sizeof(TY));
    const dim3 block(32 * p.warps, p.warps == 1 ? 4 : 1);
    const int64_t beside = std::max<int64_t>(1, (p.ve * p.nv <= 16 ? 1024 : 512) / (block.x * block.y));
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>((n.rows + block.y - 1) / block.y, num_sms() * beside));
    auto launch = [&](auto tv) {
        using TV = decltype(tv);
        return with_plan<TY>(p, [&](auto ve, auto nv) {
            if (n.post_weight) norm_fwd_kernel<TY, TR, TV, ve, nv, true><<<grid, block, 0, s>>>(a);
            else norm_fwd_kernel<TY, TR, TV, ve, nv, false><<<grid, block, 0, s>>>(a);
            SL_RETURN_IF_LAUNCH_FAILED("sl_norm_forward");
            return static_cast<int>(SL_OK);
        });
    };
    if constexpr (sizeof(TY) == 2)
        if (n.weight_dtype == SL_F32) return launch(float{});
    return launch(TY{});
}

template <typename TY, typename TR>
int backward(const sl_norm_args& n, cudaStream_t s) {
    Args<TY, TR> a = make_args<TY, TR>(n);
    const bool full = n.post_weight || n.gate || n.dscale || n.cols > kSimpleCols;
    const Plan p = backward_plan(n.cols, wide_ok<TY, TR>(n), sizeof(TY), full);
    const dim3 block(32 * p.warps, backward_rows(p, full));
    const Split sp = make_split(a.T, a.gate_rows, ctas_wanted(p, full), a.need_gate);
    a.rows_per_cta = sp.rows; a.ctas = sp.ctas; a.seg = sp.seg; a.gate_direct = sp.direct;
    a.part = static_cast<float*>(n.workspace);
    a.part_s = a.part + 5 * sp.ctas * a.D;
    const unsigned grid = static_cast<unsigned>(sp.ctas);
    int rc;
    if (full) {
        rc = with_full_plan<TY>(p, [&](auto ve, auto nv, auto ring) {
            using G = Ring<TY, TR, ve, nv>;
            size_t bytes = 0;
            int stages = 1;
            // Gates of whole runs of rows: one run a CTA (always so where its gradient is asked for).
            const bool shared = !n.gate || (a.gate_rows > 1 && (a.gate_rows == a.T || sp.seg > 0));
            if constexpr (ring) {
                // This row, the next, and one or two on their way.  Three fit at every width and type; the tightest is a
                // 16-bit gate a row over a 32-bit stream at 4096 columns, 7 granules x 8 KB a row beside 3 vectors of 16 KB.
                const size_t lap = 16 * block.x, stage = G::granules(!shared && G::kGates && a.gate_rows == 1 && !a.gate_f32) * lap;
                // (vectors; the last of four is a gate that rows share)
                bytes = (shared ? 2 : G::kVectors ? (a.gate_rows == 1 ? 3 : 4) : 0) * G::kVec * lap;
                stages = static_cast<int>(std::min<size_t>(4, (kFullSmem - bytes) / stage));
                if (stages < 3) return fail(SL_ERR_UNSUPPORTED, "sl_norm_backward: rows do not fit");
                bytes += stages * stage;
            }
            auto go = [&](auto kernel) {
                if (bytes > 40 * 1024)  // with what the kernel has besides, beyond the default
                    if (int e = cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)), "sl_norm_backward"))
                        return e;
                ++g_launched;
                kernel<<<grid, block, bytes, s>>>(a, stages);
                SL_RETURN_IF_LAUNCH_FAILED("sl_norm_backward");
                return static_cast<int>(SL_OK);
            };
            const bool l = a.layer || n.bias || n.post_bias;
            if constexpr (ring) {
                if (shared && n.post_weight) return l ? go(norm_bwd_shared_kernel<TY, TR, ve, nv, true, true>) : go(norm_bwd_shared_kernel<TY, TR, ve, nv, true, false>);
                if (shared) return l ? go(norm_bwd_shared_kernel<TY, TR, ve, nv, false, true>) : go(norm_bwd_shared_kernel<TY, TR, ve, nv, false, false>);
            }
            if (n.post_weight) return l ? go(norm_bwd_full_kernel<TY, TR, ve, nv, true, true, ring>) : go(norm_bwd_full_kernel<TY, TR, ve, nv, true, false, ring>);
            return l ? go(norm_bwd_full_kernel<TY, TR, ve, nv, false, true, ring>) : go(norm_bwd_full_kernel<TY, TR, ve, nv, false, false, ring>);
        });
    } else {
        const size_t join = block.y > 1 ? 2 * sizeof(float) * n.cols : 0;
        rc = with_plan<TY>(p, [&](auto ve, auto nv) {
            ++g_launched;
            norm_bwd_kernel<TY, TR, ve, nv><<<grid, block, join, s>>>(a);
            SL_RETURN_IF_LAUNCH_FAILED("sl_norm_backward");
            return static_cast<int>(SL_OK);
        });
    }
    if (rc) return rc;
    const int64_t plane = sp.ctas * a.D;
    ReduceList l{};
    void* dst[4] = {n.dweight, n.dbias, n.dpost_weight, n.dpost_bias};
    for (int k = 0; k < 4; ++k) l.r[k] = {a.part + k * plane, dst[k], a.D, sp.ctas, 1, a.vec_f32};
    if (a.need_gate && sp.seg) l.r[4] = {a.part + 4 * plane, n.dgate, a.D, sp.seg, sp.ctas / sp.seg, a.gate_f32};
    l.r[5] = {a.part_s, n.dscale, 1, sp.ctas, 1, 1};
    bool any = false;
    for (const Reduce& r : l.r) any |= r.dst != nullptr;
    if (!any) return SL_OK;
    const int64_t groups = std::max<int64_t>(1, l.r[4].groups);
    const dim3 grid2(static_cast<unsigned>((a.D + 31) / 32), static_cast<unsigned>(std::min<int64_t>(groups, 4096)), 6);
    ++g_launched;
    norm_reduce_kernel<TY><<<grid2, dim3(32, 32), 0, s>>>(l);
    SL_RETURN_IF_LAUNCH_FAILED("sl_norm_backward");
    return SL_OK;
}

}  // namespace
}  // namespace norm

template <typename TY>
int norm_forward(const sl_norm_args& n, cudaStream_t s) {
    if constexpr (sizeof(TY) == 2)
        if (n.residual_dtype == SL_F32) return norm::forward<TY, float>(n, s);
    return norm::forward<TY, TY>(n, s);
}
template <typename TY>
int norm_backward(const sl_norm_args& n, cudaStream_t s) {
    if constexpr (sizeof(TY) == 2)
        if (n.residual_dtype == SL_F32) return norm::backward<TY, float>(n, s);
    return norm::backward<TY, TY>(n, s);
}

}  // namespace slb
