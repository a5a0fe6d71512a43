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
#include <algorithm>
#include <type_traits>

#include "typed.cuh"

namespace slb {
namespace {

constexpr int kMaxThreads = 512;

template <typename TY, typename TR>
struct Args {
    const TY* y;
    const TR* r;
    const void *w, *b, *gate, *pw, *pb;
    TR* out;
    TY* h;
    float* stats;  // [4][T]: mean, 1/deviation of out's norm; of y's
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

// Sums of two values over the CTA, the same in every thread.  `ws` holds two
// buffers that alternate, so one barrier a call is enough.
__device__ __forceinline__ void row_sum2(float& a, float& b, float2* ws, int& flip) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    const int warps = blockDim.x >> 5;
    if (warps == 1) return;
    float2* w = ws + flip * 32;
    flip ^= 1;
    if ((threadIdx.x & 31) == 0) w[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    a = b = 0.f;
    for (int k = 0; k < warps; ++k) {
        const float2 q = w[k];
        a += q.x;
        b += q.y;
    }
}

template <int NV, int VE>
__device__ __forceinline__ void row_stats(const float (&v)[NV][VE], const bool (&in)[NV], int layer, float inv_d,
                                          float eps, float2* ws, int& flip, float& mean, float& rstd) {
    float a = 0.f, z = 0.f;
    mean = 0.f;
    if (layer) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < VE; ++k) a += in[j] ? v[j][k] : 0.f;
        row_sum2(a, z, ws, flip);
        mean = a * inv_d;
        a = 0.f;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < VE; ++k) {
            const float c = in[j] ? v[j][k] - mean : 0.f;
            a = fmaf(c, c, a);
        }
    row_sum2(a, z, ws, flip);
    rstd = 1.f / sqrtf(fmaf(a, inv_d, eps));
}

template <typename TY, typename TR, int VE, int NV, bool POST>
__global__ void __launch_bounds__(kMaxThreads)
norm_fwd_kernel(Args<TY, TR> a) {
    __shared__ float2 ws[64];
    int flip = 0;
    const float inv_d = 1.f / static_cast<float>(a.D);
    const float scale = a.scale_dev ? *a.scale_dev : a.scale;
    int64_t col[NV];
    bool in[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        col[j] = (static_cast<int64_t>(j) * blockDim.x + threadIdx.x) * VE;
        in[j] = col[j] < a.D;
    }
    for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
        float y[NV][VE], r[NV][VE];
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (in[j]) {
                load_f<TY, VE>(a.y + t * a.D + col[j], y[j]);
                load_f<TR, VE>(a.r + t * a.D + col[j], r[j]);
            }
        float mean, rstd;
        if (POST) {
            row_stats<NV, VE>(y, in, a.layer, inv_d, a.post_eps, ws, flip, mean, rstd);
            if (a.stats && threadIdx.x == 0) {
                a.stats[2 * a.T + t] = mean;
                a.stats[3 * a.T + t] = rstd;
            }
        }
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (in[j]) {
                if (POST) {
                    float w[VE], b[VE];
                    load_v<TY, VE>(a.pw, a.vec_f32, col[j], w);
#pragma unroll
                    for (int k = 0; k < VE; ++k) y[j][k] = (y[j][k] - mean) * rstd * w[k];
                    if (a.pb) {
                        load_v<TY, VE>(a.pb, a.vec_f32, col[j], b);
#pragma unroll
                        for (int k = 0; k < VE; ++k) y[j][k] += b[k];
                    }
                }
                if (a.gate) {
                    float g[VE];
                    load_v<TY, VE>(a.gate, a.gate_f32, (t / a.gate_rows) * a.D + col[j], g);
#pragma unroll
                    for (int k = 0; k < VE; ++k) y[j][k] *= g[k];
                }
                // the stream is held in its own type, and the norm reads what it holds
#pragma unroll
                for (int k = 0; k < VE; ++k) r[j][k] = to_f(from_f<TR>(fmaf(scale, y[j][k], r[j][k])));
                store_f<TR, VE>(a.out + t * a.D + col[j], r[j]);
            }
        row_stats<NV, VE>(r, in, a.layer, inv_d, a.eps, ws, flip, mean, rstd);
        if (a.stats && threadIdx.x == 0) {
            a.stats[t] = mean;
            a.stats[a.T + t] = rstd;
        }
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (in[j]) {
                float w[VE], b[VE], o[VE];
                load_v<TY, VE>(a.w, a.vec_f32, col[j], w);
#pragma unroll
                for (int k = 0; k < VE; ++k) o[k] = (r[j][k] - mean) * rstd * w[k];
                if (a.b) {
                    load_v<TY, VE>(a.b, a.vec_f32, col[j], b);
#pragma unroll
                    for (int k = 0; k < VE; ++k) o[k] += b[k];
                }
                store_f<TY, VE>(a.h + t * a.D + col[j], o);
            }
    }
}

// A CTA walks rows_per_cta rows and keeps the vectors' gradients of its
// columns in registers; they are written once per CTA and summed over the
// CTAs in order by norm_reduce_kernel, so they do not depend on timing.
template <typename TY, typename TR, int VE, int NV, bool POST>
__global__ void __launch_bounds__(kMaxThreads)
norm_bwd_kernel(Args<TY, TR> a) {
    __shared__ float2 ws[64];
    int flip = 0;
    const float inv_d = 1.f / static_cast<float>(a.D);
    const float scale = a.scale_dev ? *a.scale_dev : a.scale;
    int64_t col[NV];
    bool in[NV];
    float aw[NV][VE] = {}, ab[NV][VE] = {}, apw[NV][VE] = {}, apb[NV][VE] = {}, ag[NV][VE] = {};
    float as = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        col[j] = (static_cast<int64_t>(j) * blockDim.x + threadIdx.x) * VE;
        in[j] = col[j] < a.D;
    }
    // With gates shared by whole runs of rows (seg CTAs to a run) no CTA
    // crosses a run's end.
    int64_t t0, t1;
    if (a.seg > 0) {
        const int64_t run = blockIdx.x / a.seg, part = blockIdx.x % a.seg;
        t0 = run * a.gate_rows + part * a.rows_per_cta;
        t1 = min(t0 + a.rows_per_cta, min((run + 1) * a.gate_rows, a.T));
    } else {
        t0 = blockIdx.x * a.rows_per_cta;
        t1 = min(t0 + a.rows_per_cta, a.T);
    }
    const bool reads_y = POST || a.need_gate || a.need_scale;
    for (int64_t t = t0; t < t1; ++t) {
        float x[NV][VE], d[NV][VE], dn[NV][VE], y[NV][VE];
        const float mean = a.stats[t], rstd = a.stats[a.T + t];
        float c1 = 0.f, c2 = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (in[j]) {
                const int64_t i = t * a.D + col[j];
                load_f<TR, VE>(a.out + i, x[j]);
                if (a.dh) load_f<TY, VE>(a.dh + i, dn[j]);
                if (a.dout) load_f<TR, VE>(a.dout + i, d[j]);
                if (reads_y) load_f<TY, VE>(a.y + i, y[j]);
            }
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (in[j]) {
                float w[VE];
                load_v<TY, VE>(a.w, a.vec_f32, col[j], w);
#pragma unroll
                for (int k = 0; k < VE; ++k) {
                    if (!a.dh) dn[j][k] = 0.f;
                    if (!a.dout) d[j][k] = 0.f;
                    x[j][k] = (x[j][k] - mean) * rstd;
                    aw[j][k] = fmaf(dn[j][k], x[j][k], aw[j][k]);
                    ab[j][k] += dn[j][k];
                    dn[j][k] *= w[k];
                    c1 += dn[j][k];
                    c2 = fmaf(dn[j][k], x[j][k], c2);
                }
            }
        row_sum2(c1, c2, ws, flip);
        c1 = a.layer ? c1 * inv_d : 0.f;
        c2 *= inv_d;
        float pmean = 0.f, prstd = 0.f;
        if (POST) {
            pmean = a.stats[2 * a.T + t];
            prstd = a.stats[3 * a.T + t];
        }
        float e1 = 0.f, e2 = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (in[j]) {
                const int64_t i = t * a.D + col[j];
#pragma unroll
                for (int k = 0; k < VE; ++k) d[j][k] = fmaf(rstd, dn[j][k] - fmaf(x[j][k], c2, c1), d[j][k]);
                store_f<TR, VE>(a.dr + i, d[j]);
                float pw[VE], pb[VE], g[VE];
                if (POST) {
                    load_v<TY, VE>(a.pw, a.vec_f32, col[j], pw);
                    if (a.pb) load_v<TY, VE>(a.pb, a.vec_f32, col[j], pb);
                }
                if (a.gate) load_v<TY, VE>(a.gate, a.gate_f32, (t / a.gate_rows) * a.D + col[j], g);
#pragma unroll
                for (int k = 0; k < VE; ++k) {
                    float u = reads_y ? y[j][k] : 0.f;
                    if (POST) {
                        y[j][k] = (y[j][k] - pmean) * prstd;
                        u = a.pb ? fmaf(y[j][k], pw[k], pb[k]) : y[j][k] * pw[k];
                    }
                    const float gk = a.gate ? g[k] : 1.f;
                    as = fmaf(d[j][k], gk * u, as);
                    const float du = scale * d[j][k];
                    if (a.need_gate) {
                        const float dg = du * u;
                        if (a.gate_rows == 1) g[k] = dg;
                        else ag[j][k] += dg;
                    }
                    d[j][k] = du * gk;
                    if (POST) {
                        apw[j][k] = fmaf(d[j][k], y[j][k], apw[j][k]);
                        apb[j][k] += d[j][k];
                        d[j][k] *= pw[k];
                        e1 += d[j][k];
                        e2 = fmaf(d[j][k], y[j][k], e2);
                    }
                }
                if (a.need_gate && a.gate_rows == 1) {
                    if (a.gate_f32) store_f<float, VE>(static_cast<float*>(a.dgate) + i, g);
                    else store_f<TY, VE>(static_cast<TY*>(a.dgate) + i, g);
                }
                if (!POST && a.need_dy) store_f<TY, VE>(a.dy + i, d[j]);
            }
        if (POST && a.need_dy) {
            row_sum2(e1, e2, ws, flip);
            e1 = a.layer ? e1 * inv_d : 0.f;
            e2 *= inv_d;
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (in[j]) {
#pragma unroll
                    for (int k = 0; k < VE; ++k) d[j][k] = prstd * (d[j][k] - fmaf(y[j][k], e2, e1));
                    store_f<TY, VE>(a.dy + t * a.D + col[j], d[j]);
                }
        }
        if (a.gate_direct && (t + 1 == t1 || (t + 1) % a.gate_rows == 0)) {  // a run of rows ends
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (in[j]) {
                    const int64_t i = (t / a.gate_rows) * a.D + col[j];
                    if (a.gate_f32) store_f<float, VE>(static_cast<float*>(a.dgate) + i, ag[j]);
                    else store_f<TY, VE>(static_cast<TY*>(a.dgate) + i, ag[j]);
#pragma unroll
                    for (int k = 0; k < VE; ++k) ag[j][k] = 0.f;
                }
        }
    }
    const int64_t plane = a.ctas * a.D;
#pragma unroll
    for (int j = 0; j < NV; ++j)
        if (in[j]) {
            float* q = a.part + blockIdx.x * a.D + col[j];
            store_f<float, VE>(q, aw[j]);
            store_f<float, VE>(q + plane, ab[j]);
            if (POST) {
                store_f<float, VE>(q + 2 * plane, apw[j]);
                store_f<float, VE>(q + 3 * plane, apb[j]);
            }
            if (a.need_gate && a.seg > 0) store_f<float, VE>(q + 4 * plane, ag[j]);
        }
    if (a.need_scale) {
        float z = 0.f;
        row_sum2(as, z, ws, flip);
        if (threadIdx.x == 0) a.part_s[blockIdx.x] = as;
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
            for (int64_t k = threadIdx.y; k < q.seg; k += 32) a += q.src[(g * q.seg + k) * q.n + c];
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

struct Plan {
    int ve, nv, threads;
};

Plan make_plan(int64_t D, bool wide, int64_t elem) {
    const int ve = wide ? static_cast<int>(16 / elem) : 1;
    Plan p{ve, 1, 0};
    const int64_t vecs = (D + ve - 1) / ve;
    while (p.nv < 32 && (vecs + p.nv - 1) / p.nv > kMaxThreads) p.nv *= 2;
    p.threads = static_cast<int>(((vecs + p.nv - 1) / p.nv + 31) / 32 * 32);
    return p;
}

// The backward pass's split of the rows over CTAs.
struct Split {
    int64_t rows, ctas, seg;
    bool direct;
};
Split make_split(int64_t T, int64_t gate_rows, int threads, bool need_gate) {
    const int64_t per_sm = std::max<int64_t>(1, 1024 / threads);
    const int64_t want = static_cast<int64_t>(num_sms()) * per_sm;
    Split s{(T + want - 1) / want, 0, 0, false};
    if (s.rows < 1) s.rows = 1;
    if (need_gate && gate_rows > 1) {
        if (gate_rows >= s.rows) {
            s.seg = (gate_rows + s.rows - 1) / s.rows;
            s.rows = (gate_rows + s.seg - 1) / s.seg;
            s.ctas = s.seg * (T / gate_rows);
            return s;
        }
        s.rows = (s.rows + gate_rows - 1) / gate_rows * gate_rows;
        s.direct = true;
    }
    s.ctas = (T + s.rows - 1) / s.rows;
    return s;
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
    a.stats = n.stats;
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
    if (p.ve == W) {
        if (p.nv == 1) return f(integral_constant<int, W>{}, integral_constant<int, 1>{});
        if (p.nv == 2) return f(integral_constant<int, W>{}, integral_constant<int, 2>{});
        if (p.nv == 4 || W == 8) return f(integral_constant<int, W>{}, integral_constant<int, 4>{});
        return f(integral_constant<int, W>{}, integral_constant<int, W == 8 ? 4 : 8>{});
    }
    if (p.nv <= 4) return f(integral_constant<int, 1>{}, integral_constant<int, 4>{});
    return f(integral_constant<int, 1>{}, integral_constant<int, 32>{});
}

template <typename TY, typename TR>
int forward(const sl_norm_args& n, cudaStream_t s) {
    const Args<TY, TR> a = make_args<TY, TR>(n);
    const Plan p = make_plan(n.cols, wide_ok<TY, TR>(n), sizeof(TY));
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(n.rows, INT_MAX));
    return with_plan<TY>(p, [&](auto ve, auto nv) {
        if (n.post_weight) norm_fwd_kernel<TY, TR, ve, nv, true><<<grid, p.threads, 0, s>>>(a);
        else norm_fwd_kernel<TY, TR, ve, nv, false><<<grid, p.threads, 0, s>>>(a);
        SL_RETURN_IF_LAUNCH_FAILED("sl_norm_forward");
        return static_cast<int>(SL_OK);
    });
}

template <typename TY, typename TR>
int backward(const sl_norm_args& n, cudaStream_t s) {
    Args<TY, TR> a = make_args<TY, TR>(n);
    const Plan p = make_plan(n.cols, wide_ok<TY, TR>(n), sizeof(TY));
    const Split sp = make_split(a.T, a.gate_rows, p.threads, a.need_gate);
    a.rows_per_cta = sp.rows; a.ctas = sp.ctas; a.seg = sp.seg; a.gate_direct = sp.direct;
    a.part = static_cast<float*>(n.workspace);
    a.part_s = a.part + 5 * sp.ctas * a.D;
    const int rc = with_plan<TY>(p, [&](auto ve, auto nv) {
        if (n.post_weight) norm_bwd_kernel<TY, TR, ve, nv, true><<<static_cast<unsigned>(sp.ctas), p.threads, 0, s>>>(a);
        else norm_bwd_kernel<TY, TR, ve, nv, false><<<static_cast<unsigned>(sp.ctas), p.threads, 0, s>>>(a);
        SL_RETURN_IF_LAUNCH_FAILED("sl_norm_backward");
        return static_cast<int>(SL_OK);
    });
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
    const dim3 grid(static_cast<unsigned>((a.D + 31) / 32), static_cast<unsigned>(std::min<int64_t>(groups, 4096)), 6);
    norm_reduce_kernel<TY><<<grid, dim3(32, 32), 0, s>>>(l);
    SL_RETURN_IF_LAUNCH_FAILED("sl_norm_backward");
    return SL_OK;
}

int check(const sl_norm_args* n, const char* fn, bool back) {
    SL_REQUIRE(n != nullptr, fn, "NULL arguments");
    SL_REQUIRE(n->rows >= 0 && n->cols >= 1 && n->cols <= SL_NORM_MAX_COLS, fn, "columns must be 1 to 16384");
    SL_REQUIRE(n->kind == SL_NORM_LAYER || n->kind == SL_NORM_RMS, fn, "unknown kind");
    SL_REQUIRE(known_dtype(n->dtype) && (n->residual_dtype == n->dtype || n->residual_dtype == SL_F32), fn, "unsupported residual type");
    SL_REQUIRE(n->weight_dtype == n->dtype || n->weight_dtype == SL_F32, fn, "unsupported weight type");
    SL_REQUIRE(!n->gate || n->gate_dtype == n->dtype || n->gate_dtype == SL_F32, fn, "unsupported gate type");
    SL_REQUIRE(!n->gate || n->rows == 0 || (n->gate_groups >= 1 && n->rows % n->gate_groups == 0), fn,
               "the rows must divide into the gate's rows");
    if (n->rows == 0) return SL_OK;
    SL_REQUIRE(n->weight && n->out, fn, "NULL operand");
    SL_REQUIRE(back || (n->y && n->residual && n->h), fn, "NULL operand");
    SL_REQUIRE(!back || (n->stats && n->dresidual && n->workspace), fn, "NULL operand");
    SL_REQUIRE(!back || n->y || !(n->post_weight || n->dgate || n->dscale), fn, "the block's output is needed");
    SL_REQUIRE(!n->dgate || n->gate, fn, "a gradient of a gate that is not there");
    const int64_t e = dtype_bytes(n->dtype), er = dtype_bytes(n->residual_dtype), ew = dtype_bytes(n->weight_dtype),
                  eg = dtype_bytes(n->gate ? n->gate_dtype : SL_F32);
    for (const void* q : {n->y, n->dh, static_cast<const void*>(n->h), static_cast<const void*>(n->dy)})
        SL_REQUIRE(!off_by(q, e), fn, "misaligned operand");
    for (const void* q : {n->residual, n->dout, static_cast<const void*>(n->out), static_cast<const void*>(n->dresidual)})
        SL_REQUIRE(!off_by(q, er), fn, "misaligned operand");
    for (const void* q : {n->weight, n->bias, n->post_weight, n->post_bias, static_cast<const void*>(n->dweight),
                          static_cast<const void*>(n->dbias), static_cast<const void*>(n->dpost_weight),
                          static_cast<const void*>(n->dpost_bias)})
        SL_REQUIRE(!off_by(q, ew), fn, "misaligned vector");
    SL_REQUIRE(!off_by(n->gate, eg) && !off_by(n->dgate, eg) && !off_by(n->workspace, 16) && !off_by(n->stats, 4), fn,
               "misaligned operand");
    return SL_OK;
}

template <typename F>
int with_types(const sl_norm_args& n, F f) {
    if (n.dtype == SL_F32) return f(float{}, float{});
    if (n.dtype == SL_BF16) return n.residual_dtype == SL_F32 ? f(__nv_bfloat16{}, float{}) : f(__nv_bfloat16{}, __nv_bfloat16{});
    return n.residual_dtype == SL_F32 ? f(__half{}, float{}) : f(__half{}, __half{});
}

}  // namespace
}  // namespace slb

using namespace slb;

extern "C" int64_t sl_norm_workspace_bytes(int64_t rows, int64_t cols, int64_t gate_groups) {
    if (rows <= 0 || cols <= 0 || cols > SL_NORM_MAX_COLS) return 0;
    // the most CTAs that make_split gives for any type and alignment, and a run's last CTA each
    const int threads = std::min({make_plan(cols, true, 2).threads, make_plan(cols, true, 4).threads, make_plan(cols, false, 4).threads});
    const int64_t most = static_cast<int64_t>(num_sms()) * std::max(1, 1024 / threads) + std::max<int64_t>(gate_groups, 1);
    return (5 * cols + 1) * std::min(rows, most) * 4 + 16;
}

extern "C" int sl_norm_forward(const sl_norm_args* n, void* stream) {
    if (int rc = check(n, "sl_norm_forward", false)) return rc;
    if (n->rows == 0) return SL_OK;
    return with_types(*n, [&](auto ty, auto tr) { return forward<decltype(ty), decltype(tr)>(*n, as_stream(stream)); });
}

extern "C" int sl_norm_backward(const sl_norm_args* n, void* stream) {
    if (int rc = check(n, "sl_norm_backward", true)) return rc;
    if (n->rows == 0) return SL_OK;
    return with_types(*n, [&](auto ty, auto tr) { return backward<decltype(ty), decltype(tr)>(*n, as_stream(stream)); });
}
