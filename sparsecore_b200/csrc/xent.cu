// Softmax cross entropy of logits z = x . W^T over a vocabulary, without the
// logits ever being whole, and its gradients.
//
//   m_t = max_v z_tv      s_t = sum_v exp(z_tv - m_t)
//   loss_t = m_t + ln s_t - z_t,target
//   G_tv = exp(z_tv - m_t) / s_t - [v = target_t]       (times the loss's gradient)
//   dx = G . W            dW = G^T . x
//
// Forward: a matrix product whose epilogue leaves, of every 128 columns of
// a row, their maximum and the sum of exponentials below it; a second small
// kernel joins them.  Backward: pieces of the vocabulary, each with its
// logits made again, turned into G in the epilogue, and multiplied twice.
//
// 16-bit inputs are multiplied as they are.  32-bit ones are split into two
// fp16 planes, a = 2^-k (a_hi + a_lo) with 22 bits between them (2^-k from
// the operand's largest value), and three products hi.hi, hi.lo, lo.hi are
// summed in 32 bits: the result is as exact as a 32-bit product's, on the
// 16-bit matrix units.
#include <algorithm>

#include "xent.cuh"

namespace slb {
namespace xent {
namespace {

constexpr int kThreads = 256;

struct Layout {
    int64_t dp;                              // columns of a plane's row
    int64_t tgt, row_max, row_inv, x, w, prep;  // offsets in `prep`, and its size
    int64_t zt, part, fwd;                   // in the forward call's scratch
    int64_t piece, gp;                       // vocabulary columns of a piece, of a G row
    int64_t g, acc, slabs, slab_floats, bwd; // in the backward call's
};

int64_t up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

Layout layout(int64_t T, int64_t D, int64_t V, int dtype, bool copy_w) {
    Layout l{};
    const int64_t planes = dtype == SL_F32 ? 2 : 1;
    l.dp = up(D, 64);
    int64_t o = 256;
    auto take = [&](int64_t bytes) { const int64_t at = o; o += up(bytes, 256); return at; };
    l.tgt = take(4 * T);
    l.row_max = take(4 * T);
    l.row_inv = take(4 * T);
    l.x = take(planes * T * l.dp * 2);
    l.w = take(copy_w ? planes * V * l.dp * 2 : 0);
    l.prep = o;
    o = 0;
    l.zt = take(4 * T);
    l.part = take((V + kPart - 1) / kPart * T * 8);
    take(8 * ((T + 7) / 8));  // the finish's sums
    l.fwd = o;
    o = 0;
    // A piece's G: 256 MB at most, a multiple of the tile's 256 columns.
    const int64_t most = std::max<int64_t>(256, ((int64_t(256) << 20) / (T * planes * 2)) / 256 * 256);
    const int64_t pieces = std::max<int64_t>(1, (V + most - 1) / most);
    l.piece = up((V + pieces - 1) / pieces, 256);
    l.gp = up(std::min(l.piece, V), 64);
    l.g = take(planes * T * l.gp * 2);
    l.acc = take(V > l.piece ? 4 * T * D : 0);
    l.slab_floats = kSlabFloats;
    l.slabs = take(4 * l.slab_floats);
    l.bwd = o;
    return l;
}

// ── operands ──

// Largest finite magnitude of a 32-bit operand; the order of a maximum does
// not change it.
__global__ void __launch_bounds__(kThreads)
absmax_kernel(const float* __restrict__ a, int64_t rows, int64_t cols, const int64_t* __restrict__ targets,
              int64_t ignore, unsigned* out) {
    float m = 0.f;
    const int64_t n = rows * cols, step = static_cast<int64_t>(gridDim.x) * kThreads;
    for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; i < n; i += step) {
        if (targets && targets[i / cols] == ignore) continue;
        const float v = fabsf(a[i]);
        if (v <= 3.4028234e38f) m = fmaxf(m, v);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane_id() == 0 && m > 0.f) atomicMax(out, __float_as_uint(m));
}

// Rows of an operand as planes, padded with zeros to `dp` columns; rows of
// tokens that do not count become zeros, whatever they hold.
template <typename T>
__global__ void __launch_bounds__(kThreads)
planes_kernel(const T* __restrict__ src, int64_t rows, int64_t cols, int64_t dp, const unsigned* max_bits,
              const int* __restrict__ tgt, void* dst) {
    const int64_t n = rows * dp, step = static_cast<int64_t>(gridDim.x) * kThreads;
    const float scale = sizeof(T) == 4 ? exp2f(static_cast<float>(plane_exponent(*max_bits))) : 1.f;
    for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; i < n; i += step) {
        const int64_t r = i / dp, c = i - r * dp;
        const bool on = c < cols && !(tgt && tgt[r] == kIgnored);
        if constexpr (sizeof(T) == 4) {
            const float v = on ? src[r * cols + c] * scale : 0.f;
            const __half hi = __float2half_rn(v);
            static_cast<__half*>(dst)[i] = hi;
            static_cast<__half*>(dst)[n + i] = __float2half_rn(v - __half2float(hi));
        } else {
            static_cast<T*>(dst)[i] = on ? src[r * cols + c] : from_f<T>(0.f);
        }
    }
}

__global__ void __launch_bounds__(kThreads)
targets_kernel(const int64_t* __restrict__ targets, int64_t T, int64_t V, int64_t ignore, int* __restrict__ tgt,
               float* __restrict__ zt, Header* head) {
    const int64_t t = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x;
    bool on = false;
    if (t < T) {
        const int64_t v = targets[t];
        on = v != ignore;
        const bool bad = on && (v < 0 || v >= V);
        tgt[t] = !on ? kIgnored : bad ? kInvalid : static_cast<int>(v);
        zt[t] = bad ? __int_as_float(0x7fffffff) : 0.f;  // no such token: its loss is NaN
    }
    const int c = __popc(__ballot_sync(0xffffffffu, on));
    if (lane_id() == 0 && c) atomicAdd(&head->count, c);
}

// ── joining the partial sums ──

__global__ void __launch_bounds__(kThreads)
finish_kernel(Problem p, int64_t parts, float* __restrict__ rows, float* loss, double* sums, int mean) {
    __shared__ double s[kThreads / 32];
    __shared__ bool last;
    const int warp = threadIdx.x >> 5, lane = lane_id();
    const int64_t t = blockIdx.x * static_cast<int64_t>(kThreads / 32) + warp;
    double mine = 0.0;
    if (t < p.T) {
        float m = -INFINITY, sum = 0.f;
        for (int64_t k = lane; k < parts; k += 32) {
            const float2 q = p.part[k * p.T + t];
            const float n = fmaxf(m, q.x);
            // an empty side has m = -inf; equal infinities stay a NaN, as they are in the definition
            sum = (sum == 0.f ? 0.f : sum * expf(m - n)) + (q.y == 0.f ? 0.f : q.y * expf(q.x - n));
            m = n;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float qm = __shfl_xor_sync(0xffffffffu, m, o), qs = __shfl_xor_sync(0xffffffffu, sum, o);
            const float n = fmaxf(m, qm);
            sum = (sum == 0.f ? 0.f : sum * expf(m - n)) + (qs == 0.f ? 0.f : qs * expf(qm - n));
            m = n;
        }
        const int tg = p.tgt[t];
        const float l = tg == kIgnored ? 0.f : m + logf(sum) - p.zt[t];
        if (lane == 0) {
            p.row_max[t] = m;
            p.row_inv[t] = tg == kInvalid ? __int_as_float(0x7fffffff) : 1.f / sum;
            if (rows) rows[t] = l;
            mine = l;
        }
    }
    if (!loss) return;
    if (lane == 0) s[warp] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
        double a = 0.0;
        for (int k = 0; k < kThreads / 32; ++k) a += s[k];
        sums[blockIdx.x] = a;
        __threadfence();
        last = atomicAdd(&p.head->done, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    // The CTA that comes last adds all sums in their order, whoever it is.
    double a = 0.0;
    for (int64_t k = threadIdx.x; k < gridDim.x; k += kThreads) a += __ldcg(sums + k);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    __syncthreads();
    if (lane == 0) s[warp] = a;
    __syncthreads();
    if (threadIdx.x == 0) {
        a = 0.0;
        for (int k = 0; k < kThreads / 32; ++k) a += s[k];
        *loss = static_cast<float>(mean ? a / p.head->count : a);
        p.head->done = 0;
    }
}

__global__ void grad_scale_kernel(Header* head, const float* grad, int mean) {
    float g = grad ? *grad : __uint_as_float(head->max_g);
    if (mean) g = head->count ? g / static_cast<float>(head->count) : 0.f;
    head->g = g;
}

unsigned blocks_for(int64_t n) {
    return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>((n + kThreads - 1) / kThreads, num_sms() * 16)));
}

template <typename T>
void to_planes(const void* src, int64_t rows, int64_t cols, int64_t dp, const unsigned* bits, const int* tgt, void* dst,
               cudaStream_t s) {
    planes_kernel<T><<<blocks_for(rows * dp), kThreads, 0, s>>>(static_cast<const T*>(src), rows, cols, dp, bits, tgt, dst);
}

void to_planes(int dtype, const void* src, int64_t rows, int64_t cols, int64_t dp, const unsigned* bits, const int* tgt,
               void* dst, cudaStream_t s) {
    if (dtype == SL_F32) to_planes<float>(src, rows, cols, dp, bits, tgt, dst, s);
    else if (dtype == SL_BF16) to_planes<__nv_bfloat16>(src, rows, cols, dp, bits, tgt, dst, s);
    else to_planes<__half>(src, rows, cols, dp, bits, tgt, dst, s);
}

// 16-bit weights are read where they lie when their rows start on 16 bytes.
bool copies_w(const sl_xent_args& a) { return a.dtype == SL_F32 || a.dim % 8 != 0 || off_by(a.weight, 16); }

int check(const sl_xent_args* a, const char* fn) {
    SL_REQUIRE(a != nullptr, fn, "NULL arguments");
    SL_REQUIRE(known_dtype(a->dtype), fn, "unknown dtype");
    SL_REQUIRE(a->tokens >= 0 && a->dim >= 1 && a->vocab >= 1, fn, "negative or empty shape");
    SL_REQUIRE(a->tokens <= INT_MAX / 2 && a->dim <= (1 << 20) && a->vocab <= INT_MAX / 2, fn, "shape beyond 2^30 rows or 2^20 columns");
    SL_REQUIRE(a->reduction >= SL_XENT_MEAN && a->reduction <= SL_XENT_NONE, fn, "unknown reduction");
    if (a->tokens == 0) return SL_OK;
    SL_REQUIRE(a->x && a->weight && a->targets && a->prep && a->scratch, fn, "NULL operand");
    SL_REQUIRE(!off_by(a->x, dtype_bytes(a->dtype)) && !off_by(a->weight, dtype_bytes(a->dtype)) && !off_by(a->targets, 8) &&
                   !off_by(a->prep, 256) && !off_by(a->scratch, 256),
               fn, "misaligned operand");
    return SL_OK;
}

struct Setup {
    Layout l;
    Problem p;
    Operand x, w;
    char *prep, *scratch;
};

Setup setup(const sl_xent_args& a) {
    Setup s;
    const bool copy = copies_w(a);
    s.l = layout(a.tokens, a.dim, a.vocab, a.dtype, copy);
    s.prep = static_cast<char*>(a.prep);
    s.scratch = static_cast<char*>(a.scratch);
    s.p = Problem{};
    s.p.head = reinterpret_cast<Header*>(s.prep);
    s.p.tgt = reinterpret_cast<int*>(s.prep + s.l.tgt);
    s.p.row_max = reinterpret_cast<float*>(s.prep + s.l.row_max);
    s.p.row_inv = reinterpret_cast<float*>(s.prep + s.l.row_inv);
    s.p.T = a.tokens; s.p.D = a.dim; s.p.V = a.vocab;
    s.p.f32 = a.dtype == SL_F32;
    s.p.bf16 = a.dtype == SL_BF16;
    s.x = {s.prep + s.l.x, a.tokens, a.dim, s.l.dp, a.tokens * s.l.dp};
    s.w = copy ? Operand{s.prep + s.l.w, a.vocab, a.dim, s.l.dp, a.vocab * s.l.dp}
               : Operand{a.weight, a.vocab, a.dim, a.dim, 0};
    return s;
}

int forward(const sl_xent_args& a, cudaStream_t st) {
    Setup s = setup(a);
    const int64_t T = a.tokens, V = a.vocab;
    if (int rc = cuda_status(cudaMemsetAsync(s.prep, 0, 256, st), "sl_xent_forward")) return rc;
    s.p.zt = reinterpret_cast<float*>(s.scratch + s.l.zt);
    s.p.part = reinterpret_cast<float2*>(s.scratch + s.l.part);
    int* tgt = reinterpret_cast<int*>(s.prep + s.l.tgt);
    targets_kernel<<<static_cast<unsigned>((T + kThreads - 1) / kThreads), kThreads, 0, st>>>(a.targets, T, V, a.ignore_index, tgt, s.p.zt, s.p.head);
    if (s.p.f32) {
        absmax_kernel<<<blocks_for(T * a.dim), kThreads, 0, st>>>(static_cast<const float*>(a.x), T, a.dim, a.targets, a.ignore_index, &s.p.head->max_x);
        absmax_kernel<<<blocks_for(V * a.dim), kThreads, 0, st>>>(static_cast<const float*>(a.weight), V, a.dim, nullptr, 0, &s.p.head->max_w);
    }
    to_planes(a.dtype, a.x, T, a.dim, s.l.dp, &s.p.head->max_x, tgt, s.prep + s.l.x, st);
    if (copies_w(a)) to_planes(a.dtype, a.weight, V, a.dim, s.l.dp, &s.p.head->max_w, nullptr, s.prep + s.l.w, st);
    SL_RETURN_IF_LAUNCH_FAILED("sl_xent_forward");
    if (int rc = gemm_stats(s.p, s.x, s.w, st)) return rc;
    const int64_t parts = (V + kPart - 1) / kPart, blocks = (T + 7) / 8;
    double* sums = reinterpret_cast<double*>(s.scratch + s.l.fwd - up(8 * blocks, 256));
    finish_kernel<<<static_cast<unsigned>(blocks), kThreads, 0, st>>>(s.p, parts, a.loss_rows, a.loss, sums, a.reduction == SL_XENT_MEAN);
    SL_RETURN_IF_LAUNCH_FAILED("sl_xent_forward");
    return SL_OK;
}

int backward(const sl_xent_args& a, cudaStream_t st) {
    Setup s = setup(a);
    const int64_t T = a.tokens, V = a.vocab;
    if (a.reduction == SL_XENT_NONE) {
        if (int rc = cuda_status(cudaMemsetAsync(&s.p.head->max_g, 0, 4, st), "sl_xent_backward")) return rc;
        absmax_kernel<<<blocks_for(T), kThreads, 0, st>>>(a.grad, T, 1, a.targets, a.ignore_index, &s.p.head->max_g);
        s.p.g_rows = a.grad;
    }
    grad_scale_kernel<<<1, 1, 0, st>>>(s.p.head, a.reduction == SL_XENT_NONE ? nullptr : a.grad, a.reduction == SL_XENT_MEAN);
    SL_RETURN_IF_LAUNCH_FAILED("sl_xent_backward");
    float* slabs = reinterpret_cast<float*>(s.scratch + s.l.slabs);
    for (int64_t v0 = 0; v0 < V; v0 += s.l.piece) {
        const int64_t cols = std::min(s.l.piece, V - v0);
        const Operand g{s.scratch + s.l.g, T, cols, s.l.gp, T * s.l.gp};
        if (int rc = gemm_grad(s.p, s.x, s.w, v0, cols, g, st)) return rc;
        if (a.dx) {
            const Output o{a.dx, a.dtype, V > s.l.piece ? reinterpret_cast<float*>(s.scratch + s.l.acc) : nullptr, v0 == 0,
                           v0 + cols == V, slabs, s.l.slab_floats, false};
            if (int rc = gemm_dx(s.p, g, cols, s.w, v0, o, st)) return rc;
        }
        if (a.dweight) {
            const Output o{static_cast<char*>(a.dweight) + v0 * a.dim * dtype_bytes(a.dtype), a.dtype, nullptr, true, true,
                           slabs, s.l.slab_floats, true};
            if (int rc = gemm_dw(s.p, g, cols, s.x, o, st)) return rc;
        }
    }
    return SL_OK;
}

}  // namespace
}  // namespace xent
}  // namespace slb

using namespace slb;

extern "C" int sl_xent_sizes(const sl_xent_args* a, int64_t* prep, int64_t* forward, int64_t* backward) {
    const char* fn = "sl_xent_sizes";
    SL_REQUIRE(a && prep && forward && backward, fn, "NULL argument");
    SL_REQUIRE(known_dtype(a->dtype) && a->tokens >= 0 && a->dim >= 1 && a->vocab >= 1, fn, "bad shape or type");
    const xent::Layout l = xent::layout(std::max<int64_t>(a->tokens, 1), a->dim, a->vocab, a->dtype, xent::copies_w(*a));
    *prep = l.prep;
    *forward = l.fwd;
    *backward = l.bwd;
    return SL_OK;
}

extern "C" int sl_xent_forward(const sl_xent_args* a, void* stream) {
    if (int rc = xent::check(a, "sl_xent_forward")) return rc;
    if (a->tokens == 0) return SL_OK;
    SL_REQUIRE(a->reduction == SL_XENT_NONE ? a->loss_rows != nullptr : a->loss != nullptr, "sl_xent_forward", "NULL loss");
    return xent::forward(*a, as_stream(stream));
}

extern "C" int sl_xent_backward(const sl_xent_args* a, void* stream) {
    if (int rc = xent::check(a, "sl_xent_backward")) return rc;
    if (a->tokens == 0) return SL_OK;
    SL_REQUIRE(a->grad != nullptr, "sl_xent_backward", "NULL gradient");
    SL_REQUIRE(!off_by(a->dx, dtype_bytes(a->dtype)) && !off_by(a->dweight, dtype_bytes(a->dtype)), "sl_xent_backward", "misaligned output");
    if (!a->dx && !a->dweight) return SL_OK;
    return xent::backward(*a, as_stream(stream));
}
