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
// logits made again, turned into G in the epilogue, and multiplied twice:
// 8 T D V operations in all, where keeping the logits would leave 6.
//
// 16-bit inputs are multiplied as they are.  32-bit ones are split into two
// fp16 planes, a = 2^-k (a_hi + a_lo) with 22 bits between them (2^-k from
// the operand's largest value), and three products hi.hi, hi.lo, lo.hi are
// summed in 32 bits: the result is as exact as a 32-bit product's where the
// operands' rows are of one order of size, on the 16-bit matrix units.
#include <algorithm>

#include "xent.cuh"

namespace slb {
namespace xent {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxBlocks = 1024;  // of an operand's pass

struct Layout {
    int64_t dp;                              // columns of a plane's row
    int64_t row_max, row_inv, x, w, prep;    // offsets in `prep`, and its size
    int64_t zt, part, sums, counts, maxima, fwd;  // in the forward call's scratch
    int64_t piece, gp;                       // vocabulary columns of a piece, of a G row
    int64_t g, acc, slabs, bwd;              // in the backward call's
};

int64_t up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

Layout layout(int64_t T, int64_t D, int64_t V, int dtype, bool copy_x, bool copy_w, bool keep_g) {
    Layout l{};
    const int64_t planes = dtype == SL_F32 ? 2 : 1;
    l.dp = up(D, 64);
    int64_t o = 256;
    auto take = [&](int64_t bytes) { const int64_t at = o; o += up(bytes, 256); return at; };
    l.row_max = take(4 * T);
    l.row_inv = take(4 * T);
    l.x = take(copy_x ? planes * T * l.dp * 2 : 0);
    l.w = take(copy_w ? planes * V * l.dp * 2 : 0);
    if (keep_g) l.g = take(planes * T * up(V, 64) * 2);
    l.prep = o;
    o = 0;
    l.zt = take(4 * T);
    l.part = take((V + kPart - 1) / kPart * T * 8);
    l.sums = take(8 * std::max<int64_t>((T + 31) / 32, kMostCtas));
    l.counts = take(4 * std::max<int64_t>((T + 31) / 32, kMostCtas));
    l.maxima = take(4 * kMaxBlocks * 2);
    l.fwd = o;
    o = 0;
    // A piece's G: 512 MB at most, a multiple of the tile's 256 columns.  Fewer
    // pieces mean fewer sums of dx joined in memory and fewer ends of launches:
    // 8192 x 2048 x 128000 bf16 takes 19.2, 16.2, 14.5 and 14.8 ms with pieces
    // of 96, 256, 512 and 1024 MB.
    const int64_t most = std::max<int64_t>(256, ((int64_t(512) << 20) / (T * planes * 2)) / 256 * 256);
    const int64_t pieces = std::max<int64_t>(1, (V + most - 1) / most);
    l.piece = up((V + pieces - 1) / pieces, 256);
    l.gp = up(std::min(l.piece, V), 64);
    if (!keep_g) l.g = take(planes * T * l.gp * 2);
    l.acc = take(V > l.piece ? 4 * T * D : 0);
    const bool two = dtype == SL_F32;
    const int64_t rest = V - (V - 1) / l.piece * l.piece;  // of the last piece
    int64_t floats = 0;
    for (const int64_t cols : {std::min(l.piece, V), rest})
        floats = std::max({floats, split_sum(T, D, cols, two).floats, split_sum(cols, D, T, two).floats});
    l.slabs = take(4 * floats);
    l.bwd = std::max<int64_t>(o, 256);
    return l;
}

// ── operands ──

// Sizes of the two operands' passes: rows of x, then rows of w.
struct Source {
    const void *x, *w;
    const int64_t* targets;
    int64_t T, V, D, ignore;
};

__device__ __forceinline__ unsigned block_max(unsigned v, unsigned* s) {
    v = __reduce_max_sync(0xffffffffu, v);
    if (lane_id() == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane_id() < kThreads / 32 ? s[lane_id()] : 0u;
    __syncthreads();
    return __reduce_max_sync(0xffffffffu, v);
}

__device__ __forceinline__ unsigned finite_bits(float v) {
    const unsigned b = __float_as_uint(v) & 0x7FFFFFFFu;
    return b < 0x7F800000u ? b : 0u;
}

// Largest finite magnitudes of 32-bit operands, a warp a row: CTAs below
// `x_blocks` take x (rows of tokens that do not count are left out), the
// others w; one value a CTA, joined by planes_kernel.  16384 x 768 and 256 x
// 768: 13 us of 8 for 51 MB (the pass after it finds x in L2: 20 us).
__global__ void __launch_bounds__(kThreads)
absmax_kernel(Source q, int x_blocks, unsigned* part, int vec) {
    __shared__ unsigned s[kThreads / 32];
    let_follow();
    follow();
    const bool is_w = blockIdx.x >= x_blocks;
    const int64_t rows = is_w ? q.V : q.T, first = is_w ? blockIdx.x - x_blocks : blockIdx.x;
    const int64_t step = (is_w ? gridDim.x - x_blocks : x_blocks) * static_cast<int64_t>(kThreads / 32);
    const float* src = static_cast<const float*>(is_w ? q.w : q.x);
    unsigned m = 0;
    for (int64_t r = first * (kThreads / 32) + (threadIdx.x >> 5); r < rows; r += step) {
        if (!is_w && q.targets[r] == q.ignore) continue;
        const float* row = src + r * q.D;
        if (vec) {
#pragma unroll 4
            for (int64_t c = lane_id() * 4; c < q.D; c += 128) {
                const float4 v = *reinterpret_cast<const float4*>(row + c);
                m = max(max(m, max(finite_bits(v.x), finite_bits(v.y))), max(finite_bits(v.z), finite_bits(v.w)));
            }
        } else {
            for (int64_t c = lane_id(); c < q.D; c += 32) m = max(m, finite_bits(row[c]));
        }
    }
    m = block_max(m, s);
    if (threadIdx.x == 0) part[blockIdx.x] = m;
}

// Rows of the operands as planes, padded with zeros to `dp` columns, a warp a
// row; rows of tokens that do not count become zeros, whatever they hold.
template <typename T>
__global__ void __launch_bounds__(kThreads)
planes_kernel(Source q, int64_t dp, const unsigned* part, int x_blocks, int w_blocks, Header* head, void* xp,
              void* wp, int vec) {
    __shared__ unsigned s[kThreads / 32];
    let_follow();
    follow();
    Factor scale_x{1.f, 1.f}, scale_w{1.f, 1.f};
    if (sizeof(T) == 4) {
        unsigned mx = 0, mw = 0;
        for (int k = threadIdx.x; k < x_blocks; k += kThreads) mx = max(mx, part[k]);
        for (int k = threadIdx.x; k < w_blocks; k += kThreads) mw = max(mw, part[x_blocks + k]);
        mx = block_max(mx, s);
        mw = block_max(mw, s);
        scale_x = power_of_two(plane_exponent(mx));
        scale_w = power_of_two(plane_exponent(mw));
        if (blockIdx.x == 0 && threadIdx.x == 0) head->max_x = mx, head->max_w = mw;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) head->done = 0;
    const int64_t rows = q.T + (wp ? q.V : 0), step = static_cast<int64_t>(gridDim.x) * (kThreads / 32);
    for (int64_t r = blockIdx.x * static_cast<int64_t>(kThreads / 32) + (threadIdx.x >> 5); r < rows; r += step) {
        const bool is_w = r >= q.T;
        const int64_t row = is_w ? r - q.T : r;
        const bool on = is_w || q.targets[row] != q.ignore;
        const T* src = static_cast<const T*>(is_w ? q.w : q.x) + row * q.D;
        const Factor scale = is_w ? scale_w : scale_x;
        const int64_t plane = (is_w ? q.V : q.T) * dp;
        uint16_t* dst = static_cast<uint16_t*>(is_w ? wp : xp) + row * dp;
        for (int64_t c = lane_id() * 8; c < dp; c += 256) {
            float v[8] = {};
            if (on) {
                if (vec && c < q.D) {
                    load_f<T, 8>(src + c, v);
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[k] = c + k < q.D ? to_f(src[c + k]) : 0.f;
                }
            }
            if constexpr (sizeof(T) == 4) {
                float lo[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    v[k] = v[k] * scale.a * scale.b;
                    lo[k] = v[k] - __half2float(__float2half_rn(v[k]));
                }
                store_f<__half, 8>(reinterpret_cast<__half*>(dst) + c, v);
                store_f<__half, 8>(reinterpret_cast<__half*>(dst) + plane + c, lo);
            } else {
                store_f<T, 8>(reinterpret_cast<T*>(dst) + c, v);
            }
        }
    }
}

// Largest finite magnitude of the single losses' gradients.
__global__ void __launch_bounds__(1024)
grad_max_kernel(Problem p) {
    __shared__ unsigned s[32];
    let_follow();
    follow();
    unsigned m = 0;
    for (int64_t t = threadIdx.x; t < p.T; t += 1024)
        if (p.targets[t] != p.ignore) m = max(m, finite_bits(p.g_rows[t]));
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane_id() == 0) s[threadIdx.x >> 5] = m;
    __syncthreads();
    if (threadIdx.x < 32) {
        m = __reduce_max_sync(0xffffffffu, s[threadIdx.x]);
        if (threadIdx.x == 0) p.head->max_g = m;
    }
}

// ── joining the partial sums ──

// (max, sum of exponentials below it) of two sets of logits.  An empty set is
// (-inf, 0); equal infinities give a NaN, as they do in the definition.
__device__ __forceinline__ float2 join(float2 a, float2 b) {
    const float m = fmaxf(a.x, b.x);
    return make_float2(m, (a.y == 0.f ? 0.f : a.y * expf(a.x - m)) + (b.y == 0.f ? 0.f : b.y * expf(b.x - m)));
}

// 32 rows a CTA, blockDim.y threads a row.
__global__ void __launch_bounds__(1024)
finish_kernel(Problem p, int parts, float* __restrict__ rows, float* loss, double* sums, int* counts) {
    __shared__ float2 s[32][33];
    __shared__ double total[32];
    __shared__ int found[32];
    __shared__ bool last;
    let_follow();
    follow();
    const int64_t t0 = blockIdx.x * static_cast<int64_t>(32);
    float2 q = make_float2(-INFINITY, 0.f);
    if (t0 + threadIdx.x < p.T) {
#pragma unroll 4
        for (int k = threadIdx.y; k < parts; k += blockDim.y) q = join(q, p.part[k * p.T + t0 + threadIdx.x]);
    }
    s[threadIdx.y][threadIdx.x] = q;
    __syncthreads();
    double a = 0.0;
    int n = 0;
    for (int r = threadIdx.y; r < 32; r += blockDim.y) {  // a warp a row
        const int64_t t = t0 + r;
        if (t >= p.T) break;
        q = threadIdx.x < blockDim.y ? s[threadIdx.x][r] : make_float2(-INFINITY, 0.f);
        for (int o = 1; o < blockDim.y; o <<= 1)
            q = join(q, make_float2(__shfl_xor_sync(0xffffffffu, q.x, o), __shfl_xor_sync(0xffffffffu, q.y, o)));
        const int tg = target_of(p, t);
        const float nan = __int_as_float(0x7fffffff);  // of a target that does not exist
        const float l = tg == kIgnored ? 0.f : tg == kInvalid ? nan : q.x + logf(q.y) - p.zt[t];
        if (threadIdx.x == 0) {
            p.row_max[t] = q.x;
            p.row_inv[t] = tg == kInvalid ? nan : 1.f / q.y;
            if (rows) rows[t] = l;
        }
        a += l;
        n += tg != kIgnored;
    }
    if (threadIdx.x == 0) total[threadIdx.y] = a, found[threadIdx.y] = n;
    __syncthreads();
    if (threadIdx.x == 0 && threadIdx.y == 0) {
        for (int k = 1; k < blockDim.y; ++k) a += total[k], n += found[k];
        sums[blockIdx.x] = a;
        counts[blockIdx.x] = n;
        __threadfence();
        last = atomicAdd(&p.head->done, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    // The CTA that comes last adds all sums in their order, whoever it is.
    const int tid = threadIdx.y * 32 + threadIdx.x, threads = blockDim.y * 32;
    a = 0.0;
    n = 0;
    for (int64_t k = tid; k < gridDim.x; k += threads) a += __ldcg(sums + k), n += __ldcg(counts + k);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    n = __reduce_add_sync(0xffffffffu, n);
    if (threadIdx.x == 0) total[threadIdx.y] = a, found[threadIdx.y] = n;
    __syncthreads();
    if (tid) return;
    a = 0.0, n = 0;
    for (int k = 0; k < blockDim.y; ++k) a += total[k], n += found[k];
    p.head->count = n;
    if (loss) *loss = static_cast<float>(p.mean ? a / n : a);
}

// 16-bit weights are read where they lie when their rows start on 16 bytes.
bool copies_w(const sl_xent_args& a) { return a.dtype == SL_F32 || a.dim % 8 != 0 || off_by(a.weight, 16); }
// x too, where no gradient is asked for: rows that do not count then need
// not be zeros, since a row of logits depends on its own row of x alone.
bool copies_x(const sl_xent_args& a) { return a.train || a.dtype == SL_F32 || a.dim % 8 != 0 || off_by(a.x, 16); }

// A vocabulary of one tile: the forward pass has a row's logits together and
// leaves G (of all tokens: at most 256 columns) for the backward pass, which
// then has no logits to make again.  Single losses' gradients are not known
// in time.  16384 x 768 x 256 fp32: two launches less and 153 -> 134 us.
bool one_tile(const sl_xent_args& a) {
    return a.vocab <= kOneTile && copies_x(a) && !(a.train && a.reduction == SL_XENT_NONE);
}
Layout layout(const sl_xent_args& a) {
    return layout(std::max<int64_t>(a.tokens, 1), a.dim, a.vocab, a.dtype, copies_x(a), copies_w(a), a.train && one_tile(a));
}

int check_shape(const sl_xent_args* a, const char* fn) {
    SL_REQUIRE(a != nullptr, fn, "NULL arguments");
    SL_REQUIRE(known_dtype(a->dtype), fn, "unknown dtype");
    SL_REQUIRE(a->tokens >= 0 && a->dim >= 1 && a->vocab >= 1, fn, "negative or empty shape");
    SL_REQUIRE(a->tokens <= INT_MAX / 2 && a->dim <= (1 << 20) && a->vocab <= INT_MAX / 2, fn, "shape beyond 2^30 rows or 2^20 columns");
    SL_REQUIRE(a->reduction >= SL_XENT_MEAN && a->reduction <= SL_XENT_NONE, fn, "unknown reduction");
    return SL_OK;
}
int check(const sl_xent_args* a, const char* fn) {
    if (int rc = check_shape(a, fn)) return rc;
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
    s.l = layout(a);
    s.prep = static_cast<char*>(a.prep);
    s.scratch = static_cast<char*>(a.scratch);
    s.p = Problem{};
    s.p.head = reinterpret_cast<Header*>(s.prep);
    s.p.targets = a.targets;
    s.p.ignore = a.ignore_index;
    s.p.row_max = reinterpret_cast<float*>(s.prep + s.l.row_max);
    s.p.row_inv = reinterpret_cast<float*>(s.prep + s.l.row_inv);
    s.p.T = a.tokens; s.p.D = a.dim; s.p.V = a.vocab;
    s.p.f32 = a.dtype == SL_F32;
    s.p.bf16 = a.dtype == SL_BF16;
    s.p.mean = a.reduction == SL_XENT_MEAN;
    s.x = copies_x(a) ? Operand{s.prep + s.l.x, a.tokens, a.dim, s.l.dp, a.tokens * s.l.dp}
                      : Operand{a.x, a.tokens, a.dim, a.dim, 0};
    s.w = copy ? Operand{s.prep + s.l.w, a.vocab, a.dim, s.l.dp, a.vocab * s.l.dp}
               : Operand{a.weight, a.vocab, a.dim, a.dim, 0};
    return s;
}

int blocks_for(int64_t rows) {
    const int64_t most = std::min<int64_t>(kMaxBlocks, static_cast<int64_t>(num_sms()) * 6);
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((rows + kThreads / 32 - 1) / (kThreads / 32), most)));
}

int forward(const sl_xent_args& a, cudaStream_t st) {
    Setup s = setup(a);
    const int64_t T = a.tokens, V = a.vocab;
    s.p.zt = reinterpret_cast<float*>(s.scratch + s.l.zt);
    s.p.part = reinterpret_cast<float2*>(s.scratch + s.l.part);
    unsigned* maxima = reinterpret_cast<unsigned*>(s.scratch + s.l.maxima);
    const bool cx = copies_x(a), cw = copies_w(a);
    const Source src{a.x, a.weight, a.targets, cx ? T : 0, V, a.dim, a.ignore_index};
    const int vec = a.dim % 8 == 0 && !off_by(a.x, 16) && !off_by(a.weight, 16);
    const int bx = blocks_for(T), bw = blocks_for(V);
    void *xp = s.prep + s.l.x, *wp = cw ? s.prep + s.l.w : nullptr;
    const int blocks = blocks_for(src.T + (cw ? V : 0));
    if (s.p.f32) {
        launch_following(absmax_kernel, bx + bw, kThreads, 0, st, src, bx, maxima, vec);
        launch_following(planes_kernel<float>, blocks, kThreads, 0, st, src, s.l.dp, maxima, bx, bw, s.p.head, xp, wp, vec);
    } else if (cx || cw) {
        const unsigned* none = nullptr;
        launch_following(s.p.bf16 ? planes_kernel<__nv_bfloat16> : planes_kernel<__half>, blocks, kThreads, 0, st, src, s.l.dp,
                         none, 0, 0, s.p.head, xp, wp, vec);
    }
    SL_RETURN_IF_LAUNCH_FAILED("sl_xent_forward");
    double* sums = reinterpret_cast<double*>(s.scratch + s.l.sums);
    int* counts = reinterpret_cast<int*>(s.scratch + s.l.counts);
    if (one_tile(a)) {
        const Operand g{a.train ? s.prep + s.l.g : nullptr, T, V, s.l.gp, T * s.l.gp};
        return gemm_losses(s.p, s.x, s.w, g, {a.loss, a.loss_rows, sums, counts}, st);
    }
    if (int rc = gemm_stats(s.p, s.x, s.w, st)) return rc;
    const int parts = static_cast<int>((V + kPart - 1) / kPart);
    int groups = 1;
    while (groups < parts && groups < 32) groups *= 2;
    launch_following(finish_kernel, static_cast<unsigned>((T + 31) / 32), dim3(32, groups), 0, st, s.p, parts, a.loss_rows,
                     a.loss, sums, counts);
    SL_RETURN_IF_LAUNCH_FAILED("sl_xent_forward");
    return SL_OK;
}

int backward(const sl_xent_args& a, cudaStream_t st) {
    Setup s = setup(a);
    const int64_t T = a.tokens, V = a.vocab;
    if (a.reduction == SL_XENT_NONE) {
        s.p.g_rows = a.grad;
        launch_following(grad_max_kernel, 1, 1024, 0, st, s.p);
        SL_RETURN_IF_LAUNCH_FAILED("sl_xent_backward");
    } else {
        s.p.grad = a.grad;
    }
    float* slabs = reinterpret_cast<float*>(s.scratch + s.l.slabs);
    const bool one = one_tile(a);  // the forward call left G
    for (int64_t v0 = 0; v0 < V; v0 += s.l.piece) {
        const int64_t cols = std::min(s.l.piece, V - v0);
        const Operand g{(one ? s.prep : s.scratch) + s.l.g, T, cols, s.l.gp, T * s.l.gp};
        if (!one)
            if (int rc = gemm_grad(s.p, s.x, s.w, v0, cols, g, st)) return rc;
        if (a.dx) {
            const Output o{a.dx, a.dtype, V > s.l.piece ? reinterpret_cast<float*>(s.scratch + s.l.acc) : nullptr, v0 == 0,
                           v0 + cols == V, slabs, false};
            if (int rc = gemm_dx(s.p, g, cols, s.w, v0, o, st)) return rc;
        }
        if (a.dweight) {
            const Output o{static_cast<char*>(a.dweight) + v0 * a.dim * dtype_bytes(a.dtype), a.dtype, nullptr, true, true,
                           slabs, true};
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
    SL_REQUIRE(prep && forward && backward, fn, "NULL argument");
    if (int rc = xent::check_shape(a, fn)) return rc;
    const xent::Layout l = xent::layout(*a);
    *prep = l.prep;
    *forward = l.fwd;
    *backward = l.bwd;
    return SL_OK;
}

extern "C" int sl_xent_forward(const sl_xent_args* a, void* stream) {
    g_launched = 0;
    if (int rc = xent::check(a, "sl_xent_forward")) return rc;
    if (a->tokens == 0) return SL_OK;
    SL_REQUIRE(a->reduction == SL_XENT_NONE ? a->loss_rows != nullptr : a->loss != nullptr, "sl_xent_forward", "NULL loss");
    return xent::forward(*a, as_stream(stream));
}

extern "C" int sl_xent_backward(const sl_xent_args* a, void* stream) {
    g_launched = 0;
    if (int rc = xent::check(a, "sl_xent_backward")) return rc;
    if (a->tokens == 0) return SL_OK;
    SL_REQUIRE(a->grad != nullptr && a->train, "sl_xent_backward", "NULL gradient, or a forward call without train");
    SL_REQUIRE(!off_by(a->dx, dtype_bytes(a->dtype)) && !off_by(a->dweight, dtype_bytes(a->dtype)), "sl_xent_backward", "misaligned output");
    if (!a->dx && !a->dweight) return SL_OK;
    return xent::backward(*a, as_stream(stream));
}
