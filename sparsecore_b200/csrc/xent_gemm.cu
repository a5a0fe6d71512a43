// The matrix products of the linear cross entropy and their epilogues, on
// the tensor cores.
//
// A pair of CTAs (one on each of two SMs) multiplies tiles of 256 x 256 along
// the whole sum, one after another (the grid is as large as the GPU).  In
// each CTA one thread keeps TMA loads of 64-column slices of the operands
// going round a ring of shared-memory stages, one thread of the first CTA
// issues the MMAs, and eight warps take finished sums out of tensor memory,
// which holds two tiles: one is multiplied while the other is read.
//
// 32-bit operands come as two fp16 planes, a stage holding both, and are
// multiplied as lo.hi, hi.lo and hi.hi.  The matrix units cut rather than
// round when they add to a sum, so a sum in tensor memory is at most kChunk
// stages long; the epilogue's warps add the chunks in registers, rounding to
// nearest.
//
// What bounds it: the tensor cores.  Losses of 4096 tokens over 50001 columns
// of 768 in 32 bits take 636 us, 1483 TFLOP/s of fp16 products; of 8192 tokens
// over 128000 columns of 2048 in bf16 2.92 ms, 1471 TFLOP/s (0.90 and 0.89 of
// the 1646 measured for a library product in a burst).  256 x 256 tiles of a
// pair load 128 operand bytes a clock and SM, half of what a 128 x 256 tile
// of one SM would.  Small problems are bound by a tile's own latency: 16384 x
// 768 over 256 columns has 64 tiles for 74 pairs.
#include <algorithm>

#include "umma.cuh"
#include "xent.cuh"

namespace slb {
namespace xent {
namespace {

enum Mode : int { kStats, kGrad, kOut, kLosses };

constexpr int kTile = 256;
constexpr int kSlice = 64;                       // of the sum, in a stage: 128 bytes a row
constexpr int kBox = 128 * kSlice * 2;           // bytes of one operand's plane in a stage
constexpr int kRing = 12;                        // boxes in shared memory: 6 stages, or 3 of two planes
// Stages added up in tensor memory before the epilogue takes the sum out.  Of
// two planes: 2 where the sum is the result (errors of 4e-7 of it; 4 stages:
// 9e-7), 4 where the logits' epilogue is long and has to be covered.  Of one
// plane: 8 for the logits, whose loss is given in 32 bits, and 32 for the
// gradients: a sum of one sign loses 1.5e-3 over 4096 stages there, 1.2e-5 over
// 32, at no cost (8192 x 2048 x 128000 bf16: 14.29 ms uncut, 14.12 with 32
// stages, 14.37 with 16).
template <int PL, int MODE>
constexpr int kChunk = MODE == kOut ? (PL == 2 ? 2 : 32) : PL == 2 ? 4 : 8;
constexpr int kEpilogueWarps = 8;
constexpr int kThreads = 128 + 32 * kEpilogueWarps;  // a warpgroup of loads and MMAs, two of results
// Registers a thread: of 168 x 384 at launch, 40 x 128 stay with the first
// warpgroup and 232 x 256 hold the results (128 sums a thread).
constexpr int kRegsLow = 40, kRegsHigh = 232;
static_assert(kRegsLow * 128 + kRegsHigh * 256 <= 168 * kThreads, "registers of the launch");
constexpr size_t kSmem = kRing * kBox + 1024 + 4096;

struct Args {
    Problem p;
    int64_t M, N, K;
    int tiles_m, tiles_n, splits, per_split;  // per_split: stages
    bool a_mn, b_mn;
    int64_t v0;
    void* g;
    int64_t g_stride, g_plane;
    Output o;
    Losses l;
    int64_t slab_stride;
    unsigned* status;
};

struct Shared {
    uint64_t full[kRing / 2], empty[kRing / 2], tmem_full[2], tmem_empty[2];
    uint32_t tmem;
    // kLosses: what the two threads of a row tell each other, and the CTA's sums
    float most[2][128], sum[2][128], target[2][128];
    double loss[kEpilogueWarps];
    int count[kEpilogueWarps], last;
};
static_assert(sizeof(Shared) <= 4096, "room behind the ring");

// Whether all the epilogue's warps got their sums: they wait for one another.
__device__ __forceinline__ bool epilogue_agrees(bool ok) {
    int all;
    asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n bar.red.and.pred q, 1, %2, p;\n selp.b32 %0, 1, 0, q;\n}\n"
                 : "=r"(all)
                 : "r"(static_cast<int>(ok)), "n"(32 * kEpilogueWarps)
                 : "memory");
    return all;
}

// A barrier of the epilogue's warps alone.
__device__ __forceinline__ void epilogue_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpilogueWarps) : "memory"); }

// Tiles in groups of 8 rows of tiles, down the columns of a group: what runs
// at one time shares few operand rows.
__device__ __forceinline__ void locate(const Args& a, int id, int& m, int& n, int& split) {
    const int per = a.tiles_m * a.tiles_n;
    split = id / per;
    id -= split * per;
    const int group = id / (8 * a.tiles_n), first = group * 8, rows = min(8, a.tiles_m - first);
    id -= group * 8 * a.tiles_n;
    m = first + id % rows;
    n = id / rows;
}

// Off by 2^-22 at most, as much as the logits' own last bits make it.
__device__ __forceinline__ float exp2_fast(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

__device__ __forceinline__ void store32(void* dst, const uint32_t (&v)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

__device__ __forceinline__ void load32(const void* src, uint32_t (&v)[8]) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "l"(src)
                 : "memory");
}

constexpr float kLog2e = 1.4426950408889634f;

// What brings a sum of 32-bit operands' planes back to the logit.  Never 0,
// which would make NaN of the columns behind the last: logits that would need a
// smaller one are below 2^-76 either way, the planes' sums below 2^50.
__device__ __forceinline__ Factor logit_scale(const Problem& p) {
    return power_of_two(max(-126, -plane_exponent(p.head->max_x) - plane_exponent(p.head->max_w)));
}

// Maximum and sum of exponentials of this thread's row t over 128 columns
// from n0; z holds the logits over `u`.
__device__ __forceinline__ void epilogue_stats(const Args& a, float (&z)[128], int64_t t, int64_t n0, float u) {
    const int n = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(128), a.N - n0)));
    if (t >= a.M || n == 0) return;
    const int tg = target_of(a.p, t);
    if (tg >= n0 && tg < n0 + n) {
        const int at = static_cast<int>(tg - n0);
        float q = 0.f;
#pragma unroll
        for (int j = 0; j < 128; ++j) q = j == at ? z[j] : q;
        a.p.zt[t] = q * u;
    }
    float m = -INFINITY, s[4] = {0.f, 0.f, 0.f, 0.f};
    if (n < 128) {
#pragma unroll
        for (int j = 0; j < 128; ++j) z[j] = j < n ? z[j] : -INFINITY;  // exp gives 0
    }
#pragma unroll
    for (int j = 0; j < 128; ++j) m = fmaxf(m, z[j]);
    m *= u;
    const float from = m == -INFINITY ? 0.f : m;  // of logits that are all -inf the sum is 0
#pragma unroll
    for (int j = 0; j < 128; ++j) s[j & 3] += exp2_fast(fmaf(z[j], u, -from) * kLog2e);
    a.p.part[n0 / kPart * a.M + t] = make_float2(m, (s[0] + s[1]) + (s[2] + s[3]));
}

// 128 columns of G (less the `one` of the target column `at`), as planes:
// v = e * c, from e in z.  An MMA has both operands of one type, so G of 16-bit
// operands is rounded to theirs (half a step, 2^-9 or 2^-12 of an element and without
// a sign; the gradients are rounded to the same type in the end).
template <int PL>
__device__ __forceinline__ void store_grad(const Args& a, const float (&z)[128], int64_t t, int64_t n0, float c, int at, float one) {
    const int64_t room = min(static_cast<int64_t>(128), a.g_stride - n0);
    char* dst = static_cast<char*>(a.g) + 2 * (t * a.g_stride + n0);
#pragma unroll
    for (int j = 0; j < 128; j += 16) {
        if (j >= room) break;
        uint32_t hi[8], lo[8];
        float v[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = z[j + k] * c;
        if (at >> 4 == j >> 4) {
#pragma unroll
            for (int k = 0; k < 16; ++k) v[k] -= j + k == at ? one : 0.f;
        }
#pragma unroll
        for (int k = 0; k < 16; k += 2) {
            if (PL == 1 && a.p.bf16) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[k], v[k + 1]);
                hi[k / 2] = reinterpret_cast<const uint32_t&>(h);
            } else {
                const __half2 h = __floats2half2_rn(v[k], v[k + 1]);
                hi[k / 2] = reinterpret_cast<const uint32_t&>(h);
                if (PL == 2) {
                    const float2 f = __half22float2(h);
                    const __half2 l = __floats2half2_rn(v[k] - f.x, v[k + 1] - f.y);
                    lo[k / 2] = reinterpret_cast<const uint32_t&>(l);
                }
            }
        }
        store32(dst + 2 * j, hi);
        if (PL == 2) store32(dst + 2 * (a.g_plane + j), lo);
    }
}

// G = exp(z - m) / s - [target].
template <int PL>
__device__ __forceinline__ void epilogue_grad(const Args& a, float (&z)[128], int64_t t, int64_t n0, float u) {
    if (t >= a.M || n0 >= a.g_stride) return;
    const int tg = target_of(a.p, t);
    float one = a.p.bf16 ? 1.f : kGradScale;
    if (a.p.g_rows) {  // single losses' gradients, over the largest
        const float top = __uint_as_float(a.p.head->max_g), g = a.p.g_rows[t];
        // without a finite one above zero: zeros, and what is not finite, which stays so
        one = top > 0.f ? one * (g / top) : g == 0.f ? 0.f : __int_as_float(0x7fffffff);
    }
    if (tg == kIgnored) one = 0.f;  // its logits are zeros
    const float m = a.p.row_max[t];
    const int64_t from = tg - a.v0 - n0;
    const int at = tg >= 0 && from >= 0 && from < 128 ? static_cast<int>(from) : -1;
#pragma unroll
    for (int j = 0; j < 128; ++j) z[j] = exp2_fast(fmaf(z[j], u, -m) * kLog2e);
    store_grad<PL>(a, z, t, n0, a.p.row_inv[t] * one, at, one);
}

// A row of at most 256 columns, in two threads that exchange their maxima and
// sums: its loss and, where asked for, its G.
template <int PL>
__device__ __forceinline__ void epilogue_losses(const Args& a, Shared& sh, float (&z)[128], int64_t t, int row, int half, float u,
                                                double& loss, int& count) {
    const int n = max(0, min(128, static_cast<int>(a.N) - half * 128));
    const int tg = t < a.M ? target_of(a.p, t) : kIgnored;
    const int at = tg >= half * 128 && tg < half * 128 + 128 ? tg - half * 128 : -1;
    float m = -INFINITY, zt = 0.f, s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 128; ++j) {
        z[j] = j < n ? z[j] * u : -INFINITY;
        m = fmaxf(m, z[j]);
    }
    if (at >= 0) {
#pragma unroll
        for (int j = 0; j < 128; ++j) zt = j == at ? z[j] : zt;
    }
    sh.most[half][row] = m;
    sh.target[half][row] = zt;
    epilogue_sync();
    m = fmaxf(sh.most[0][row], sh.most[1][row]);
#pragma unroll
    for (int j = 0; j < 128; ++j) {
        z[j] = exp2_fast((z[j] - m) * kLog2e);
        s[j & 3] += z[j];
    }
    sh.sum[half][row] = (s[0] + s[1]) + (s[2] + s[3]);
    epilogue_sync();
    const float total = sh.sum[0][row] + sh.sum[1][row], nan = __int_as_float(0x7fffffff);
    if (half == 0 && t < a.M) {
        const float l = tg == kIgnored ? 0.f : tg == kInvalid ? nan : m + logf(total) - (sh.target[0][row] + sh.target[1][row]);
        if (a.l.rows) a.l.rows[t] = l;
        loss += l;
        count += tg != kIgnored;
    }
    epilogue_sync();  // before the next tile's maxima
    if (a.g == nullptr || t >= a.M || half * 128 >= a.g_stride) return;
    const float one = tg == kIgnored ? 0.f : a.p.bf16 ? 1.f : kGradScale;
    store_grad<PL>(a, z, t, half * 128, tg == kInvalid ? nan : one / total, at, one);
}

// The sum of all losses: every CTA's in its place, and the CTA that comes last
// adds them up in their order.
__device__ __forceinline__ void finish_losses(const Args& a, Shared& sh, double loss, int count) {
    const int warp = (threadIdx.x >> 5) - 4, lane = lane_id();
    auto sum = [&]() {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, o);
        count = __reduce_add_sync(0xffffffffu, count);
        if (lane == 0) sh.loss[warp] = loss, sh.count[warp] = count;
        epilogue_sync();
        loss = 0.0, count = 0;
        for (int k = 0; k < kEpilogueWarps; ++k) loss += sh.loss[k], count += sh.count[k];
        epilogue_sync();
    };
    sum();
    if (warp == 0 && lane == 0) {
        a.l.sums[blockIdx.x] = loss;
        a.l.counts[blockIdx.x] = count;
        __threadfence();
        sh.last = atomicAdd(&a.p.head->done, 1u) == gridDim.x - 1;
    }
    epilogue_sync();
    if (!sh.last) return;
    __threadfence();
    loss = 0.0, count = 0;
    for (int k = warp * 32 + lane; k < gridDim.x; k += 32 * kEpilogueWarps) loss += __ldcg(a.l.sums + k), count += __ldcg(a.l.counts + k);
    sum();
    if (warp == 0 && lane == 0) {
        a.p.head->count = count;
        if (a.l.loss) *a.l.loss = static_cast<float>(a.p.mean ? loss / count : loss);
    }
}

// What is multiplied into a finished sum.
__device__ __forceinline__ Factor out_scale(const Problem& p, bool by_x, bool f32) {
    float g = p.g_rows ? __uint_as_float(p.head->max_g) : *p.grad;
    if (p.mean) g = p.head->count ? g / static_cast<float>(p.head->count) : 0.f;
    if (!f32) return {p.bf16 ? g : g * (1.f / kGradScale), 1.f};
    const double s = scalbn(static_cast<double>(g), -15 - plane_exponent(by_x ? p.head->max_x : p.head->max_w));
    if (s != 0.0 && fabs(s) < 0x1p-126) return {static_cast<float>(s * 0x1p100), 0x1p-100f};
    if (fabs(s) >= 0x1p128 && isfinite(g)) return {static_cast<float>(s * 0x1p-100), 0x1p100f};
    return {static_cast<float>(s), 1.f};
}
static_assert(kGradScale == 32768.f, "2^15 in out_scale");

__device__ __forceinline__ void store_out(const Output& o, int64_t i, float v) {
    if (o.dtype == SL_F32) static_cast<float*>(o.dst)[i] = v;
    else if (o.dtype == SL_BF16) static_cast<__nv_bfloat16*>(o.dst)[i] = __float2bfloat16_rn(v);
    else static_cast<__half*>(o.dst)[i] = __float2half_rn(v);
}

__device__ __forceinline__ void epilogue_out(const Args& a, float (&z)[128], int64_t m, int64_t n0, int split, Factor by) {
    if (m >= a.M) return;
    if (a.splits > 1) {
        float* dst = a.o.slabs + split * a.slab_stride + m * (static_cast<int64_t>(a.tiles_n) * kTile) + n0;
#pragma unroll
        for (int j = 0; j < 128; j += 8) {
            uint32_t v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = __float_as_uint(z[j + k]);
            store32(dst + j, v);
        }
        return;
    }
    const int n = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(128), a.N - n0)));
    const int64_t row = m * a.N + n0;
    if (a.o.acc) {
        float* q = a.o.acc + row;
        if (n == 128 && (reinterpret_cast<uintptr_t>(q) & 31) == 0) {
#pragma unroll
            for (int j = 0; j < 128; j += 8) {
                uint32_t v[8];
                if (!a.o.first) {
                    load32(q + j, v);
#pragma unroll
                    for (int k = 0; k < 8; ++k) z[j + k] += __uint_as_float(v[k]);
                }
                if (!a.o.last) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[k] = __float_as_uint(z[j + k]);
                    store32(q + j, v);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 128; ++j)
                if (j < n) {
                    if (!a.o.first) z[j] += q[j];
                    if (!a.o.last) q[j] = z[j];
                }
        }
        if (!a.o.last) return;
    }
    float scale = by.a;
    if (by.b != 1.f) {
#pragma unroll
        for (int j = 0; j < 128; ++j) z[j] = z[j] * by.a * by.b;
        scale = 1.f;
    }
    const int64_t bytes = a.o.dtype == SL_F32 ? 4 : 2;
    char* dst = static_cast<char*>(a.o.dst) + row * bytes;
    if (n == 128 && (reinterpret_cast<uintptr_t>(dst) & 31) == 0) {
#pragma unroll
        for (int j = 0; j < 128; j += 16) {
            uint32_t v[8];
            if (a.o.dtype == SL_F32) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[k] = __float_as_uint(z[j + 8 * h + k] * scale);
                    store32(dst + 4 * (j + 8 * h), v);
                }
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float p = z[j + 2 * k] * scale, q = z[j + 2 * k + 1] * scale;
                    const __nv_bfloat162 b = __floats2bfloat162_rn(p, q);
                    const __half2 h = __floats2half2_rn(p, q);
                    v[k] = a.o.dtype == SL_BF16 ? reinterpret_cast<const uint32_t&>(b) : reinterpret_cast<const uint32_t&>(h);
                }
                store32(dst + 2 * j, v);
            }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 128; ++j)
        if (j < n) store_out(a.o, row + j, z[j] * scale);
}

template <int PL, int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Args a) {
    constexpr int kStages = kRing / (2 * PL);
    constexpr int kStageBytes = 2 * PL * kBox;
    extern __shared__ char raw[];
    char* ring = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
    Shared& sh = *reinterpret_cast<Shared*>(ring + kRing * kBox);
    const int warp = threadIdx.x >> 5, lane = lane_id();
    const uint32_t rank = cluster_rank();
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&sh.full[s], 1);
            mbar_init(&sh.empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&sh.tmem_full[b], 1);
            mbar_init(&sh.tmem_empty[b], 2 * kEpilogueWarps);
        }
        fence_barrier_init();
    }
    if (warp == 1) tmem_alloc_pair(&sh.tmem, 512);
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    let_follow();
    follow();
    if (MODE == kStats && blockIdx.x == 0 && threadIdx.x == 0) a.p.head->done = 0;  // for the finish
    const uint32_t tmem = sh.tmem;
    const int tiles = a.tiles_m * a.tiles_n * a.splits, pairs = gridDim.x / 2, pair = blockIdx.x / 2;
    const int all = static_cast<int>((a.K + kSlice - 1) / kSlice);
    const int chunk = min(all, kChunk<PL, MODE>);

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsLow));
        if (warp == 0 && lane == 0) {  // loads
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            for (int id = pair; id < tiles && ok; id += pairs) {
                int tm, tn, split;
                locate(a, id, tm, tn, split);
                const int row_a = tm * kTile + static_cast<int>(rank) * 128, row_b = tn * kTile + static_cast<int>(rank) * 128;
                const int k1 = min(all, (split + 1) * a.per_split);
                for (int k = split * a.per_split; k < k1; ++k) {
                    if (!mbar_wait(&sh.empty[stage], phase ^ 1, a.status)) { ok = false; break; }
                    if (rank == 0) mbar_expect_tx(&sh.full[stage], 2 * kStageBytes);
                    const uint32_t bar = leader_addr(&sh.full[stage]);
                    char* dst = ring + stage * kStageBytes;
                    const int x = k * kSlice;
#pragma unroll
                    for (int pl = 0; pl < PL; ++pl, dst += 2 * kBox) {
                        if (a.a_mn) {
                            tma_load_3d_pair(dst, &map_a, row_a, x, pl, bar);
                            tma_load_3d_pair(dst + kBox / 2, &map_a, row_a + 64, x, pl, bar);
                        } else {
                            tma_load_3d_pair(dst, &map_a, x, row_a, pl, bar);
                        }
                        if (a.b_mn) {
                            tma_load_3d_pair(dst + kBox, &map_b, row_b, x, pl, bar);
                            tma_load_3d_pair(dst + kBox + kBox / 2, &map_b, row_b + 64, x, pl, bar);
                        } else {
                            tma_load_3d_pair(dst + kBox, &map_b, x, row_b, pl, bar);
                        }
                    }
                    if (++stage == kStages) stage = 0, phase ^= 1;
                }
            }
            // The last stages are free again before the CTA ends: every commit of
            // the other CTA's thread has then arrived here.
            for (int s = 0; s < kStages && ok; ++s) {
                ok = mbar_wait(&sh.empty[stage], phase ^ 1, a.status);
                if (++stage == kStages) stage = 0, phase ^= 1;
            }
            if (!ok)  // given up: let the copies in flight land before the CTA may end
                for (int i = 0; i < 2000; ++i) __nanosleep(1000);
        } else if (warp == 1 && lane == 0 && rank == 0) {  // MMAs of both CTAs
            const uint32_t idesc = umma_idesc(a.p.bf16, a.a_mn, a.b_mn, kTile);
            const uint32_t step_a = (a.a_mn ? 16 * 128 : 32) >> 4, step_b = (a.b_mn ? 16 * 128 : 32) >> 4;
            uint32_t stage = 0, phase = 0, done = 0;
            bool ok = true;
            for (int id = pair; id < tiles && ok; id += pairs) {
                int tm, tn, split;
                locate(a, id, tm, tn, split);
                const int k1 = min(all, (split + 1) * a.per_split);
                for (int k0 = split * a.per_split; k0 < k1 && ok; k0 += chunk, ++done) {
                    const uint32_t buf = done & 1;
                    if (!mbar_wait_cluster(&sh.tmem_empty[buf], ((done >> 1) & 1) ^ 1, a.status)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t d = tmem + buf * kTile;
                    uint32_t add = 0;
                    const int end = min(k1, k0 + chunk);
                    for (int k = k0; k < end; ++k) {
                        if (!mbar_wait_cluster(&sh.full[stage], phase, a.status)) { ok = false; break; }
                        tc_fence_after();
                        const uint32_t base = smem_addr(ring + stage * kStageBytes);
                        uint64_t da[PL], db[PL];
#pragma unroll
                        for (int pl = 0; pl < PL; ++pl) {
                            da[pl] = umma_desc(base + pl * 2 * kBox, a.a_mn);
                            db[pl] = umma_desc(base + pl * 2 * kBox + kBox, a.b_mn);
                        }
                        // the small products first, while the sum is small
#pragma unroll
                        for (int pr = PL == 2 ? 0 : 2; pr < 3; ++pr) {
                            const uint64_t qa = da[pr == 0 ? PL - 1 : 0], qb = db[pr == 1 ? PL - 1 : 0];
#pragma unroll
                            for (int i = 0; i < kSlice / 16; ++i) {
                                umma_pair(d, qa + i * step_a, qb + i * step_b, idesc, add);
                                add = 1;
                            }
                        }
                        umma_commit_pair(&sh.empty[stage]);
                        if (++stage == kStages) stage = 0, phase ^= 1;
                    }
                    umma_commit_pair(&sh.tmem_full[buf]);
                }
            }
        }
    } else {  // results
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsHigh));
        const int quarter = warp & 3, half = (warp - 4) >> 2;
        const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
        const Factor u = MODE == kOut ? out_scale(a.p, a.o.by_x, PL == 2) : PL == 2 ? logit_scale(a.p) : Factor{1.f, 1.f};
        uint32_t done = 0;
        bool ok = true;
        double loss = 0.0;
        int count = 0;
        for (int id = pair; id < tiles && ok; id += pairs) {
            int tm, tn, split;
            locate(a, id, tm, tn, split);
            const int k1 = min(all, (split + 1) * a.per_split);
            float z[128] = {};
            for (int k0 = split * a.per_split; k0 < k1; k0 += chunk, ++done) {
                const uint32_t buf = done & 1;
                if (!__all_sync(0xffffffffu, mbar_wait(&sh.tmem_full[buf], (done >> 1) & 1, a.status))) { ok = false; break; }
                tc_fence_after();
                const uint32_t at = tmem + lanes + buf * kTile + half * 128;
#pragma unroll
                for (int j = 0; j < 128; j += 32) {
                    uint32_t r[32];
                    tmem_load32(at + j, r);
                    tmem_load_wait();
#pragma unroll
                    for (int k = 0; k < 32; ++k) z[j + k] += __uint_as_float(r[k]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(leader_addr(&sh.tmem_empty[buf]));
            }
            if (MODE == kLosses) ok = epilogue_agrees(ok);
            if (!ok) break;
            const int64_t t = static_cast<int64_t>(tm) * kTile + rank * 128 + quarter * 32 + lane;
            const int64_t n0 = static_cast<int64_t>(tn) * kTile + half * 128;
            if (MODE != kOut && PL == 2 && u.b != 1.f) {
#pragma unroll
                for (int j = 0; j < 128; ++j) z[j] *= u.b;
            }
            if (MODE == kStats) epilogue_stats(a, z, t, n0, u.a);
            else if (MODE == kGrad) epilogue_grad<PL>(a, z, t, n0, u.a);
            else if (MODE == kLosses) epilogue_losses<PL>(a, sh, z, t, quarter * 32 + lane, half, u.a, loss, count);
            else epilogue_out(a, z, t, n0, split, u);
        }
        if (MODE == kLosses && ok) finish_losses(a, sh, loss, count);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // no CTA leaves while the other may still signal it
    tc_fence_after();
    if (warp == 1) tmem_free_pair(tmem, 512);
}

// Sum of a split product's slabs, in their order; W columns a thread.
template <int W>
__global__ void __launch_bounds__(256)
join_kernel(Problem p, Output o, int64_t M, int64_t N, int64_t stride, int64_t slab, int splits, bool f32) {
    let_follow();
    follow();
    const Factor scale = out_scale(p, o.by_x, f32);
    const int64_t step = static_cast<int64_t>(gridDim.x) * 256 * W;
    const int across = static_cast<int>(N);
    for (int64_t i = (blockIdx.x * static_cast<int64_t>(256) + threadIdx.x) * W; i < M * N; i += step) {
        const int64_t m = i / across;
        const float* q = o.slabs + m * stride + (i - m * across);
        float v[W] = {}, f[W];
        for (int s0 = 0; s0 < splits; s0 += 8) {  // eight loads under way
            float g[8][W];
#pragma unroll
            for (int s = 0; s < 8; ++s)
                if (s0 + s < splits) load_f<float, W>(q + (s0 + s) * slab, g[s]);
#pragma unroll
            for (int s = 0; s < 8; ++s)
                if (s0 + s < splits) {
#pragma unroll
                    for (int k = 0; k < W; ++k) v[k] += g[s][k];
                }
        }
        if (o.acc) {
            if (!o.first) {
                load_f<float, W>(o.acc + i, f);
#pragma unroll
                for (int k = 0; k < W; ++k) v[k] += f[k];
            }
            if (!o.last) store_f<float, W>(o.acc + i, v);
        }
        if (o.last) {
#pragma unroll
            for (int k = 0; k < W; ++k) store_out(o, i + k, v[k] * scale.a * scale.b);
        }
    }
}

template <int PL, int MODE>
int launch(const Operand& A, const Operand& B, const Args& a, cudaStream_t s) {
    // The first runtime call of this thread, maybe (a backward pass has its
    // own): it makes the context current that the encoder needs.
    if (int rc = cuda_status(cudaFuncSetAttribute(gemm_kernel<PL, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                  static_cast<int>(kSmem)), "sl_xent"))
        return rc;
    CUtensorMap ma, mb;
    auto map = [&](CUtensorMap* m, const Operand& o, bool mn) {
        return make_tmap_16bit(m, o.base, a.p.bf16, o.cols, o.rows, PL, o.stride, PL == 2 ? o.plane : o.stride * o.rows, mn ? 64 : 128);
    };
    if (!map(&ma, A, a.a_mn) || !map(&mb, B, a.b_mn)) return fail(SL_ERR_CUDA, "sl_xent: tensor map could not be made");
    const int64_t tiles = static_cast<int64_t>(a.tiles_m) * a.tiles_n * a.splits;
    const int64_t pairs = std::min<int64_t>(tiles, std::min(kMostCtas / 2, std::max(1, num_sms() / 2)));
    launch_following(gemm_kernel<PL, MODE>, static_cast<unsigned>(2 * pairs), kThreads, kSmem, s, ma, mb, a);
    SL_RETURN_IF_LAUNCH_FAILED("sl_xent");
    return SL_OK;
}

template <int MODE>
int run(Args& a, const Operand& A, const Operand& B, cudaStream_t s) {
    a.status = device_status_word();
    if (a.status == nullptr) return fail(SL_ERR_CUDA, "sl_xent: no device status word");
    a.tiles_m = static_cast<int>((a.M + kTile - 1) / kTile);
    a.tiles_n = static_cast<int>((a.N + kTile - 1) / kTile);
    const int64_t tiles = static_cast<int64_t>(a.tiles_m) * a.tiles_n;
    SL_REQUIRE(tiles * 2 <= INT_MAX, "sl_xent", "too many tiles");
    const int all = static_cast<int>((a.K + kSlice - 1) / kSlice);
    a.splits = 1;
    a.per_split = all;
    if (MODE == kOut) {
        const SplitSum sp = split_sum(a.M, a.N, a.K, a.p.f32);
        a.splits = sp.splits;
        a.per_split = sp.per_split;
        a.slab_stride = a.M * a.tiles_n * kTile;
    }
    if (int rc = a.p.f32 ? launch<2, MODE>(A, B, a, s) : launch<1, MODE>(A, B, a, s)) return rc;
    if (a.splits > 1) {
        const int64_t stride = static_cast<int64_t>(a.tiles_n) * kTile;
        // four columns a thread where that still fills the GPU
        const int w = a.N % 4 == 0 && a.M * a.N >= num_sms() * 2048 ? 4 : 1;
        const unsigned blocks = static_cast<unsigned>(std::min<int64_t>((a.M * a.N / w + 255) / 256, num_sms() * 16));
        launch_following(w == 4 ? join_kernel<4> : join_kernel<1>, blocks, 256, 0, s, a.p, a.o, a.M, a.N, stride, a.slab_stride,
                         a.splits, a.p.f32);
        SL_RETURN_IF_LAUNCH_FAILED("sl_xent");
    }
    return SL_OK;
}

Operand rows_from(Operand o, int64_t from, int64_t n) {
    o.base = static_cast<const char*>(o.base) + 2 * from * o.stride;
    o.rows = n;
    return o;
}

}  // namespace

// The tiles go over the 74 pairs of SMs in waves; splitting the sum fills the
// last wave (and the first, where there are few tiles) for the price of
// writing, reading and joining the parts.  In clocks: a slice of 64 takes
// 512 (1536 for three products), a tile's end about 3000, a join's launch
// 5000 and memory 3000 bytes a clock.  4096 x 768 from 12544 columns in 32
// bits (48 tiles): 3 parts, 250 -> 190 us.
SplitSum split_sum(int64_t M, int64_t N, int64_t K, bool two_planes) {
    constexpr int64_t kPairs = 74;
    const int64_t tiles_n = (N + kTile - 1) / kTile, tiles = (M + kTile - 1) / kTile * tiles_n, all = (K + kSlice - 1) / kSlice;
    const int64_t slice = two_planes ? 1536 : 512, slab = M * tiles_n * kTile;
    SplitSum best{1, static_cast<int>(all), 0};
    int64_t least = INT64_MAX;
    for (int64_t s = 1; s <= 64 && 4 * (s - 1) < all && (s == 1 || s * slab <= kMostSlabFloats); ++s) {
        const int64_t per = (all + s - 1) / s, parts = (all + per - 1) / per;
        const int64_t cost = (tiles * parts + kPairs - 1) / kPairs * (per * slice + 3000) +
                             (parts > 1 ? 5000 + M * N * 4 * (parts + 1) / 3000 : 0);
        if (cost < least) {
            least = cost;
            best = {static_cast<int>(parts), static_cast<int>(per), parts > 1 ? parts * slab : 0};
        }
    }
    return best;
}

int gemm_stats(const Problem& p, const Operand& x, const Operand& w, cudaStream_t s) {
    Args a{};
    a.p = p; a.M = p.T; a.N = p.V; a.K = p.D;
    return run<kStats>(a, x, w, s);
}

int gemm_losses(const Problem& p, const Operand& x, const Operand& w, const Operand& g, const Losses& l, cudaStream_t s) {
    Args a{};
    a.p = p; a.M = p.T; a.N = p.V; a.K = p.D; a.l = l;
    a.g = const_cast<void*>(g.base); a.g_stride = g.stride; a.g_plane = g.plane;
    return run<kLosses>(a, x, w, s);
}

int gemm_grad(const Problem& p, const Operand& x, const Operand& w, int64_t v0, int64_t cols, const Operand& g, cudaStream_t s) {
    Args a{};
    a.p = p; a.M = p.T; a.N = cols; a.K = p.D;
    a.v0 = v0; a.g = const_cast<void*>(g.base); a.g_stride = g.stride; a.g_plane = g.plane;
    return run<kGrad>(a, x, rows_from(w, v0, cols), s);
}

int gemm_dx(const Problem& p, const Operand& g, int64_t cols, const Operand& w, int64_t v0, const Output& o, cudaStream_t s) {
    Args a{};
    a.p = p; a.M = p.T; a.N = p.D; a.K = cols; a.b_mn = true; a.o = o;
    return run<kOut>(a, g, rows_from(w, v0, cols), s);
}

int gemm_dw(const Problem& p, const Operand& g, int64_t cols, const Operand& x, const Output& o, cudaStream_t s) {
    Args a{};
    a.p = p; a.M = cols; a.N = p.D; a.K = p.T; a.a_mn = a.b_mn = true; a.o = o;
    return run<kOut>(a, g, x, s);
}

}  // namespace xent
}  // namespace slb
