// One AdamW step over a list of tensors in one launch, with the moments in
// 32 or in 8 bits.
//
//   m <- m + (1 - b1) (g - m)        v <- b2 v + (1 - b2) g^2
//   p <- p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// 8-bit moments: the 256 elements of a block share one fp32 scale, and an
// element is an e4m3 value times it.  The second moment is held as its
// square root, which halves the range its exponent has to cover.  An EMA
// moves an element by 0.1 % of its value in a step, far below the spacing of
// 3-bit mantissas, so rounding to nearest would freeze it; the values are
// rounded up or down by 16 dither bits instead (a hash of the element's
// number, the tensor's number, the step and the caller's seed), which keeps
// every moment right on average.  A root above zero is never held as zero:
// its element's next update would be divided by eps alone.
#include <cuda_fp8.h>

#include <cmath>

#include "typed.cuh"

namespace slb {
namespace {

constexpr int kThreads = 256;
constexpr int kPer = 8;                      // elements a thread takes at once
constexpr int kTile = kThreads * kPer;       // 2048: eight 8-bit blocks, one a warp
constexpr int kBlock = SL_ADAMW_BLOCK;       // elements of a scale
static_assert(kBlock == 32 * kPer, "a warp owns one block of the 8-bit moments");

struct Item {
    void* p;
    const void* g;
    void* m;
    void* v;
    float* sm;
    float* su;
    const int32_t* live;
    int64_t n;
    int64_t first;  // number of its first tile
    uint32_t number;
};

// The table travels in the launch's parameters: no copy to the device, and a
// captured launch keeps its own.
template <int MAX>
struct Table {
    Item item[MAX];
    int count;
    int64_t tiles;
};

struct Hyper {
    float decay, step_size, inv_root, one_b1, b2, one_b2, eps;
    uint32_t key;  // seed + step * constant
};

__host__ __device__ __forceinline__ uint32_t mix32(uint32_t v) {
    v = (v ^ (v >> 16)) * 0x5B2C9E6Du;
    v = (v ^ (v >> 13)) * 0x3F4A7C15u;
    return v ^ (v >> 16);
}

// kPer elements from `i`; whole packs where `vec`, else up to `left` of them.
template <typename T>
__device__ __forceinline__ void load(const T* src, int64_t i, int left, bool vec, T (&out)[kPer]) {
    if (vec) {
        const Pack<T, kPer> q = *reinterpret_cast<const Pack<T, kPer>*>(src + i);
#pragma unroll
        for (int k = 0; k < kPer; ++k) out[k] = q.v[k];
    } else {
#pragma unroll
        for (int k = 0; k < kPer; ++k) out[k] = k < left ? src[i + k] : T{};
    }
}
template <typename T>
__device__ __forceinline__ void store(T* dst, int64_t i, int left, bool vec, const T (&in)[kPer]) {
    if (vec) {
        Pack<T, kPer> q;
#pragma unroll
        for (int k = 0; k < kPer; ++k) q.v[k] = in[k];
        *reinterpret_cast<Pack<T, kPer>*>(dst + i) = q;
    } else {
#pragma unroll
        for (int k = 0; k < kPer; ++k)
            if (k < left) dst[i + k] = in[k];
    }
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

__device__ __forceinline__ float e4m3_to_f(uint8_t c) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}

// |a| (already times 448 / top) to e4m3 by 16 dither bits.  Adding the bits
// below the three kept mantissa bits and cutting there rounds up with the
// probability of the part cut off; values below the smallest normal 2^-6
// are moved up into the binade above it, whose spacing 2^-9 is theirs.
__device__ __forceinline__ uint32_t to_e4m3(float a, uint32_t bits16) {
    a = fminf(a, 448.f);
    const bool small = a < 0.015625f;
    const uint32_t raw = __float_as_uint(small ? a + 0.015625f : a) + (bits16 << 4);
    return (raw >> 20) - (120u << 3) - (small ? 8u : 0u);
}

template <typename T, bool EIGHT, int MAX>
__global__ void __launch_bounds__(kThreads)
adamw_multi_kernel(const __grid_constant__ Table<MAX> t, Hyper h, const Hyper* dev) {
    if (dev) h = *dev;
    const int lane = lane_id(), warp = threadIdx.x >> 5;
    for (int64_t tile = blockIdx.x; tile < t.tiles; tile += gridDim.x) {
        int lo = 0, hi = t.count;
        while (hi - lo > 1) {  // last tensor whose first tile is not behind
            const int mid = (lo + hi) >> 1;
            if (t.item[mid].first <= tile) lo = mid; else hi = mid;
        }
        const Item& d = t.item[lo];
        const int64_t i = (tile - d.first) * kTile + threadIdx.x * kPer;
        const int64_t rest = d.n - i;
        const int left = rest >= kPer ? kPer : rest > 0 ? static_cast<int>(rest) : 0;
        if (!EIGHT && left == 0) continue;
        T* P = static_cast<T*>(d.p);
        const T* G = static_cast<const T*>(d.g);
        const bool whole = left == kPer;
        const bool pv = whole && aligned16(P), gv = whole && aligned16(G);
        T p[kPer], g[kPer];
        float m[kPer], u[kPer];  // u: the second moment
        bool on[kPer];
        load(P, i, left, pv, p);
        load(G, i, left, gv, g);
        if (d.live) {
            int32_t c[kPer];
            if (whole && aligned16(d.live)) {
                const int4 a = reinterpret_cast<const int4*>(d.live + i)[0], b = reinterpret_cast<const int4*>(d.live + i)[1];
                c[0] = a.x; c[1] = a.y; c[2] = a.z; c[3] = a.w; c[4] = b.x; c[5] = b.y; c[6] = b.z; c[7] = b.w;
            } else {
#pragma unroll
                for (int k = 0; k < kPer; ++k) c[k] = k < left ? d.live[i + k] : -1;
            }
#pragma unroll
            for (int k = 0; k < kPer; ++k) on[k] = c[k] >= 0;
        } else {
#pragma unroll
            for (int k = 0; k < kPer; ++k) on[k] = k < left;
        }
        const int64_t block = (tile - d.first) * (kTile / kBlock) + warp;
        const bool block_on = block * kBlock < d.n;  // the same in all lanes of the warp
        bool mv = whole, uv = whole;
        if (EIGHT) {
            if (!block_on) continue;
            const uint8_t* M = static_cast<const uint8_t*>(d.m);
            const uint8_t* U = static_cast<const uint8_t*>(d.v);
            mv = whole && (reinterpret_cast<uintptr_t>(M) & 7) == 0;
            uv = whole && (reinterpret_cast<uintptr_t>(U) & 7) == 0;
            uint8_t cm[kPer], cu[kPer];
            load(M, i, left, mv, cm);
            load(U, i, left, uv, cu);
            const float sm = d.sm[block], su = d.su[block];
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                m[k] = e4m3_to_f(cm[k]) * sm;
                const float r = e4m3_to_f(cu[k]) * su;
                u[k] = r * r;
            }
        } else {
            const float* M = static_cast<const float*>(d.m);
            const float* U = static_cast<const float*>(d.v);
            mv = whole && aligned16(M);
            uv = whole && aligned16(U);
            load(M, i, left, mv, m);
            load(U, i, left, uv, u);
        }
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const float gf = to_f(g[k]);
            const float m1 = fmaf(gf - m[k], h.one_b1, m[k]);
            const float v1 = fmaf(u[k], h.b2, gf * gf * h.one_b2);
            const float root = sqrtf(v1);
            if (on[k]) {
                p[k] = from_f<T>(fmaf(-h.step_size, m1 / fmaf(root, h.inv_root, h.eps), to_f(p[k]) * h.decay));
                m[k] = m1;
                u[k] = EIGHT ? root : v1;
            } else if (EIGHT) {
                u[k] = sqrtf(u[k]);
            }
        }
        store(P, i, left, pv, p);
        if (!EIGHT) {
            store(static_cast<float*>(d.m), i, left, mv, m);
            store(static_cast<float*>(d.v), i, left, uv, u);
            continue;
        }
        // The largest finite values of the block set the new scales; one that
        // is not finite stays a NaN of its own and spoils no other element.
        float tm = 0.f, tu = 0.f;
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            if (k >= left) m[k] = u[k] = 0.f;
            if (fabsf(m[k]) <= 3.4028234e38f) tm = fmaxf(tm, fabsf(m[k]));
            if (u[k] <= 3.4028234e38f) tu = fmaxf(tu, u[k]);
        }
        tm = fmaxf(warp_max(tm), 0x1p-100f);
        tu = fmaxf(warp_max(tu), 0x1p-100f);
        const float im = 448.f / tm, iu = 448.f / tu;
        const uint32_t key = mix32(h.key + 0x85EBCA77u * d.number);
        uint8_t cm[kPer], cu[kPer];
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const uint32_t bits = mix32(static_cast<uint32_t>(i + k) * 0x9E3779B1u + key);
            const float am = fabsf(m[k]);
            uint32_t c = to_e4m3(am * im, bits & 0xFFFFu) | (m[k] < 0.f ? 0x80u : 0u);
            cm[k] = static_cast<uint8_t>(am <= 3.4028234e38f ? c : 0x7Fu);
            c = to_e4m3(u[k] * iu, bits >> 16);
            if (c == 0 && u[k] > 0.f) c = 1;
            cu[k] = static_cast<uint8_t>(u[k] <= 3.4028234e38f ? c : 0x7Fu);
        }
        store(static_cast<uint8_t*>(d.m), i, left, mv, cm);
        store(static_cast<uint8_t*>(d.v), i, left, uv, cu);
        if (lane == 0) {
            d.sm[block] = tm * (1.f / 448.f);
            d.su[block] = tu * (1.f / 448.f);
        }
    }
}

Hyper make_hyper(double lr, double b1, double b2, double eps, double wd, int64_t step, uint32_t seed) {
    Hyper h;
    h.decay = static_cast<float>(1.0 - lr * wd);
    h.step_size = static_cast<float>(lr / (1.0 - std::pow(b1, static_cast<double>(step))));
    h.inv_root = static_cast<float>(1.0 / std::sqrt(1.0 - std::pow(b2, static_cast<double>(step))));
    h.one_b1 = static_cast<float>(1.0 - b1);
    h.b2 = static_cast<float>(b2);
    h.one_b2 = static_cast<float>(1.0 - b2);
    h.eps = static_cast<float>(eps);
    h.key = seed + 0x9E3779B1u * static_cast<uint32_t>(step);
    return h;
}

// The step counter and the learning rate read on the device: what a captured
// step needs, whose host arguments are frozen.
__global__ void adamw_hyper_kernel(int64_t* step, const float* lr_dev, double lr, double b1, double b2, double eps,
                                   double wd, uint32_t seed, Hyper* out) {
    const int64_t s = ++*step;
    if (lr_dev) lr = static_cast<double>(*lr_dev);
    Hyper h;
    h.decay = static_cast<float>(1.0 - lr * wd);
    h.step_size = static_cast<float>(lr / (1.0 - pow(b1, static_cast<double>(s))));
    h.inv_root = static_cast<float>(1.0 / sqrt(1.0 - pow(b2, static_cast<double>(s))));
    h.one_b1 = static_cast<float>(1.0 - b1);
    h.b2 = static_cast<float>(b2);
    h.one_b2 = static_cast<float>(1.0 - b2);
    h.eps = static_cast<float>(eps);
    h.key = seed + 0x9E3779B1u * static_cast<uint32_t>(s);
    *out = h;
}

template <typename T, bool EIGHT, int MAX>
int launch(const sl_adamw_item* items, int64_t count, const Hyper& h, const Hyper* dev, cudaStream_t s) {
    for (int64_t at = 0; at < count;) {
        Table<MAX> t;
        t.count = 0;
        t.tiles = 0;
        for (; at < count && t.count < MAX; ++at) {
            const sl_adamw_item& a = items[at];
            if (a.n == 0) continue;
            t.item[t.count++] = {a.p, a.g, a.m, a.v, a.scale_m, a.scale_v, a.live, a.n, t.tiles, static_cast<uint32_t>(a.number)};
            t.tiles += (a.n + kTile - 1) / kTile;
        }
        if (t.count == 0) continue;
        const int64_t cap = static_cast<int64_t>(num_sms()) * 8;
        const int64_t grid = t.tiles < cap ? t.tiles : cap;
        adamw_multi_kernel<T, EIGHT, MAX><<<static_cast<unsigned>(grid), kThreads, 0, s>>>(t, h, dev);
        SL_RETURN_IF_LAUNCH_FAILED("sl_adamw_multi");
    }
    return SL_OK;
}

template <typename T, bool EIGHT>
int pick(const sl_adamw_item* items, int64_t count, const Hyper& h, const Hyper* dev, cudaStream_t s) {
    return count <= 48 ? launch<T, EIGHT, 48>(items, count, h, dev, s) : launch<T, EIGHT, 384>(items, count, h, dev, s);
}

}  // namespace
}  // namespace slb

using namespace slb;

extern "C" int64_t sl_adamw_hyper_bytes(void) { return sizeof(Hyper); }

extern "C" int sl_adamw_hyper(int64_t* step_dev, const float* lr_dev, double lr, double beta1, double beta2, double eps,
                              double weight_decay, uint32_t seed, void* hyper_dev, void* stream) {
    SL_REQUIRE(step_dev != nullptr && hyper_dev != nullptr, "sl_adamw_hyper", "NULL array");
    SL_REQUIRE(lr >= 0.0 && eps >= 0.0 && beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "sl_adamw_hyper",
               "invalid hyper-parameters");
    adamw_hyper_kernel<<<1, 1, 0, as_stream(stream)>>>(step_dev, lr_dev, lr, beta1, beta2, eps, weight_decay, seed,
                                                       static_cast<Hyper*>(hyper_dev));
    SL_RETURN_IF_LAUNCH_FAILED("sl_adamw_hyper");
    return SL_OK;
}

extern "C" int sl_adamw_multi(const sl_adamw_item* items, int64_t count, int dtype, int state_bits, double lr,
                              double beta1, double beta2, double eps, double weight_decay, int64_t step, uint32_t seed,
                              const void* hyper_dev, void* stream) {
    const char* fn = "sl_adamw_multi";
    SL_REQUIRE(count >= 0, fn, "negative count");
    SL_REQUIRE(known_dtype(dtype), fn, "unknown dtype");
    SL_REQUIRE(state_bits == 8 || state_bits == 32, fn, "state_bits must be 8 or 32");
    SL_REQUIRE(hyper_dev != nullptr || step >= 1, fn, "step must be >= 1");
    SL_REQUIRE(hyper_dev != nullptr || (lr >= 0.0 && eps >= 0.0 && beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0),
               fn, "invalid hyper-parameters");
    if (count == 0) return SL_OK;
    SL_REQUIRE(items != nullptr, fn, "NULL items");
    const int64_t esz = dtype_bytes(dtype);
    for (int64_t k = 0; k < count; ++k) {
        const sl_adamw_item& a = items[k];
        SL_REQUIRE(a.n >= 0, fn, "negative length");
        if (a.n == 0) continue;
        SL_REQUIRE(a.p && a.g && a.m && a.v, fn, "NULL tensor");
        SL_REQUIRE(state_bits == 32 || (a.scale_m && a.scale_v), fn, "8-bit moments need their scales");
        SL_REQUIRE(!off_by(a.p, esz) && !off_by(a.g, esz) && !off_by(a.live, 4) && !off_by(a.scale_m, 4) && !off_by(a.scale_v, 4) &&
                       (state_bits == 8 || (!off_by(a.m, 4) && !off_by(a.v, 4))),
                   fn, "misaligned tensor");
    }
    const Hyper* dev = static_cast<const Hyper*>(hyper_dev);
    const Hyper h = dev ? Hyper{} : make_hyper(lr, beta1, beta2, eps, weight_decay, step, seed);
    cudaStream_t s = as_stream(stream);
    if (state_bits == 32) {
        if (dtype == SL_F32) return pick<float, false>(items, count, h, dev, s);
        if (dtype == SL_BF16) return pick<__nv_bfloat16, false>(items, count, h, dev, s);
        return pick<__half, false>(items, count, h, dev, s);
    }
    if (dtype == SL_F32) return pick<float, true>(items, count, h, dev, s);
    if (dtype == SL_BF16) return pick<__nv_bfloat16, true>(items, count, h, dev, s);
    return pick<__half, true>(items, count, h, dev, s);
}
