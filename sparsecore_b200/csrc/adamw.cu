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
// its element's next update would be divided by eps alone.  What is not finite
// is held as NaN, an infinite root (of a gradient whose square passes 32 bits)
// as the byte 0xFF: m / root is 0 then, as with 32-bit moments.
//
// 32-bit moments are bound by memory: 12.2 M weights in padded arrays (32
// bytes a slot, padding read too) take 67 us, 5.8 TB/s.  8-bit ones are bound
// by instructions, about 65 an element, half of them integer and logic ones
// for the dither: 335 M bf16 weights take 0.88 ms where their 10 bytes each
// would take 0.52.
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
    bool plain;     // no padding, all addresses on 16 bytes (8-bit moments: on 8)
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
__device__ __forceinline__ void load(const T* src, int64_t i, int left, bool vec, float (&out)[kPer]) {
    if (vec) {
        load_f<T, kPer>(src + i, out);
    } else {
#pragma unroll
        for (int k = 0; k < kPer; ++k) out[k] = k < left ? to_f(src[i + k]) : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void store(T* dst, int64_t i, int left, bool vec, const float (&in)[kPer]) {
    if (vec) {
        store_f<T, kPer>(dst + i, in);
    } else {
#pragma unroll
        for (int k = 0; k < kPer; ++k)
            if (k < left) dst[i + k] = from_f<T>(in[k]);
    }
}

// Square roots to half a step but for rare cases (one Newton step on an
// approximate 1 / root, so that what the 8-bit values are cut from is as exact
// as a 32-bit number can be).  Of infinity NaN; of a subnormal number, which the
// approximation takes for 0, up to 0x1p-62 (see kExactBelow).
__device__ __forceinline__ void roots(float (&v)[kPer]) {
    float y[kPer], r[kPer], e[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y[k]) : "f"(v[k]));
        y[k] = fminf(y[k], 1e19f);  // of 0: no infinity
    }
    vmul(r, v, y);
    vmul(e, r, -1.f);
    vfma(e, e, r, v);
    vmul(y, y, 0.5f);
    vfma(v, e, y, r);
}

// Eight e4m3 values.
__device__ __forceinline__ void from_e4m3(uint2 c, float (&out)[kPer]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t w = (k < 2 ? c.x : c.y) >> (16 * (k & 1));
        const __half2 h(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xFFFFu), __NV_E4M3));
        const float2 f = __half22float2(h);
        out[2 * k] = f.x;
        out[2 * k + 1] = f.y;
    }
}

// a >= 0 (already over its scale, up to 448) rounded up or down to an e4m3
// value by 16 dither bits.  Adding the bits below the three kept mantissa bits
// and cutting there rounds up with the probability of the part cut off; values
// below the smallest normal 2^-6 are moved up into the binade above it, whose
// spacing 2^-9 is theirs, and back.  Whether to is a saturated product, not a
// comparison: the kernel is bound by the integer and logic units.
__device__ __forceinline__ void dithered(float (&a)[kPer], const uint32_t (&bits16)[kPer]) {
    float small[kPer];  // 1 below 2^-6, else 0
#pragma unroll
    for (int k = 0; k < kPer; ++k) small[k] = __saturatef(fmaf(a[k], -0x1p100f, 0x1p94f));
    vfma(a, small, 0x1p-6f, a);
#pragma unroll
    for (int k = 0; k < kPer; ++k) a[k] = __uint_as_float((__float_as_uint(a[k]) + bits16[k] * 16u) & 0xFFF00000u);
    vfma(a, small, -0x1p-6f, a);
}

__device__ __forceinline__ uint2 to_e4m3(const float (&q)[kPer]) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
        w[k] = __nv_cvt_float2_to_fp8x2(make_float2(q[2 * k], q[2 * k + 1]), __NV_SATFINITE, __NV_E4M3);
    return make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
}

// Eight bytes of the 8-bit moments; those from `left` on are not touched.
__device__ __forceinline__ uint2 load8(const uint8_t* src, int left, bool vec) {
    if (vec) return *reinterpret_cast<const uint2*>(src);
    uint32_t w[2] = {0, 0};
    for (int k = 0; k < left; ++k) w[k >> 2] |= static_cast<uint32_t>(src[k]) << (8 * (k & 3));
    return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ void store8(uint8_t* dst, int left, bool vec, uint2 v) {
    if (vec) {
        *reinterpret_cast<uint2*>(dst) = v;
    } else {
        for (int k = 0; k < left; ++k) dst[k] = static_cast<uint8_t>((k < 4 ? v.x : v.y) >> (8 * (k & 3)));
    }
}

// max that keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float rcp_fast(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// Which of a thread's elements take the step: those of a padded array whose
// column is not below 0, and never those behind the tensor's end.
__device__ __forceinline__ uint32_t taking_part(const int32_t* live, int64_t i, int left) {
    uint32_t on = (1u << left) - 1;
    if (live == nullptr) return on;
    if (left == kPer && aligned16(live + i)) {
        const int4 a = reinterpret_cast<const int4*>(live + i)[0], b = reinterpret_cast<const int4*>(live + i)[1];
        const int32_t c[kPer] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int k = 0; k < kPer; ++k) on &= ~((static_cast<uint32_t>(c[k]) >> 31) << k);
    } else {
        for (int k = 0; k < left; ++k) on &= ~((static_cast<uint32_t>(live[i + k]) >> 31) << k);
    }
    return on;
}

// Eight elements of a tensor with 32-bit moments.
template <typename T, bool PLAIN>
__device__ __forceinline__ void step32(const Item& d, const Hyper& h, int64_t i, int left) {
    T* P = static_cast<T*>(d.p);
    const T* G = static_cast<const T*>(d.g);
    float* M = static_cast<float*>(d.m);
    float* V = static_cast<float*>(d.v);
    const bool whole = left == kPer;
    const bool pv = PLAIN || (whole && aligned16(P)), gv = PLAIN || (whole && aligned16(G)),
               mv = PLAIN || (whole && aligned16(M)), vv = PLAIN || (whole && aligned16(V));
    float p[kPer], g[kPer], m[kPer], v[kPer];
    load(P, i, left, pv, p);
    load(G, i, left, gv, g);
    load(M, i, left, mv, m);
    load(V, i, left, vv, v);
    const uint32_t on = PLAIN ? 0xFFu : taking_part(d.live, i, left);
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const float gf = g[k];
        const float m1 = fmaf(gf - m[k], h.one_b1, m[k]);
        const float v1 = fmaf(v[k], h.b2, gf * gf * h.one_b2);
        if (PLAIN || (on >> k & 1)) {
            p[k] = fmaf(-h.step_size, m1 / fmaf(sqrtf(v1), h.inv_root, h.eps), p[k] * h.decay);
            m[k] = m1;
            v[k] = v1;
        }
    }
    store(P, i, left, pv, p);
    store(M, i, left, mv, m);
    store(V, i, left, vv, v);
}

// Blocks with second moments that are subnormal or infinite take a path of
// their own with each root rounded: a call with nothing kept over it, since what
// it needs would be taken from every other block's registers (335 M bf16
// weights: 874 us without it, 881 so, 931 inlined).  A block takes it where it
// has something that is not finite, where its largest root is below 0x1p-44, or
// where eps would not hide a root below 0x1p-62 from the update.  Beside a root of
// 0x1p-44 such a one is held as the smallest 8-bit value, whatever its digits are.
constexpr float kExactBelow = 0x1p-44f, kExactEps = 1e-12f;

// Eight elements of a block with 8-bit moments; a warp has the whole block.
// The kernel is bound by its instructions as much as by its bytes (10 of a
// 16-bit weight), so the quotient is an approximate one (2^-22 of p's update),
// and padding, ends and odd addresses are kept out of the
// ordinary path.
template <typename T, bool PLAIN, bool EXACT = false>
__device__ __forceinline__ bool step8(const Item& d, const Hyper& h, uint32_t key, int64_t i, int64_t block, int left) {
    T* P = static_cast<T*>(d.p);
    const T* G = static_cast<const T*>(d.g);
    uint8_t* M = static_cast<uint8_t*>(d.m) + i;
    uint8_t* U = static_cast<uint8_t*>(d.v) + i;
    const bool whole = left == kPer;
    const bool pv = PLAIN || (whole && aligned16(P)), gv = PLAIN || (whole && aligned16(G)),
               mv = PLAIN || (whole && (reinterpret_cast<uintptr_t>(M) & 7) == 0),
               uv = PLAIN || (whole && (reinterpret_cast<uintptr_t>(U) & 7) == 0);
    float p[kPer], g[kPer], m[kPer], u[kPer];
    load(P, i, left, pv, p);
    load(G, i, left, gv, g);
    const uint2 cm = load8(M, left, mv), cu = load8(U, left, uv);
    const uint32_t on = PLAIN ? 0xFFu : taking_part(d.live, i, left);
    from_e4m3(cm, m);
    from_e4m3(cu, u);
    if constexpr (EXACT) {
#pragma unroll
        for (int k = 0; k < kPer; ++k)
            if (((k < 4 ? cu.x : cu.y) >> (8 * (k & 3)) & 0xFF) == 0xFF) u[k] = INFINITY;
    }
    // Each step is rounded by itself, in the formula's order: the 8-bit values
    // are then those of the formula in 32-bit operations, and not now and then
    // their neighbours.  (The additions one by one: in pairs they would be made
    // one with the products before them.)
    float m1[kPer], root[kPer], q[kPer];
    vmul(m, m, d.sm[block]);
    vfma(m1, m, -1.f, g);
    vmul(m1, m1, h.one_b1);
    vmul(u, u, d.su[block]);
    vmul(root, u, u);
    vmul(root, root, h.b2);
    vmul(g, g, g);
    vmul(g, g, h.one_b2);
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        m1[k] = __fadd_rn(m[k], m1[k]);
        root[k] = __fadd_rn(root[k], g[k]);
    }
    if constexpr (EXACT) {
#pragma unroll
        for (int k = 0; k < kPer; ++k) root[k] = sqrtf(root[k]);
    } else {
        roots(root);
    }
    vfma(q, root, h.inv_root, h.eps);
#pragma unroll
    for (int k = 0; k < kPer; ++k) q[k] = rcp_fast(q[k]);
    vmul(q, q, m1);
    if constexpr (PLAIN) {
        vmul(p, p, h.decay);
        vfma(p, q, -h.step_size, p);
#pragma unroll
        for (int k = 0; k < kPer; ++k) m[k] = m1[k], u[k] = root[k];
    } else {
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            if (on >> k & 1) {
                p[k] = fmaf(-h.step_size, q[k], p[k] * h.decay);
                m[k] = m1[k];
                u[k] = root[k];
            }
        }
    }
    float tm = 0.f, tu = 0.f;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        tm = max_nan(tm, fabsf(m[k]));
        tu = max_nan(tu, u[k]);
    }
    // the largest magnitudes' bits: what is not finite is above all that is
    uint32_t bm = __reduce_max_sync(0xffffffffu, __float_as_uint(tm)), bu = __reduce_max_sync(0xffffffffu, __float_as_uint(tu));
    uint32_t bad = 0;
    if constexpr (EXACT) {  // elements that are not finite are no part of the scales: held as NaN, an infinite root as 0xFF
        bm = bu = 0;
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const uint32_t a = __float_as_uint(m[k]) & 0x7FFFFFFFu, b = __float_as_uint(u[k]) & 0x7FFFFFFFu;
            if (a >= 0x7F800000u) bad |= 1u << k, m[k] = 0.f; else bm = max(bm, a);
            if (b >= 0x7F800000u) bad |= (b == 0x7F800000u ? 0x10000u : 0x100u) << k, u[k] = 0.f; else bu = max(bu, b);
        }
        bm = __reduce_max_sync(0xffffffffu, bm);
        bu = __reduce_max_sync(0xffffffffu, bu);
    } else {
        const uint32_t low = h.eps < kExactEps ? 0x7F800000u : __float_as_uint(kExactBelow);
        if (bm >= 0x7F800000u || bu - low >= 0x7F800000u - low)
            if (bu != 0 || bm >= 0x7F800000u) return false;
    }
    store(P, i, left, pv, p);
    const float fm = fmaxf(__uint_as_float(bm), 0x1p-100f), fu = fmaxf(__uint_as_float(bu), 0x1p-100f);
    const float im = __frcp_rn(fm) * 448.f, iu = __frcp_rn(fu) * 448.f;
    const uint32_t first = static_cast<uint32_t>(i) * 0x9E3779B1u + key;
    uint32_t lo[kPer], hi[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const uint32_t bits = mix32(first + k * 0x9E3779B1u);
        lo[k] = bits & 0xFFFFu;
        hi[k] = bits >> 16;
    }
    float am[kPer], floor[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        am[k] = fabsf(m[k]) * im;
        floor[k] = __saturatef(u[k] * 0x1p126f);  // of what is not zero the smallest e4m3 value
    }
    vmul(u, u, iu);
    vmul(floor, floor, 0x1p-9f);
    dithered(am, lo);
    dithered(u, hi);
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        m[k] = copysignf(am[k], m[k]);
        u[k] = fmaxf(u[k], floor[k]);
    }
    if (EXACT && bad) {
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            if (bad >> k & 1) m[k] = __int_as_float(0x7fffffff);
            if (bad >> (8 + k) & 1) u[k] = __int_as_float(0x7fffffff);
        }
    }
    uint2 held = to_e4m3(u);
    if constexpr (EXACT) {
#pragma unroll
        for (int k = 0; k < kPer; ++k)
            if (bad >> (16 + k) & 1) (k < 4 ? held.x : held.y) |= 0xFFu << (8 * (k & 3));
    }
    store8(M, left, mv, to_e4m3(m));
    store8(U, left, uv, held);
    if (lane_id() == 0) {
        d.sm[block] = fm * (1.f / 448.f);
        d.su[block] = fu * (1.f / 448.f);
    }
    return true;
}

// Key of a tensor's dither.
__device__ __forceinline__ uint32_t dither_key(const Hyper& h, const Item& d) { return mix32(h.key + 0x85EBCA77u * d.number); }

template <typename T>
__device__ __noinline__ void step8_exact(const Item& d, Hyper h, int64_t tile) {
    const int64_t block = (tile - d.first) * (kTile / kBlock) + (threadIdx.x >> 5), i = (tile - d.first) * kTile + threadIdx.x * kPer;
    const int64_t rest = d.n - i;
    step8<T, false, true>(d, h, dither_key(h, d), i, block, rest >= kPer ? kPer : rest > 0 ? static_cast<int>(rest) : 0);
}

template <typename T, bool EIGHT, int MAX>
__global__ void __launch_bounds__(kThreads, 4)
adamw_multi_kernel(const __grid_constant__ Table<MAX> t, const Hyper host, const Hyper* dev) {
    Hyper h = host;
    if (dev) h = *dev;
    int at = 0;
    int64_t end = 0;
    uint32_t key = 0;
    for (int64_t tile = blockIdx.x; tile < t.tiles; tile += gridDim.x) {
        if (tile >= end) {  // the last tensor whose first tile is not behind this one
            int hi = t.count;
            while (hi - at > 1) {
                const int mid = (at + hi) >> 1;
                if (t.item[mid].first <= tile) at = mid; else hi = mid;
            }
            end = at + 1 < t.count ? t.item[at + 1].first : t.tiles;
            key = dither_key(h, t.item[at]);
        }
        const Item& d = t.item[at];
        const int64_t i = (tile - d.first) * kTile + threadIdx.x * kPer;
        const bool full = (tile - d.first + 1) * kTile <= d.n;  // for the whole CTA
        const int64_t rest = d.n - i;
        const int left = rest >= kPer ? kPer : rest > 0 ? static_cast<int>(rest) : 0;
        if constexpr (EIGHT) {
            const int64_t block = (tile - d.first) * (kTile / kBlock) + (threadIdx.x >> 5);
            bool done = true;
            if (full && d.plain) done = step8<T, true>(d, h, key, i, block, kPer);
            else if (block * kBlock < d.n) done = step8<T, false>(d, h, key, i, block, left);
            if (!done) {
                step8_exact<T>(d, h, tile);
                h = host;  // made again, as the tensor is, so that nothing is kept over the call
                if (dev) h = *dev;
                at = 0, end = 0;
            }
        } else {
            if (full && d.plain) step32<T, true>(d, h, i, kPer);
            else if (left) step32<T, false>(d, h, i, left);
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
            const int64_t state = EIGHT ? 8 : 16;
            const bool plain = !a.live && !off_by(a.p, 16) && !off_by(a.g, 16) && !off_by(a.m, state) && !off_by(a.v, state);
            t.item[t.count++] = {a.p, a.g, a.m, a.v, a.scale_m, a.scale_v, a.live, a.n, t.tiles, static_cast<uint32_t>(a.number), plain};
            t.tiles += (a.n + kTile - 1) / kTile;
        }
        if (t.count == 0) continue;
        const int64_t cap = static_cast<int64_t>(num_sms()) * 8;
        const int64_t grid = t.tiles < cap ? t.tiles : cap;
        ++g_launched;
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
    g_launched = 0;
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
