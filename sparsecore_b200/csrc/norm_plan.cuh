// How the norm kernels spread rows over threads and CTAs, and their entry by
// element type.
#pragma once

#include <algorithm>

#include "typed.cuh"

namespace slb {

// By the element type of y (norm_f32.cu, norm_bf16.cu, norm_f16.cu).
template <typename TY>
int norm_forward(const sl_norm_args& n, cudaStream_t s);
template <typename TY>
int norm_backward(const sl_norm_args& n, cudaStream_t s);

namespace norm {

constexpr int kMaxThreads = 512;
constexpr size_t kFullSmem = 224 * 1024;  // of the general backward kernel's rows and vectors

// How a row is spread: vectors of ve elements, nv of them a thread, over
// 32 * warps threads.
struct Plan {
    int ve, nv, warps;
};

// Vectors a thread that kernels are made for.  The fewest warps whose threads
// hold a row with at most `most` elements each.
inline int round_nv(int64_t n) {
    for (int k : {1, 2, 4, 6, 8, 32})
        if (n <= k) return k;
    return 32;
}
inline Plan make_plan(int64_t D, bool wide, int64_t elem, int most) {
    const int ve = wide ? static_cast<int>(16 / elem) : 1;
    const int64_t vecs = (D + ve - 1) / ve;
    if (!wide) most = 32;
    Plan p{ve, 0, 1};
    while ((vecs + 32 * p.warps - 1) / (32 * p.warps) > most / ve && p.warps < kMaxThreads / 32) p.warps *= 2;
    p.nv = round_nv((vecs + 32 * p.warps - 1) / (32 * p.warps));
    return p;
}
// Forward rows: up to 32 elements a thread, for few sums across threads
// (8191 x 4096 bf16 with both norms and a gate: 57 us, 62 with 16).
inline Plan forward_plan(int64_t D, bool wide, int64_t elem) { return make_plan(D, wide, elem, 32); }
// Backward rows without anything after the block: up to 16 elements a thread
// (16384 x 768 in 32 bits: 39 us with 2 warps a row, 53 us with one), 32 beyond
// 4096 columns; wider ones and the rest go to the general kernel.
constexpr int64_t kSimpleCols = 8192;
inline Plan backward_plan(int64_t D, bool wide, int64_t elem, bool full) {
    return make_plan(D, wide, elem, full ? 8 : D > 4096 ? 32 : 16);
}
// Rows a CTA takes at a time: several only where a row is one warp's, since
// the sums of a row of more warps pass a barrier of the CTA.
inline int backward_rows(const Plan& p, bool full) { return !full && p.warps == 1 ? 4 : 1; }

// The backward pass's split of the rows over CTAs of `rows` rows at a time.
struct Split {
    int64_t rows, ctas, seg;
    bool direct;
};
inline Split make_split(int64_t T, int64_t gate_rows, int64_t want, bool need_gate) {
    Split s{std::max<int64_t>(1, (T + want - 1) / want), 0, 0, false};
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

// CTAs that the rows are spread over: what an SM's registers hold side by side.
inline int64_t ctas_wanted(const Plan& p, bool full) {
    const int elems = p.ve * p.nv, threads = full || (elems > 8 && elems <= 16) ? 512 : elems > 16 ? 256 : 1024;
    return static_cast<int64_t>(num_sms()) * std::max(1, threads / (32 * p.warps * backward_rows(p, full)));
}

}  // namespace norm
}  // namespace slb
