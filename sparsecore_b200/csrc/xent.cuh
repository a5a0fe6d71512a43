// What the parts of the linear cross entropy share: the layout of its
// buffers and of its operands as 16-bit planes, and how its kernels follow
// one another.
#pragma once

#include <utility>

#include "typed.cuh"

namespace slb {
namespace xent {

// A pass is a chain of short kernels.  Each may start while the one before it
// ends: it sets itself up, and then waits until all of that one's results are
// there (and so those of all before).  Every thread calls follow() before its
// first access to global memory.  33 x 1024 x 32003 fp16, losses only: 34 -> 31 us;
// 16384 x 768 x 256 fp32 trained: 141 -> 134 (graph replay 129 -> 126).
__device__ __forceinline__ void follow() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_follow() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... P, typename... A>
void launch_following(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, A&&... a) {
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t c{};
    c.gridDim = grid;
    c.blockDim = block;
    c.dynamicSmemBytes = smem;
    c.stream = s;
    c.attrs = &early;
    c.numAttrs = 1;
    ++g_launched;
    cudaLaunchKernelEx(&c, kernel, std::forward<A>(a)...);  // errors: cudaGetLastError, as of any launch
}

constexpr int kPart = 128;          // vocabulary columns of one partial (max, sum) of a row
constexpr int64_t kMostSlabFloats = int64_t(16) << 20;  // sums that a split product may leave to be joined
// softmax - onehot is held in fp16 times 2^15: in two planes 22 bits of what is
// above 2^-17, and what is below to within 2^-40.
constexpr float kGradScale = 32768.f;

// First bytes of the `prep` buffer.
struct Header {
    unsigned max_x, max_w, max_g;  // bits of the largest finite |.|
    int count;                     // tokens that count
    unsigned done;                 // CTAs of the finish that have written their sums
};

enum : int { kIgnored = -1, kInvalid = -2 };  // in place of a target

// Exponent of the power of two that brings values of up to `bits` (a float's
// bits, subnormal ones too) into [2^14, 2^15): -113 to 163.  Two fp16 planes
// then hold 22 bits of what is above 2^-17 of the largest, and what is smaller
// to within 2^-39 of the largest: an operand is as exact as a sum with its
// largest values in it can be, not element by element.
__device__ __forceinline__ int plane_exponent(unsigned bits) {
    if (bits == 0) return 0;
    return 14 - (bits >= 0x800000u ? static_cast<int>(bits >> 23) - 127 : -118 - __clz(bits));
}

// a * b, the second 1 but where the product is beyond a float's exponents.
struct Factor {
    float a, b;
};
__device__ __forceinline__ float pow2(int k) { return __int_as_float((k + 127) << 23); }  // -126 <= k <= 127
__device__ __forceinline__ Factor power_of_two(int k) {  // -252 <= k <= 254
    const int h = max(-126, min(127, k));
    return {pow2(h), pow2(k - h)};
}

// One operand: planes of [rows, stride] 16-bit values whose sum is it.
struct Operand {
    const void* base;
    int64_t rows, cols, stride;  // of a plane, in elements
    int64_t plane;               // elements from one plane to the next
};

struct Problem {
    Header* head;
    const int64_t* targets; // [T]
    int64_t ignore;
    float* row_max;         // [T] the softmax's maximum of each row, and
    float* row_inv;         // [T] one over its sum
    float* zt;              // [T] logit of the target
    float2* part;           // [parts][T]
    const float* grad;      // the loss's gradient, or
    const float* g_rows;    // [T] gradients of the single losses
    bool mean;
    int64_t T, D, V;
    bool f32;               // planes of fp16 pairs, scaled
    bool bf16;
};

// Target of token t; kIgnored, or kInvalid where there is no such column.
__device__ __forceinline__ int target_of(const Problem& p, int64_t t) {
    const int64_t v = p.targets[t];
    return v == p.ignore ? kIgnored : v < 0 || v >= p.V ? kInvalid : static_cast<int>(v);
}

// How a product [M, N] with a sum of K is split over the sum, and the floats
// that its parts leave to be joined (0: not split).
struct SplitSum {
    int splits, per_split;  // slices of 64 of the sum
    int64_t floats;
};
SplitSum split_sum(int64_t M, int64_t N, int64_t K, bool two_planes);

// C[m, n] = sum over k of A . B^T, and what becomes of it.
int gemm_stats(const Problem& p, const Operand& x, const Operand& w, cudaStream_t s);
// A vocabulary of one tile (up to 256): losses, their sum and the gradient of
// the logits (if g.base) at once.  loss, rows: written where set; sums,
// counts: one for each of the launch's CTAs (kMostCtas at most).
constexpr int kOneTile = 256, kMostCtas = 512;
struct Losses {
    float *loss, *rows;
    double* sums;
    int* counts;
};
int gemm_losses(const Problem& p, const Operand& x, const Operand& w, const Operand& g, const Losses& l, cudaStream_t s);
// Columns [v0, v0 + cols) of the gradient of the logits, as planes in g.
int gemm_grad(const Problem& p, const Operand& x, const Operand& w, int64_t v0, int64_t cols, const Operand& g,
              cudaStream_t s);

struct Output {
    void* dst;        // [M, N] in the caller's type
    int dtype;
    float* acc;       // [M, N] sums of the pieces so far, or null
    bool first, last; // piece
    float* slabs;     // workspace of a split sum
    bool by_x;        // undo x's scale, not w's
};
// dx += G[T, cols] . W[cols, D]
int gemm_dx(const Problem& p, const Operand& g, int64_t cols, const Operand& w, int64_t v0, const Output& o, cudaStream_t s);
// dw[v0 ...] = G^T[cols, T] . X[T, D]
int gemm_dw(const Problem& p, const Operand& g, int64_t cols, const Operand& x, const Output& o, cudaStream_t s);

}  // namespace xent
}  // namespace slb
