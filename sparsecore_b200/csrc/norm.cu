// Entry points of the fused norms: checks, workspace and dispatch by type.
#include "norm_plan.cuh"

namespace slb {
namespace {

int check(const sl_norm_args* n, const char* fn, bool back) {
    SL_REQUIRE(n != nullptr, fn, "NULL arguments");
    SL_REQUIRE(n->rows >= 0 && n->rows <= INT_MAX, fn, "rows must fit 31 bits");
    SL_REQUIRE(n->cols >= 1 && n->cols <= SL_NORM_MAX_COLS, fn, "columns must be 1 to 16384");
    SL_REQUIRE(n->kind == SL_NORM_LAYER || n->kind == SL_NORM_RMS, fn, "unknown kind");
    SL_REQUIRE(known_dtype(n->dtype) && (n->residual_dtype == n->dtype || n->residual_dtype == SL_F32), fn, "unsupported residual type");
    SL_REQUIRE(n->weight_dtype == n->dtype || n->weight_dtype == SL_F32, fn, "unsupported weight type");
    SL_REQUIRE(!n->gate || n->gate_dtype == n->dtype || n->gate_dtype == SL_F32, fn, "unsupported gate type");
    SL_REQUIRE(!n->gate || n->rows == 0 || (n->gate_groups >= 1 && n->rows % n->gate_groups == 0), fn,
               "the rows must divide into the gate's rows");
    if (n->rows == 0) return SL_OK;
    SL_REQUIRE(n->weight && n->out, fn, "NULL operand");
    SL_REQUIRE(back || (n->y && n->residual && n->h), fn, "NULL operand");
    SL_REQUIRE(!back || (n->y && n->stats && n->dout && n->dh && n->dresidual && n->workspace), fn, "NULL operand");
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
    SL_REQUIRE(!off_by(n->gate, eg) && !off_by(n->dgate, eg) && !off_by(n->workspace, 16) && !off_by(n->stats, 16), fn,
               "misaligned operand");
    return SL_OK;
}

}  // namespace
}  // namespace slb

using namespace slb;

extern "C" int64_t sl_norm_workspace_bytes(int64_t rows, int64_t cols, int64_t gate_groups) {
    if (rows <= 0 || cols <= 0 || cols > SL_NORM_MAX_COLS) return 0;
    // the most CTAs that make_split gives for any type and alignment, and a run's last CTA each
    int64_t most = 0;
    for (int k = 0; k < 6; ++k)
        most = std::max(most, norm::ctas_wanted(norm::backward_plan(cols, k >= 2, k >= 4 ? 2 : 4, k & 1), k & 1));
    most += std::max<int64_t>(gate_groups, 1);
    return (5 * cols + 1) * std::min(rows, most) * 4 + 16;
}

extern "C" int sl_norm_forward(const sl_norm_args* n, void* stream) {
    if (int rc = check(n, "sl_norm_forward", false)) return rc;
    if (n->rows == 0) return SL_OK;
    if (n->dtype == SL_F32) return norm_forward<float>(*n, as_stream(stream));
    if (n->dtype == SL_BF16) return norm_forward<__nv_bfloat16>(*n, as_stream(stream));
    return norm_forward<__half>(*n, as_stream(stream));
}

extern "C" int sl_norm_backward(const sl_norm_args* n, void* stream) {
    g_launched = 0;
    if (int rc = check(n, "sl_norm_backward", true)) return rc;
    if (n->rows == 0) return SL_OK;
    if (n->dtype == SL_F32) return norm_backward<float>(*n, as_stream(stream));
    if (n->dtype == SL_BF16) return norm_backward<__nv_bfloat16>(*n, as_stream(stream));
    return norm_backward<__half>(*n, as_stream(stream));
}
