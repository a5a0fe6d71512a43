// The norm kernels of bfloat16 rows.
#include "norm_kernels.cuh"

namespace slb {
template int norm_forward<__nv_bfloat16>(const sl_norm_args&, cudaStream_t);
template int norm_backward<__nv_bfloat16>(const sl_norm_args&, cudaStream_t);
}  // namespace slb
