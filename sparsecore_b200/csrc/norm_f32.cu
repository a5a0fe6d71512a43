// The norm kernels of 32-bit rows.
#include "norm_kernels.cuh"

namespace slb {
template int norm_forward<float>(const sl_norm_args&, cudaStream_t);
template int norm_backward<float>(const sl_norm_args&, cudaStream_t);
}  // namespace slb
