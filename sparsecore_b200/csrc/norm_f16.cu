// The norm kernels of float16 rows.
#include "norm_kernels.cuh"

namespace slb {
template int norm_forward<__half>(const sl_norm_args&, cudaStream_t);
template int norm_backward<__half>(const sl_norm_args&, cudaStream_t);
}  // namespace slb
