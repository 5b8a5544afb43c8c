// nt_norm_backward.cu -- the backward group-norm kernels.
#include "nt_norm.cuh"

namespace nt {
namespace norm {
NormKernel backward_kernel(int32_t dtype, int v, bool whole, bool flat) { return pick_kernel<true>(dtype, v, whole, flat); }
cudaError_t read_backward_status(uint32_t *status, bool clear) { return read_status(status, clear); }
}  // namespace norm
}  // namespace nt
