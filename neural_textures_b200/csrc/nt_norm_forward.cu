// nt_norm_forward.cu -- the forward group-norm kernels.
#include "nt_norm.cuh"

namespace nt {
namespace norm {
NormKernel forward_kernel(int32_t dtype, int v, bool whole, bool flat) { return pick_kernel<false>(dtype, v, whole, flat); }
cudaError_t read_forward_status(uint32_t *status, bool clear) { return read_status(status, clear); }
}  // namespace norm
}  // namespace nt
