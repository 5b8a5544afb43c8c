// nt_norm_backward.cu -- the backward group-norm kernels.
#include "nt_norm.cuh"

namespace nt {
namespace norm {
NormKernel backward_kernel(int32_t dtype, int v, bool whole) { return pick_kernel<true>(dtype, v, whole); }
}  // namespace norm
}  // namespace nt
