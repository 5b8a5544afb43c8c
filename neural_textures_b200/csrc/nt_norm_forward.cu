// nt_norm_forward.cu -- the forward group-norm kernels.
#include "nt_norm.cuh"

namespace nt {
namespace norm {
NormKernel forward_kernel(int32_t dtype, int v, bool whole) { return pick_kernel<false>(dtype, v, whole); }
}  // namespace norm
}  // namespace nt
