// nt_norm_forward_apply.cu -- the forward group-norm kernels: the result.
#include "nt_norm.cuh"

namespace nt {
namespace norm {
NormKernel forward_apply_kernel(int32_t dtype, int v, bool whole, bool regular) { return pick_kernel<false, kApply>(dtype, v, whole, regular); }
}  // namespace norm
}  // namespace nt
