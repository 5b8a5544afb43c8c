// nt_norm_backward_apply.cu -- the backward group-norm kernels: the result.
#include "nt_norm.cuh"

namespace nt {
namespace norm {
NormKernel backward_apply_kernel(int32_t dtype, int v, bool whole, bool regular) { return pick_kernel<true, kApply>(dtype, v, whole, regular); }
}  // namespace norm
}  // namespace nt
