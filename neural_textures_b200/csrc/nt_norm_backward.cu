// nt_norm_backward.cu -- the backward group-norm kernels: both passes in one launch.
#include "nt_norm.cuh"

namespace nt {
namespace norm {
NormKernel backward_kernel(int32_t dtype, int v, bool whole, bool regular) { return pick_kernel<true, kBoth>(dtype, v, whole, regular); }
}  // namespace norm
}  // namespace nt
