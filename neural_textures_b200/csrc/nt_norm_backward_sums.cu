// nt_norm_backward_sums.cu -- the backward group-norm kernels: the sums.
#include "nt_norm.cuh"

namespace nt {
namespace norm {
NormKernel backward_sums_kernel(int32_t dtype, int v, bool whole, bool regular) { return pick_kernel<true, kSums>(dtype, v, whole, regular); }
}  // namespace norm
}  // namespace nt
