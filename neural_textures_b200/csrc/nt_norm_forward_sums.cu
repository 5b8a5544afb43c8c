// nt_norm_forward_sums.cu -- the forward group-norm kernels: the sums.
#include "nt_norm.cuh"

namespace nt {
namespace norm {
NormKernel forward_sums_kernel(int32_t dtype, int v, bool whole, bool regular) { return pick_kernel<false, kSums>(dtype, v, whole, regular); }
}  // namespace norm
}  // namespace nt
