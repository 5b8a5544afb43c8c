// nt_norm_forward.cu -- the forward group-norm kernels: both passes in one launch.
#include "nt_norm.cuh"

namespace nt {
namespace norm {
NormKernel forward_kernel(int32_t dtype, int v, bool whole, bool regular) { return pick_kernel<false, kBoth>(dtype, v, whole, regular); }
}  // namespace norm
}  // namespace nt
