// Layer norm, dropout and residual-form kernels over rows of __nv_bfloat16.
#include "norm_kernels.cuh"

namespace qb {
QB_INSTANTIATE_NORM(__nv_bfloat16)
}  // namespace qb
