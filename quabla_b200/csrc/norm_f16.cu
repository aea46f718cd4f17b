// Layer norm, dropout and residual-form kernels over rows of __half.
#include "norm_kernels.cuh"

namespace qb {
QB_INSTANTIATE_NORM(__half)
}  // namespace qb
