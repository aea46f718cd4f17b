// Layer norm, dropout and residual-form kernels over rows of float.
#include "norm_kernels.cuh"

namespace qb {
QB_INSTANTIATE_NORM(float)
}  // namespace qb
