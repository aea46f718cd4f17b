// Layer norm, dropout and residual-form kernels over rows of double.
#include "norm_kernels.cuh"

namespace qb {
QB_INSTANTIATE_NORM(double)
}  // namespace qb
