// The cross entropy of a linear layer, for one element type (cross_entropy_kernels.hpp).
#include "cross_entropy_kernels.hpp"

namespace mops::amd::cross_entropy {

template void forward<double>(const Inputs<double>&, wide_t<double>*, wide_t<double>*, hipStream_t);
template void gradients<double>(
    const Inputs<double>&, const wide_t<double>*, const wide_t<double>*, const wide_t<double>*, double*, double*, hipStream_t
);

} // namespace mops::amd::cross_entropy
