// The cross entropy of a linear layer, for one element type (cross_entropy_kernels.hpp).
#include "cross_entropy_kernels.hpp"

namespace mops::amd::cross_entropy {

template void forward<float>(const Inputs<float>&, wide_t<float>*, wide_t<float>*, hipStream_t);
template void gradients<float>(
    const Inputs<float>&, const wide_t<float>*, const wide_t<float>*, const wide_t<float>*, float*, float*, hipStream_t
);

} // namespace mops::amd::cross_entropy
