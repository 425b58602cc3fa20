// The cross entropy of a linear layer, for one element type (cross_entropy_kernels.hpp).
#include "cross_entropy_kernels.hpp"

namespace mops::amd::cross_entropy {

template void forward<_Float16>(const Inputs<_Float16>&, wide_t<_Float16>*, wide_t<_Float16>*, hipStream_t);
template void gradients<_Float16>(
    const Inputs<_Float16>&, const wide_t<_Float16>*, const wide_t<_Float16>*, const wide_t<_Float16>*, _Float16*, _Float16*, hipStream_t
);

} // namespace mops::amd::cross_entropy
