// The cross entropy of a linear layer, for one element type (cross_entropy_kernels.hpp).
#include "cross_entropy_kernels.hpp"

namespace mops::amd::cross_entropy {

template void forward<__bf16>(const Inputs<__bf16>&, wide_t<__bf16>*, wide_t<__bf16>*, hipStream_t);
template void gradients<__bf16>(
    const Inputs<__bf16>&, const wide_t<__bf16>*, const wide_t<__bf16>*, const wide_t<__bf16>*, __bf16*, __bf16*, hipStream_t
);

} // namespace mops::amd::cross_entropy
