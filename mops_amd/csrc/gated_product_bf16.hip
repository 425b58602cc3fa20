// The gated product by group, for one element type (gated_product_kernels.hpp).
#include "gated_product_kernels.hpp"

namespace mops::amd::gated_product {

template void forward<__bf16>(const Inputs<__bf16>&, __bf16*, hipStream_t);
template void gradients<__bf16>(const Inputs<__bf16>&, const __bf16*, __bf16*, __bf16*, hipStream_t);

} // namespace mops::amd::gated_product
