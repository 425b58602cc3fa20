// The gated product by group, for one element type (gated_product_kernels.hpp).
#include "gated_product_kernels.hpp"

namespace mops::amd::gated_product {

template void forward<_Float16>(const Inputs<_Float16>&, _Float16*, hipStream_t);
template void gradients<_Float16>(const Inputs<_Float16>&, const _Float16*, _Float16*, _Float16*, hipStream_t);

} // namespace mops::amd::gated_product
