// The gated product by group, for one element type (gated_product_kernels.hpp).
#include "gated_product_kernels.hpp"

namespace mops::amd::gated_product {

template void forward<float>(const Inputs<float>&, float*, hipStream_t);
template void gradients<float>(const Inputs<float>&, const float*, float*, float*, hipStream_t);

} // namespace mops::amd::gated_product
