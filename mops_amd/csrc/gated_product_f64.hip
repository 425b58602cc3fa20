// The gated product by group, for one element type (gated_product_kernels.hpp).
#include "gated_product_kernels.hpp"

namespace mops::amd::gated_product {

template void forward<double>(const Inputs<double>&, double*, hipStream_t);
template void gradients<double>(const Inputs<double>&, const double*, double*, double*, hipStream_t);

} // namespace mops::amd::gated_product
