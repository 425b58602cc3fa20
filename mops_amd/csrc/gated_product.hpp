// The gated product by group, as the type-independent part of the operator calls
// it (gated_product.hip); the kernels are compiled once per element type.
#ifndef MOPS_AMD_GATED_PRODUCT_HPP
#define MOPS_AMD_GATED_PRODUCT_HPP

#include <cstdint>

#include <hip/hip_runtime.h>

#include "group_units.hpp"

namespace mops::amd::gated_product {

/// (the numbers of mops/layers.h)
enum class Activation : int32_t { SILU = 0, GELU = 1, SIGMOID = 2 };

/// What the two directions have in common: rows by group, A [rows, k_size], W [groups, k_size, 2 columns].
template <typename T> struct Inputs {
    const T *A, *W;
    RowGroups groups;
    int32_t k_size, columns;
    Activation activation;
};

template <typename T> void forward(const Inputs<T>& inputs, T* output, hipStream_t stream);
/// Either gradient may be null: not wanted.
template <typename T>
void gradients(const Inputs<T>& inputs, const T* grad_output, T* grad_A, T* grad_W, hipStream_t stream);

} // namespace mops::amd::gated_product

#endif
