// C++ API of the operators of the layers around the sums over edges; what each
// of them computes is written down in mops/layers.h. Device memory only; not
// part of lab-cosmo/mops. scalar_t: float, double, mops::bfloat16, mops::float16.
#ifndef MOPS_LAYERS_HPP
#define MOPS_LAYERS_HPP

#include <cstdint>

#include "mops/exports.h"
#include "mops/tensor.hpp"

namespace mops {

/// 16-bit floating-point numbers by their bits: storage only, no arithmetic on the host.
struct MOPS_EXPORT bfloat16 {
    uint16_t bits;
};
struct MOPS_EXPORT float16 {
    uint16_t bits;
};

namespace cuda {

void MOPS_EXPORT order_by_group(Tensor<int32_t, 1> order, Tensor<int32_t, 1> offsets, Tensor<int32_t, 1> indices);

template <typename scalar_t>
void MOPS_EXPORT scaled_embedding(
    Tensor<scalar_t, 2> output, Tensor<scalar_t, 2> table, Tensor<int32_t, 1> indices, double scale
);

template <typename scalar_t>
void MOPS_EXPORT scaled_embedding_vjp(
    Tensor<scalar_t, 2> grad_table, Tensor<scalar_t, 2> grad_output, Tensor<int32_t, 1> indices,
    Tensor<int32_t, 1> order, Tensor<int32_t, 1> offsets, double scale
);

template <typename scalar_t>
void MOPS_EXPORT grouped_matrix_product(
    Tensor<scalar_t, 2> output, Tensor<scalar_t, 2> A, Tensor<scalar_t, 3> W, Tensor<int32_t, 1> offsets,
    Tensor<int32_t, 1> order
);

template <typename scalar_t>
void MOPS_EXPORT grouped_matrix_product_vjp(
    Tensor<scalar_t, 2> grad_A, Tensor<scalar_t, 3> grad_W, Tensor<scalar_t, 2> grad_output, Tensor<scalar_t, 2> A,
    Tensor<scalar_t, 3> W, Tensor<int32_t, 1> offsets, Tensor<int32_t, 1> order
);

template <typename scalar_t>
void MOPS_EXPORT gated_residual_norm(
    Tensor<scalar_t, 2> state, Tensor<scalar_t, 2> next, Tensor<scalar_t, 2> residual, Tensor<scalar_t, 2> block,
    Tensor<scalar_t, 2> gate, Tensor<scalar_t, 1> weight_block, Tensor<scalar_t, 1> weight_next,
    double residual_scale, double epsilon
);

template <typename scalar_t>
void MOPS_EXPORT gated_residual_norm_vjp(
    Tensor<scalar_t, 2> grad_residual, Tensor<scalar_t, 2> grad_block, Tensor<scalar_t, 2> grad_gate,
    Tensor<scalar_t, 1> grad_weight_block, Tensor<scalar_t, 1> grad_weight_next, Tensor<scalar_t, 2> grad_state,
    Tensor<scalar_t, 2> grad_next, Tensor<scalar_t, 2> residual, Tensor<scalar_t, 2> block, Tensor<scalar_t, 2> gate,
    Tensor<scalar_t, 1> weight_block, Tensor<scalar_t, 1> weight_next, double residual_scale, double epsilon
);

} // namespace cuda
} // namespace mops

#endif
