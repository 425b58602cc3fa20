// C++ API of the operators of the layers around the sums over edges; what each
// of them computes is written down in mops/layers.h. Device memory only; not
// part of lab-cosmo/mops. scalar_t: float, double, mops::bfloat16, mops::float16.
#ifndef MOPS_LAYERS_HPP
#define MOPS_LAYERS_HPP

#include <cstddef>
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

/// A tensor among others of any type: `size` numbers that follow each other.
enum class GradientType : int32_t { F32 = 0, F64 = 1, BF16 = 2, F16 = 3 };
struct Gradient {
    void* data;
    int64_t size;
    GradientType type;
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

/// activation: 0 silu, 1 gelu, 2 sigmoid.
template <typename scalar_t>
void MOPS_EXPORT gated_grouped_product(
    Tensor<scalar_t, 2> output, Tensor<scalar_t, 2> A, Tensor<scalar_t, 3> W, Tensor<int32_t, 1> offsets,
    Tensor<int32_t, 1> order, int32_t activation
);

template <typename scalar_t>
void MOPS_EXPORT gated_grouped_product_vjp(
    Tensor<scalar_t, 2> grad_A, Tensor<scalar_t, 3> grad_W, Tensor<scalar_t, 2> grad_output, Tensor<scalar_t, 2> A,
    Tensor<scalar_t, 3> W, Tensor<int32_t, 1> offsets, Tensor<int32_t, 1> order, int32_t activation
);

/// sum_t: float; double for double.
template <typename scalar_t, typename sum_t>
void MOPS_EXPORT linear_cross_entropy(
    Tensor<sum_t, 1> losses, Tensor<sum_t, 1> log_sums, Tensor<scalar_t, 2> A, Tensor<scalar_t, 2> W,
    Tensor<int32_t, 1> targets
);

template <typename scalar_t, typename sum_t>
void MOPS_EXPORT linear_cross_entropy_vjp(
    Tensor<scalar_t, 2> grad_A, Tensor<scalar_t, 2> grad_W, Tensor<sum_t, 1> grad_losses,
    Tensor<sum_t, 1> grad_log_sums, Tensor<scalar_t, 2> A, Tensor<scalar_t, 2> W, Tensor<int32_t, 1> targets,
    Tensor<sum_t, 1> log_sums
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

/// sum_t: float or double.
template <typename sum_t>
void MOPS_EXPORT gradient_norm(Tensor<sum_t, 1> norm, const Gradient* gradients, size_t n_gradients);

/// outputs may be the gradients themselves: in place.
template <typename sum_t>
void MOPS_EXPORT clip_gradients(
    Tensor<sum_t, 1> norm, const Gradient* outputs, const Gradient* gradients, size_t n_gradients, double max_norm
);

} // namespace cuda
} // namespace mops

#endif
