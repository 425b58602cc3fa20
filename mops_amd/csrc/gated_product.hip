// The gated product by group: arguments and entry points (the kernels:
// gated_product_kernels.hpp).
#include "mops/layers.hpp"

#include "checks.hpp"
#include "gated_product.hpp"
#include "group_checks.hpp"
#include "numbers.hpp"
#include "runtime.hpp"

namespace mops::cuda {

using namespace mops::amd;

namespace {

template <typename scalar_t>
gated_product::Inputs<device_t<scalar_t>> check_inputs(
    const checks::Validator& check, Tensor<scalar_t, 2> A, Tensor<scalar_t, 3> W, Tensor<int32_t, 1> offsets,
    Tensor<int32_t, 1> order, int32_t activation
) {
    const RowGroups groups = check_groups(check, A, W, offsets, order);
    if (W.shape[2] % 2 != 0) {
        throw std::runtime_error(
            "W must have an even number of columns (those of the gate, then as many more) in " + check.operation() +
            ", got " + std::to_string(W.shape[2])
        );
    }
    if (activation < 0 || activation > static_cast<int32_t>(gated_product::Activation::SIGMOID)) {
        throw std::runtime_error(
            "activation must be 0 (silu), 1 (gelu) or 2 (sigmoid) in " + check.operation() + ", got " +
            std::to_string(activation)
        );
    }
    return {
        data_of(A), data_of(W), groups, count_i32(W.shape[1], "W.shape[1]"), count_i32(W.shape[2], "W.shape[2]") / 2,
        static_cast<gated_product::Activation>(activation),
    };
}

/// grad_output and output have the rows of A and half the columns of W.
template <typename scalar_t>
void check_output(
    const checks::Validator& check, Tensor<scalar_t, 2> output, const char* name, Tensor<scalar_t, 2> A,
    Tensor<scalar_t, 3> W
) {
    check.same_extent(checks::axis_of(output, name, 0), checks::axis_of(A, "A", 0));
    if (output.shape[1] != W.shape[2] / 2) {
        throw std::runtime_error(
            std::string(name) + " must have " + std::to_string(W.shape[2] / 2) + " columns (half of W's) in " +
            check.operation() + ", got " + std::to_string(output.shape[1])
        );
    }
}

} // namespace

template <typename scalar_t>
void gated_grouped_product(
    Tensor<scalar_t, 2> output, Tensor<scalar_t, 2> A, Tensor<scalar_t, 3> W, Tensor<int32_t, 1> offsets,
    Tensor<int32_t, 1> order, int32_t activation
) {
    const checks::Validator check("gated_grouped_product");
    const auto inputs = check_inputs(check, A, W, offsets, order, activation);
    check_output(check, output, "output", A, W);
    if (inputs.groups.n_rows > 0 && inputs.columns > 0) {
        gated_product::forward(inputs, data_of(output), current_stream());
    }
    finish_call("gated_grouped_product");
}

template <typename scalar_t>
void gated_grouped_product_vjp(
    Tensor<scalar_t, 2> grad_A, Tensor<scalar_t, 3> grad_W, Tensor<scalar_t, 2> grad_output, Tensor<scalar_t, 2> A,
    Tensor<scalar_t, 3> W, Tensor<int32_t, 1> offsets, Tensor<int32_t, 1> order, int32_t activation
) {
    using checks::axis_of;
    const checks::Validator check("gated_grouped_product_vjp");
    const auto inputs = check_inputs(check, A, W, offsets, order, activation);
    check_output(check, grad_output, "grad_output", A, W);
    for (size_t d = 0; d < 2 && grad_A.data != nullptr; d++) {
        check.same_extent(axis_of(grad_A, "grad_A", d), axis_of(A, "A", d));
    }
    for (size_t d = 0; d < 3 && grad_W.data != nullptr; d++) {
        check.same_extent(axis_of(grad_W, "grad_W", d), axis_of(W, "W", d));
    }
    const bool of_A = grad_A.data != nullptr && inputs.groups.n_rows > 0 && inputs.k_size > 0;
    const bool of_W = grad_W.data != nullptr && inputs.groups.n_groups > 0 && inputs.k_size > 0 && inputs.columns > 0;
    if (of_A || of_W) {
        gated_product::gradients(
            inputs, data_of(grad_output), of_A ? data_of(grad_A) : nullptr, of_W ? data_of(grad_W) : nullptr,
            current_stream()
        );
    }
    finish_call("gated_grouped_product_vjp");
}

#define MOPS_GATED_PRODUCT_INSTANTIATE(T)                                                          \
    template void gated_grouped_product<T>(                                                        \
        Tensor<T, 2>, Tensor<T, 2>, Tensor<T, 3>, Tensor<int32_t, 1>, Tensor<int32_t, 1>, int32_t  \
    );                                                                                             \
    template void gated_grouped_product_vjp<T>(                                                    \
        Tensor<T, 2>, Tensor<T, 3>, Tensor<T, 2>, Tensor<T, 2>, Tensor<T, 3>, Tensor<int32_t, 1>,  \
        Tensor<int32_t, 1>, int32_t                                                                \
    );
MOPS_GATED_PRODUCT_INSTANTIATE(float)
MOPS_GATED_PRODUCT_INSTANTIATE(double)
MOPS_GATED_PRODUCT_INSTANTIATE(bfloat16)
MOPS_GATED_PRODUCT_INSTANTIATE(float16)

} // namespace mops::cuda
