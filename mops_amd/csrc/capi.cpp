// The C ABI: 60 operation entry points, the error-text accessor, the
// AMD-specific additions and the layers' operators. Every operation wrapper does the same three
// things as mops/src/<op>/capi.cpp of lab-cosmo/mops: convert each int64
// extent to size_t (rejecting negative values), call the C++ template, and
// translate exceptions into a status code plus a per-thread message.
// The wrappers are generated from the parameter lists in
// mops/detail/signatures.h.
#include <cstddef>
#include <cstdint>
#include <stdexcept>
#include <string>

#include "mops.h"
#include "mops.hpp"

#include "first_occurrences.hpp"
#include "no_alloc.hpp"
#include "edge_order.hpp"
#include "runtime.hpp"

namespace {

thread_local std::string LAST_ERROR;

size_t extent(int64_t value) {
    if (value < 0 || static_cast<uint64_t>(value) > static_cast<uint64_t>(SIZE_MAX)) {
        throw std::runtime_error(
            "integer value '" + std::to_string(value) + "' does not fit in size_t"
        );
    }
    return static_cast<size_t>(value);
}

// C view -> C++ view, one overload per struct type
#define MOPS_DEFINE_VIEW(STRUCT, ELEMENT)                                                          \
    [[maybe_unused]] mops::Tensor<ELEMENT, sizeof(STRUCT::shape) / sizeof(int64_t)> view(STRUCT t) {                \
        constexpr size_t N = sizeof(STRUCT::shape) / sizeof(int64_t);                              \
        mops::Tensor<ELEMENT, N> result;                                                           \
        result.data = t.data;                                                                      \
        for (size_t d = 0; d < N; d++) {                                                           \
            result.shape[d] = extent(t.shape[d]);                                                  \
        }                                                                                          \
        return result;                                                                             \
    }

MOPS_DEFINE_VIEW(mops_tensor_1d_f32_t, float)
MOPS_DEFINE_VIEW(mops_tensor_2d_f32_t, float)
MOPS_DEFINE_VIEW(mops_tensor_3d_f32_t, float)
MOPS_DEFINE_VIEW(mops_tensor_1d_f64_t, double)
MOPS_DEFINE_VIEW(mops_tensor_2d_f64_t, double)
MOPS_DEFINE_VIEW(mops_tensor_3d_f64_t, double)
MOPS_DEFINE_VIEW(mops_tensor_1d_i32_t, int32_t)
MOPS_DEFINE_VIEW(mops_tensor_2d_i32_t, int32_t)

// 16-bit floating-point data: given by its bits
#define MOPS_DEFINE_16_BIT_VIEW(STRUCT, ELEMENT)                                                   \
    mops::Tensor<ELEMENT, sizeof(STRUCT::shape) / sizeof(int64_t)> view(STRUCT t) {                \
        constexpr size_t N = sizeof(STRUCT::shape) / sizeof(int64_t);                              \
        mops::Tensor<ELEMENT, N> result;                                                           \
        result.data = reinterpret_cast<ELEMENT*>(t.data);                                          \
        for (size_t d = 0; d < N; d++) {                                                           \
            result.shape[d] = extent(t.shape[d]);                                                  \
        }                                                                                          \
        return result;                                                                             \
    }

MOPS_DEFINE_16_BIT_VIEW(mops_tensor_1d_bf16_t, mops::bfloat16)
MOPS_DEFINE_16_BIT_VIEW(mops_tensor_2d_bf16_t, mops::bfloat16)
MOPS_DEFINE_16_BIT_VIEW(mops_tensor_3d_bf16_t, mops::bfloat16)
MOPS_DEFINE_16_BIT_VIEW(mops_tensor_1d_f16_t, mops::float16)
MOPS_DEFINE_16_BIT_VIEW(mops_tensor_2d_f16_t, mops::float16)
MOPS_DEFINE_16_BIT_VIEW(mops_tensor_3d_f16_t, mops::float16)

// A tensor that the C ABI declares with the 2-D struct although it has three
// dimensions: the missing last extent is taken from `last`.
template <typename Element, typename Struct2D>
mops::Tensor<Element, 3> view_with_last_extent(Struct2D t, int64_t last) {
    mops::Tensor<Element, 3> result;
    result.data = t.data;
    result.shape[0] = extent(t.shape[0]);
    result.shape[1] = extent(t.shape[1]);
    result.shape[2] = extent(last);
    return result;
}

[[maybe_unused]] mops::Tensor<float, 3> view_3d(mops_tensor_2d_f32_t t, int64_t last) {
    return view_with_last_extent<float>(t, last);
}

[[maybe_unused]] mops::Tensor<double, 3> view_3d(mops_tensor_2d_f64_t t, int64_t last) {
    return view_with_last_extent<double>(t, last);
}

} // namespace

void mops::store_error_message(std::string message) { LAST_ERROR = std::move(message); }

const std::string& mops::get_last_error_message() { return LAST_ERROR; }

extern "C" const char* mops_get_last_error_message(void) { return LAST_ERROR.c_str(); }

#define MOPS_FORWARD_R1(NAME) view(NAME)
#define MOPS_FORWARD_R2(NAME) view(NAME)
#define MOPS_FORWARD_R3(NAME) view(NAME)
#define MOPS_FORWARD_I1(NAME) view(NAME)
#define MOPS_FORWARD_I2(NAME) view(NAME)
#define MOPS_FORWARD_Q3(NAME) view_3d(NAME, W.shape[2])
#define MOPS_FORWARD_FIRST(KIND, NAME) MOPS_FORWARD_##KIND(NAME)
#define MOPS_FORWARD_NEXT(KIND, NAME) , MOPS_FORWARD_##KIND(NAME)

#define MOPS_C_DEFINE(DEVICE, NAMESPACE, NAME, S, T, PARAMS)                                       \
    extern "C" MOPS_C_PROTOTYPE(DEVICE, NAME, S, PARAMS) {                                         \
        MOPS_CATCH_EXCEPTIONS_BEGIN                                                                \
        NAMESPACE NAME<T>(PARAMS(MOPS_FORWARD_FIRST, MOPS_FORWARD_NEXT));                          \
        MOPS_CATCH_EXCEPTIONS_END                                                                  \
    }

#define MOPS_C_DEFINE_ALL(NAME, PARAMS)                                                            \
    MOPS_C_DEFINE(, ::mops::, NAME, f32, float, PARAMS)                                            \
    MOPS_C_DEFINE(, ::mops::, NAME, f64, double, PARAMS)                                           \
    MOPS_C_DEFINE(cuda_, ::mops::cuda::, NAME, f32, float, PARAMS)                                 \
    MOPS_C_DEFINE(cuda_, ::mops::cuda::, NAME, f64, double, PARAMS)

MOPS_FOR_EACH_FUNCTION(MOPS_C_DEFINE_ALL)

// ---- AMD-specific additions (mops/amd.h) ---------------------------------

extern "C" int mops_amd_set_stream(void* hip_stream) {
    mops::amd::set_current_stream(static_cast<hipStream_t>(hip_stream));
    return 0;
}

extern "C" void* mops_amd_get_stream(void) { return mops::amd::current_stream(); }

extern "C" int mops_amd_set_synchronous(int synchronous) {
    return mops::amd::set_synchronous(synchronous != 0) ? 1 : 0;
}

extern "C" int mops_amd_first_occurrences(
    const int32_t* sorted_indices, int64_t n_input, int64_t n_output, int32_t* first_occurrences
) {
    MOPS_CATCH_EXCEPTIONS_BEGIN
    mops::amd::first_occurrences(
        sorted_indices,
        mops::amd::narrow_i32(extent(n_input), "n_input"),
        mops::amd::narrow_i32(extent(n_output), "n_output"),
        first_occurrences,
        mops::amd::current_stream()
    );
    mops::amd::finish_call("first_occurrences");
    MOPS_CATCH_EXCEPTIONS_END
}

extern "C" int mops_amd_accept_unsorted_indices(int accept) {
    return mops::amd::set_accept_unsorted(accept != 0) ? 1 : 0;
}

extern "C" int mops_amd_kernel_timing(int enable) {
    return mops::amd::set_kernel_timing(enable != 0) ? 1 : 0;
}

extern "C" int mops_amd_kernel_time(double* total_milliseconds, int64_t* launches) {
    MOPS_CATCH_EXCEPTIONS_BEGIN
    if (total_milliseconds == nullptr || launches == nullptr) {
        throw std::runtime_error("mops_amd_kernel_time: both result pointers must be given");
    }
    mops::amd::collect_kernel_time(total_milliseconds, launches);
    MOPS_CATCH_EXCEPTIONS_END
}

extern "C" int mops_amd_reserve_scratch(int64_t bytes) {
    MOPS_CATCH_EXCEPTIONS_BEGIN
    (void)mops::amd::scratch(extent(bytes));
    mops::amd::finish_call("reserve_scratch");
    MOPS_CATCH_EXCEPTIONS_END
}

extern "C" int64_t mops_amd_scratch_capacity(void) {
    return static_cast<int64_t>(mops::amd::scratch_capacity());
}

extern "C" int mops_amd_sparse_accumulation_scatter_add_with_weights_vjp_no_alloc_f32(
    MOPS_SASAW_VJP_PARAMS(MOPS_C_FIRST_f32, MOPS_C_NEXT_f32)
) {
    MOPS_CATCH_EXCEPTIONS_BEGIN
    mops::amd::sasaw_vjp_no_alloc(MOPS_SASAW_VJP_PARAMS(MOPS_FORWARD_FIRST, MOPS_FORWARD_NEXT));
    MOPS_CATCH_EXCEPTIONS_END
}

// ---- the layers' operators (mops/layers.h) --------------------------------

extern "C" int mops_amd_order_by_group(
    mops_tensor_1d_i32_t order, mops_tensor_1d_i32_t offsets, mops_tensor_1d_i32_t indices
) {
    MOPS_CATCH_EXCEPTIONS_BEGIN
    mops::cuda::order_by_group(view(order), view(offsets), view(indices));
    MOPS_CATCH_EXCEPTIONS_END
}

namespace {

/// The same layout, as the C++ API has it.
const mops::Gradient* gradients_of(const mops_amd_gradient_t* gradients) {
    static_assert(sizeof(mops::Gradient) == sizeof(mops_amd_gradient_t), "");
    static_assert(offsetof(mops::Gradient, size) == offsetof(mops_amd_gradient_t, size), "");
    static_assert(offsetof(mops::Gradient, type) == offsetof(mops_amd_gradient_t, type), "");
    return reinterpret_cast<const mops::Gradient*>(gradients);
}

} // namespace

#define MOPS_GRADIENTS_DEFINE(W, T)                                                                \
    extern "C" int mops_amd_gradient_norm_##W(                                                     \
        mops_tensor_1d_##W##_t norm, const mops_amd_gradient_t* gradients, int64_t n_gradients     \
    ) {                                                                                            \
        MOPS_CATCH_EXCEPTIONS_BEGIN                                                                \
        mops::cuda::gradient_norm<T>(view(norm), gradients_of(gradients), extent(n_gradients));    \
        MOPS_CATCH_EXCEPTIONS_END                                                                  \
    }                                                                                              \
    extern "C" int mops_amd_clip_gradients_##W(                                                    \
        mops_tensor_1d_##W##_t norm, const mops_amd_gradient_t* outputs,                           \
        const mops_amd_gradient_t* gradients, int64_t n_gradients, double max_norm                 \
    ) {                                                                                            \
        MOPS_CATCH_EXCEPTIONS_BEGIN                                                                \
        mops::cuda::clip_gradients<T>(                                                             \
            view(norm), gradients_of(outputs), gradients_of(gradients), extent(n_gradients), max_norm \
        );                                                                                         \
        MOPS_CATCH_EXCEPTIONS_END                                                                  \
    }
MOPS_GRADIENTS_DEFINE(f32, float)
MOPS_GRADIENTS_DEFINE(f64, double)

#define MOPS_LAYERS_DEFINE(S, T, R, SUM)                                                           \
    extern "C" int mops_amd_scaled_embedding_##S(                                                  \
        mops_tensor_2d_##S##_t output, mops_tensor_2d_##S##_t table, mops_tensor_1d_i32_t indices, \
        double scale                                                                               \
    ) {                                                                                            \
        MOPS_CATCH_EXCEPTIONS_BEGIN                                                                \
        mops::cuda::scaled_embedding<T>(view(output), view(table), view(indices), scale);          \
        MOPS_CATCH_EXCEPTIONS_END                                                                  \
    }                                                                                              \
    extern "C" int mops_amd_scaled_embedding_vjp_##S(                                              \
        mops_tensor_2d_##S##_t grad_table, mops_tensor_2d_##S##_t grad_output,                     \
        mops_tensor_1d_i32_t indices, mops_tensor_1d_i32_t order, mops_tensor_1d_i32_t offsets,    \
        double scale                                                                               \
    ) {                                                                                            \
        MOPS_CATCH_EXCEPTIONS_BEGIN                                                                \
        mops::cuda::scaled_embedding_vjp<T>(                                                       \
            view(grad_table), view(grad_output), view(indices), view(order), view(offsets), scale  \
        );                                                                                         \
        MOPS_CATCH_EXCEPTIONS_END                                                                  \
    }                                                                                              \
    extern "C" int mops_amd_grouped_matrix_product_##S(                                            \
        mops_tensor_2d_##S##_t output, mops_tensor_2d_##S##_t A, mops_tensor_3d_##S##_t W,         \
        mops_tensor_1d_i32_t offsets, mops_tensor_1d_i32_t order                                   \
    ) {                                                                                            \
        MOPS_CATCH_EXCEPTIONS_BEGIN                                                                \
        mops::cuda::grouped_matrix_product<T>(                                                     \
            view(output), view(A), view(W), view(offsets), view(order)                             \
        );                                                                                         \
        MOPS_CATCH_EXCEPTIONS_END                                                                  \
    }                                                                                              \
    extern "C" int mops_amd_grouped_matrix_product_vjp_##S(                                        \
        mops_tensor_2d_##S##_t grad_A, mops_tensor_3d_##S##_t grad_W,                              \
        mops_tensor_2d_##S##_t grad_output, mops_tensor_2d_##S##_t A, mops_tensor_3d_##S##_t W,    \
        mops_tensor_1d_i32_t offsets, mops_tensor_1d_i32_t order                                   \
    ) {                                                                                            \
        MOPS_CATCH_EXCEPTIONS_BEGIN                                                                \
        mops::cuda::grouped_matrix_product_vjp<T>(                                                 \
            view(grad_A), view(grad_W), view(grad_output), view(A), view(W), view(offsets), view(order) \
        );                                                                                         \
        MOPS_CATCH_EXCEPTIONS_END                                                                  \
    }                                                                                              \
    extern "C" int mops_amd_gated_grouped_product_##S(                                             \
        mops_tensor_2d_##S##_t output, mops_tensor_2d_##S##_t A, mops_tensor_3d_##S##_t W,         \
        mops_tensor_1d_i32_t offsets, mops_tensor_1d_i32_t order, int32_t activation               \
    ) {                                                                                            \
        MOPS_CATCH_EXCEPTIONS_BEGIN                                                                \
        mops::cuda::gated_grouped_product<T>(                                                      \
            view(output), view(A), view(W), view(offsets), view(order), activation                 \
        );                                                                                         \
        MOPS_CATCH_EXCEPTIONS_END                                                                  \
    }                                                                                              \
    extern "C" int mops_amd_gated_grouped_product_vjp_##S(                                         \
        mops_tensor_2d_##S##_t grad_A, mops_tensor_3d_##S##_t grad_W,                              \
        mops_tensor_2d_##S##_t grad_output, mops_tensor_2d_##S##_t A, mops_tensor_3d_##S##_t W,    \
        mops_tensor_1d_i32_t offsets, mops_tensor_1d_i32_t order, int32_t activation               \
    ) {                                                                                            \
        MOPS_CATCH_EXCEPTIONS_BEGIN                                                                \
        mops::cuda::gated_grouped_product_vjp<T>(                                                  \
            view(grad_A), view(grad_W), view(grad_output), view(A), view(W), view(offsets),        \
            view(order), activation                                                                \
        );                                                                                         \
        MOPS_CATCH_EXCEPTIONS_END                                                                  \
    }                                                                                              \
    extern "C" int mops_amd_linear_cross_entropy_##S(                                              \
        mops_tensor_1d_##R##_t losses, mops_tensor_1d_##R##_t log_sums, mops_tensor_2d_##S##_t A,  \
        mops_tensor_2d_##S##_t W, mops_tensor_1d_i32_t targets                                     \
    ) {                                                                                            \
        MOPS_CATCH_EXCEPTIONS_BEGIN                                                                \
        mops::cuda::linear_cross_entropy<T, SUM>(                                                  \
            view(losses), view(log_sums), view(A), view(W), view(targets)                          \
        );                                                                                         \
        MOPS_CATCH_EXCEPTIONS_END                                                                  \
    }                                                                                              \
    extern "C" int mops_amd_linear_cross_entropy_vjp_##S(                                          \
        mops_tensor_2d_##S##_t grad_A, mops_tensor_2d_##S##_t grad_W,                              \
        mops_tensor_1d_##R##_t grad_losses, mops_tensor_1d_##R##_t grad_log_sums,                  \
        mops_tensor_2d_##S##_t A, mops_tensor_2d_##S##_t W, mops_tensor_1d_i32_t targets,          \
        mops_tensor_1d_##R##_t log_sums                                                            \
    ) {                                                                                            \
        MOPS_CATCH_EXCEPTIONS_BEGIN                                                                \
        mops::cuda::linear_cross_entropy_vjp<T, SUM>(                                              \
            view(grad_A), view(grad_W), view(grad_losses), view(grad_log_sums), view(A), view(W),  \
            view(targets), view(log_sums)                                                          \
        );                                                                                         \
        MOPS_CATCH_EXCEPTIONS_END                                                                  \
    }                                                                                              \
    extern "C" int mops_amd_gated_residual_norm_##S(                                               \
        mops_tensor_2d_##S##_t state, mops_tensor_2d_##S##_t next,                                 \
        mops_tensor_2d_##S##_t residual, mops_tensor_2d_##S##_t block,                             \
        mops_tensor_2d_##S##_t gate, mops_tensor_1d_##S##_t weight_block,                          \
        mops_tensor_1d_##S##_t weight_next, double residual_scale, double epsilon                  \
    ) {                                                                                            \
        MOPS_CATCH_EXCEPTIONS_BEGIN                                                                \
        mops::cuda::gated_residual_norm<T>(                                                        \
            view(state), view(next), view(residual), view(block), view(gate), view(weight_block),  \
            view(weight_next), residual_scale, epsilon                                             \
        );                                                                                         \
        MOPS_CATCH_EXCEPTIONS_END                                                                  \
    }                                                                                              \
    extern "C" int mops_amd_gated_residual_norm_vjp_##S(                                           \
        mops_tensor_2d_##S##_t grad_residual, mops_tensor_2d_##S##_t grad_block,                   \
        mops_tensor_2d_##S##_t grad_gate, mops_tensor_1d_##S##_t grad_weight_block,                \
        mops_tensor_1d_##S##_t grad_weight_next, mops_tensor_2d_##S##_t grad_state,                \
        mops_tensor_2d_##S##_t grad_next, mops_tensor_2d_##S##_t residual,                         \
        mops_tensor_2d_##S##_t block, mops_tensor_2d_##S##_t gate,                                 \
        mops_tensor_1d_##S##_t weight_block, mops_tensor_1d_##S##_t weight_next,                   \
        double residual_scale, double epsilon                                                      \
    ) {                                                                                            \
        MOPS_CATCH_EXCEPTIONS_BEGIN                                                                \
        mops::cuda::gated_residual_norm_vjp<T>(                                                    \
            view(grad_residual), view(grad_block), view(grad_gate), view(grad_weight_block),       \
            view(grad_weight_next), view(grad_state), view(grad_next), view(residual), view(block), \
            view(gate), view(weight_block), view(weight_next), residual_scale, epsilon             \
        );                                                                                         \
        MOPS_CATCH_EXCEPTIONS_END                                                                  \
    }

MOPS_LAYERS_DEFINE(f32, float, f32, float)
MOPS_LAYERS_DEFINE(f64, double, f64, double)
MOPS_LAYERS_DEFINE(bf16, mops::bfloat16, f32, float)
MOPS_LAYERS_DEFINE(f16, mops::float16, f32, float)
