// Every row times the matrix of its group, and the gradients:
//
//   output[r, :]    = A[r, :] W[g, :, :]                 for the rows r of group g
//   grad_A[r, :]    = grad_output[r, :] W[g, :, :]^T
//   grad_W[g, :, :] = sum over the rows r of group g of A[r, :]^T grad_output[r, :]
//
// The sizes of the groups are known to the device only, so the grid has as many
// workgroups as there can be tiles of rows (most_units), and each finds out from
// the offsets which rows it has (find_unit).
#include "mops/layers.hpp"

#include <algorithm>

#include "checks.hpp"
#include "device_common.hpp"
#include "group_units.hpp"
#include "grouped_tiles.hpp"
#include "numbers.hpp"
#include "runtime.hpp"

namespace mops::amd {
namespace grouped_product {
namespace {

unsigned tiles(int32_t size, int tile) { return static_cast<unsigned>(ceil_div(static_cast<size_t>(size), tile)); }

/// Rows of `width` numbers that all begin on 16-byte boundaries.
template <typename T> bool aligned(const T* data, int32_t width) {
    return reinterpret_cast<uintptr_t>(data) % 16 == 0 && static_cast<size_t>(width) * sizeof(T) % 16 == 0;
}
template <typename T, Form FORM> int32_t q_width(const Product<T>& g) {
    return FORM == Form::GRAD_SUMS ? g.m_size : g.k_size;
}
template <typename T, Form FORM> int32_t p_width(const Product<T>& g) {
    return FORM == Form::GRAD_ROWS ? g.k_size : g.n_size;
}

template <typename T, Form FORM, int BM, int BN, int WM, int WN, int DEEP = 8, int STAGES = 2> void launch(Product<T> g, hipStream_t stream) {
    constexpr bool SUMS = FORM == Form::GRAD_SUMS;
    g.m_tiles = SUMS ? static_cast<int32_t>(tiles(g.m_size, BM)) : 1;
    g.n_tiles = static_cast<int32_t>(tiles(g.n_size, BN));
    if (!SUMS) {
        g.step = BM;
    }
    g.most_units = narrow_i32(most_units(g.groups.n_rows, g.groups.n_groups, g.step), "number of units of rows");
    const size_t workgroups = ceil_div(static_cast<size_t>(g.most_units) * g.m_tiles * g.n_tiles, 8) * 8;
    const unsigned blocks = static_cast<unsigned>(narrow_i32(workgroups, "number of tiles"));
    if (BM == 256 || (aligned(g.q, q_width<T, FORM>(g)) && aligned(g.p, p_width<T, FORM>(g)))) {
        tiles_kernel<T, FORM, BM, BN, WM, WN, DEEP, STAGES, true><<<blocks, WM * WN * WAVE, 0, stream>>>(g);
    } else if constexpr (BM < 256) {
        tiles_kernel<T, FORM, BM, BN, WM, WN, 8, 2, false><<<blocks, WM * WN * WAVE, 0, stream>>>(g);
    }
}

template <typename T, Form FORM> void rows_times(const Product<T>& g, hipStream_t stream) {
    const size_t rows = static_cast<size_t>(g.groups.n_rows);
    const size_t big = ceil_div(rows, 256) * tiles(g.n_size, 256), middle = ceil_div(rows, 128) * tiles(g.n_size, 128);
    const size_t units = static_cast<size_t>(compute_units());
    // (through registers the tiles of 256 leave none for the pieces that are on their way)
    const bool in_place = aligned(g.q, q_width<T, FORM>(g)) && aligned(g.p, p_width<T, FORM>(g));
    if (sizeof(T) == 2 && in_place && big >= units && rows >= 128 * static_cast<size_t>(g.groups.n_groups)) {
        if constexpr (sizeof(T) == 2) {
            launch<T, FORM, 256, 256, 2, 4, 8, 2>(g, stream);
        }
    } else if (middle >= units && rows >= 64 * static_cast<size_t>(g.groups.n_groups)) {
        launch<T, FORM, 128, 128, 2, 2>(g, stream);
    } else {
        launch<T, FORM, 64, 64, 2, 2>(g, stream);
    }
    MOPS_HIP_CHECK(hipGetLastError());
}

template <typename T> void sum_of_rows(Product<T> g, hipStream_t stream) {
    const size_t units = static_cast<size_t>(compute_units()), groups = static_cast<size_t>(g.groups.n_groups);
    const size_t rows = static_cast<size_t>(std::max(g.groups.n_rows, 1));
    const size_t big = static_cast<size_t>(tiles(g.m_size, 256)) * tiles(g.n_size, 256);
    const size_t middle = static_cast<size_t>(tiles(g.m_size, 128)) * tiles(g.n_size, 128);
    // (big tiles: one workgroup per compute unit, in groups that can be split if there are too few of them)
    const bool use_big = sizeof(T) == 2 && aligned(g.q, g.m_size) && aligned(g.p, g.n_size) && g.m_size >= 256 && g.n_size >= 256 &&
                         big * std::max(groups, ceil_div(rows, 2048)) >= units;
    const bool use_middle = g.m_size > 64 && g.n_size > 64;
    const size_t tiles_of_unit =
        use_big ? big : use_middle ? middle : static_cast<size_t>(tiles(g.m_size, 64)) * tiles(g.n_size, 64);
    // Rows per unit: what every workgroup that the GPU has room for would have if the work were shared out evenly. Larger
    // groups than that are split, smaller ones are not.
    const size_t room = (use_big ? 1 : 2) * units;
    size_t step = std::max<size_t>(ceil_div(rows * tiles_of_unit, room), 256);
    step = std::min(ceil_div(step, 64) * 64, ceil_div(rows, 64) * 64);
    g.step = static_cast<int32_t>(step);
    const bool splits = step < rows;
    const size_t most = most_units(g.groups.n_rows, g.groups.n_groups, g.step);
    if (splits) {
        g.partial = static_cast<wide_t<T>*>(scratch(most * partial_size(g.m_size, g.n_size) * sizeof(wide_t<T>)));
    }
    if (use_big) {
        if constexpr (sizeof(T) == 2) {
            launch<T, Form::GRAD_SUMS, 256, 256, 2, 4, 8, 2>(g, stream);
        }
    } else if (use_middle) {
        launch<T, Form::GRAD_SUMS, 128, 128, 2, 2>(g, stream);
    } else {
        launch<T, Form::GRAD_SUMS, 64, 64, 2, 2>(g, stream);
    }
    if (splits) {
        g.most_units = narrow_i32(most, "number of units of rows");
        join_units_kernel<T><<<static_cast<unsigned>(4 * units), JOIN_WAVES * WAVE, 0, stream>>>(g);
    }
    MOPS_HIP_CHECK(hipGetLastError());
}

} // namespace
} // namespace grouped_product
} // namespace mops::amd

namespace mops::cuda {

using namespace mops::amd;

namespace {

template <typename scalar_t>
RowGroups check_groups(
    const checks::Validator& check, Tensor<scalar_t, 2> A, Tensor<scalar_t, 3> W, Tensor<int32_t, 1> offsets,
    Tensor<int32_t, 1> order
) {
    using checks::axis_of;
    check.same_extent(axis_of(A, "A", 1), axis_of(W, "W", 1));
    if (offsets.shape[0] != W.shape[0] + 1) {
        throw std::runtime_error(
            "offsets must have " + std::to_string(W.shape[0] + 1) + " elements (the groups of W and one more) in " +
            check.operation() + ", got " + std::to_string(offsets.shape[0])
        );
    }
    if (order.data != nullptr) {
        check.same_extent(axis_of(order, "order", 0), axis_of(A, "A", 0));
    }
    return RowGroups{
        offsets.data, order.data, count_i32(W.shape[0], "number of groups"), count_i32(A.shape[0], "number of rows")
    };
}

} // namespace

template <typename scalar_t>
void grouped_matrix_product(
    Tensor<scalar_t, 2> output, Tensor<scalar_t, 2> A, Tensor<scalar_t, 3> W, Tensor<int32_t, 1> offsets,
    Tensor<int32_t, 1> order
) {
    const checks::Validator check("grouped_matrix_product");
    const RowGroups groups = check_groups(check, A, W, offsets, order);
    check.same_extent(checks::axis_of(output, "output", 0), checks::axis_of(A, "A", 0));
    check.same_extent(checks::axis_of(output, "output", 1), checks::axis_of(W, "W", 2));
    const int32_t K = count_i32(W.shape[1], "W.shape[1]"), L = count_i32(W.shape[2], "W.shape[2]");
    if (groups.n_rows > 0 && L > 0) {
        typedef device_t<scalar_t> T;
        grouped_product::Product<T> g{};
        g.out = data_of(output);
        g.q = data_of(A);
        g.p = data_of(W);
        g.groups = groups;
        g.n_size = L;
        g.k_size = K;
        grouped_product::rows_times<T, grouped_product::Form::FORWARD>(g, current_stream());
    }
    finish_call("grouped_matrix_product");
}

template <typename scalar_t>
void grouped_matrix_product_vjp(
    Tensor<scalar_t, 2> grad_A, Tensor<scalar_t, 3> grad_W, Tensor<scalar_t, 2> grad_output, Tensor<scalar_t, 2> A,
    Tensor<scalar_t, 3> W, Tensor<int32_t, 1> offsets, Tensor<int32_t, 1> order
) {
    using checks::axis_of;
    const checks::Validator check("grouped_matrix_product_vjp");
    const RowGroups groups = check_groups(check, A, W, offsets, order);
    check.same_extent(axis_of(grad_output, "grad_output", 0), axis_of(A, "A", 0));
    check.same_extent(axis_of(grad_output, "grad_output", 1), axis_of(W, "W", 2));
    if (grad_A.data != nullptr) {
        check.same_extent(axis_of(grad_A, "grad_A", 0), axis_of(A, "A", 0));
        check.same_extent(axis_of(grad_A, "grad_A", 1), axis_of(A, "A", 1));
    }
    if (grad_W.data != nullptr) {
        check.same_extent(axis_of(grad_W, "grad_W", 0), axis_of(W, "W", 0));
        check.same_extent(axis_of(grad_W, "grad_W", 1), axis_of(W, "W", 1));
        check.same_extent(axis_of(grad_W, "grad_W", 2), axis_of(W, "W", 2));
    }
    const int32_t K = count_i32(W.shape[1], "W.shape[1]"), L = count_i32(W.shape[2], "W.shape[2]");
    typedef device_t<scalar_t> T;
    if (grad_A.data != nullptr && groups.n_rows > 0 && K > 0) {
        grouped_product::Product<T> g{};
        g.out = data_of(grad_A);
        g.q = data_of(grad_output);
        g.p = data_of(W);
        g.groups = groups;
        g.n_size = K;
        g.k_size = L;
        grouped_product::rows_times<T, grouped_product::Form::GRAD_ROWS>(g, current_stream());
    }
    if (grad_W.data != nullptr && groups.n_groups > 0 && K > 0 && L > 0) {
        grouped_product::Product<T> g{};
        g.out = data_of(grad_W);
        g.q = data_of(A);
        g.p = data_of(grad_output);
        g.groups = groups;
        g.m_size = K;
        g.n_size = L;
        grouped_product::sum_of_rows(g, current_stream());
    }
    finish_call("grouped_matrix_product_vjp");
}

#define MOPS_GROUPED_PRODUCT_INSTANTIATE(T)                                                        \
    template void grouped_matrix_product<T>(                                                       \
        Tensor<T, 2>, Tensor<T, 2>, Tensor<T, 3>, Tensor<int32_t, 1>, Tensor<int32_t, 1>           \
    );                                                                                             \
    template void grouped_matrix_product_vjp<T>(                                                   \
        Tensor<T, 2>, Tensor<T, 3>, Tensor<T, 2>, Tensor<T, 2>, Tensor<T, 3>, Tensor<int32_t, 1>, Tensor<int32_t, 1> \
    );
MOPS_GROUPED_PRODUCT_INSTANTIATE(float)
MOPS_GROUPED_PRODUCT_INSTANTIATE(double)
MOPS_GROUPED_PRODUCT_INSTANTIATE(bfloat16)
MOPS_GROUPED_PRODUCT_INSTANTIATE(float16)

} // namespace mops::cuda
