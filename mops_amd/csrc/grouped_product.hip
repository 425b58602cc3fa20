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
#include "group_checks.hpp"
#include "group_units.hpp"
#include "grouped_launch.hpp"
#include "grouped_tiles.hpp"
#include "numbers.hpp"
#include "runtime.hpp"

namespace mops::amd {
namespace grouped_product {
namespace {

template <typename T> void forward(Product<T> g, const Matrices<T>& A, const Matrices<T>& W, hipStream_t stream) {
    size_t copies = 0;
    int tile = 0;
    auto choose = [&](bool copied) {
        copies = copied ? A.copied_bytes() + W.copied_bytes() : 0;
        g.in_place = copied || (A.in_place() && W.in_place());
        tile = tile_of_rows(g);
        share_k(g, tile);
    };
    choose(worth_copying(A, W, 2.0 * A.n_rows * g.k_size * g.n_size));
    char* workspace = nullptr;
    if (copies > 0) {
        workspace = static_cast<char*>(scratch_or_null(copies + split_bytes(g)));
        if (workspace == nullptr) {
            choose(false);
        }
    }
    char* room = nullptr;
    if (copies + split_bytes(g) > 0) {
        workspace = workspace != nullptr ? workspace : static_cast<char*>(scratch(split_bytes(g)));
        g.partial = reinterpret_cast<wide_t<T>*>(workspace + copies);
        room = copies > 0 ? workspace : nullptr;
    }
    g.q = place(A, room, stream);
    g.p = place(W, room, stream);
    launch<T, Form::FORWARD>(g, tile, stream);
    join_splits(g, stream);
}

} // namespace

template <typename T>
Gradients<T>::Gradients(
    const Product<T>& sums, const Product<T>& rows, const Matrices<T>& grad_output, const Matrices<T>& A,
    const Matrices<T>& W
)
    : sums_(sums), rows_(rows), grad_output_(grad_output), A_(A), W_(W) {
    choose(true);
}

template <typename T> void Gradients<T>::choose(bool copied) {
    const bool of_A = rows_.out != nullptr, of_W = sums_.out != nullptr;
    // (each as if it were wanted alone: its result does not depend on whether the other one is)
    const double operations = 2.0 * A_.n_rows * A_.width * W_.width;
    copies_W_ = copied && of_A && worth_copying(grad_output_, W_, operations);
    copies_A_ = copied && of_W && worth_copying(A_, grad_output_, operations);
    copies_ = (copies_A_ ? A_.copied_bytes() : 0) + (copies_W_ ? W_.copied_bytes() : 0) +
              (copies_A_ || copies_W_ ? grad_output_.copied_bytes() : 0);
    sums_.in_place = copies_A_ || (grad_output_.in_place() && A_.in_place());
    rows_.in_place = copies_W_ || (grad_output_.in_place() && W_.in_place());
    if (of_W) {
        of_sums_ = tile_of_sums(sums_);
        sums_.most_slots = most_split_units(sums_.groups.n_rows, sums_.step);
        // (few, and of no more numbers than the tiles that the GPU has room for: 80 MB at most)
        sum_bytes_ = sums_.most_slots * partial_size(sums_.m_size, sums_.n_size) * sizeof(wide_t<T>);
    }
    if (of_A) {
        of_rows_ = tile_of_rows(rows_);
        share_k(rows_, of_rows_);
        row_bytes_ = split_bytes(rows_);
    }
}

template <typename T> void Gradients<T>::run(char* workspace, hipStream_t stream) {
    Product<T> sums = sums_, rows = rows_;
    rows.partial = reinterpret_cast<wide_t<T>*>(workspace + copies_);
    sums.partial = reinterpret_cast<wide_t<T>*>(workspace + copies_ + row_bytes_);
    char *room = copies_ > 0 ? workspace : nullptr, *none = nullptr;
    const Operand<T> copied = place(grad_output_, room, stream);
    const Operand<T> original = place(grad_output_, none, stream);
    sums.p = copies_A_ ? copied : original;
    rows.q = copies_W_ ? copied : original;
    sums.q = place(A_, copies_A_ ? room : none, stream);
    rows.p = place(W_, copies_W_ ? room : none, stream);
    if (of_sums_ == of_rows_ && sums.in_place == rows.in_place) {
        const unsigned for_sums = set_tiles<Form::GRAD_SUMS>(sums, of_sums_);
        const unsigned for_rows = set_tiles<Form::GRAD_ROWS>(rows, of_rows_);
        with_tile<T>(of_sums_, sums.in_place, [&](auto size, auto m, auto n, auto is_aligned) {
            constexpr int TILE = decltype(size)::value, WM = decltype(m)::value, WN = decltype(n)::value;
            constexpr bool ALIGNED = decltype(is_aligned)::value;
            gradients_kernel<T, TILE, TILE, WM, WN, DEEP, STAGES_OF<TILE, ALIGNED>, ALIGNED>
                <<<for_sums + for_rows, WM * WN * WAVE, 0, stream>>>(sums, rows, for_sums, {}, {});
        });
        MOPS_HIP_CHECK(hipGetLastError());
    } else {
        if (sums.out != nullptr) {
            launch<T, Form::GRAD_SUMS>(sums, of_sums_, stream);
        }
        if (rows.out != nullptr) {
            launch<T, Form::GRAD_ROWS>(rows, of_rows_, stream);
        }
    }
    if (rows.out != nullptr) {
        join_splits(rows, stream);
    }
    if (sums.most_slots > 0) {
        const unsigned workgroups = 4 * static_cast<unsigned>(compute_units());
        join_units_kernel<T><<<workgroups, JOIN_WAVES * WAVE, 0, stream>>>(sums);
        MOPS_HIP_CHECK(hipGetLastError());
    }
}

template class Gradients<float>;
template class Gradients<double>;
template class Gradients<__bf16>;
template class Gradients<_Float16>;

} // namespace grouped_product
} // namespace mops::amd

namespace mops::cuda {

using namespace mops::amd;

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
        g.groups = groups;
        g.n_size = L;
        g.k_size = K;
        const grouped_product::Matrices<T> rows{data_of(A), A.shape[0], K};
        const grouped_product::Matrices<T> matrices{data_of(W), W.shape[0] * W.shape[1], L};
        grouped_product::forward(g, rows, matrices, current_stream());
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
    grouped_product::Product<T> sums{}, rows{};
    if (grad_W.data != nullptr && groups.n_groups > 0 && K > 0 && L > 0) {
        sums.out = data_of(grad_W);
        sums.groups = groups;
        sums.m_size = K;
        sums.n_size = L;
    }
    if (grad_A.data != nullptr && groups.n_rows > 0 && K > 0) {
        rows.out = data_of(grad_A);
        rows.groups = groups;
        rows.n_size = K;
        rows.k_size = L;
    }
    if (sums.out != nullptr || rows.out != nullptr) {
        grouped_product::Gradients<T> gradients(
            sums, rows, grouped_product::Matrices<T>{data_of(grad_output), A.shape[0], L},
            grouped_product::Matrices<T>{data_of(A), A.shape[0], K},
            grouped_product::Matrices<T>{data_of(W), W.shape[0] * W.shape[1], L}
        );
        void* workspace = gradients.copies() ? scratch_or_null(gradients.bytes()) : nullptr;
        if (workspace == nullptr) {
            gradients.do_without_copies();
            workspace = gradients.bytes() > 0 ? scratch(gradients.bytes()) : nullptr;
        }
        gradients.run(static_cast<char*>(workspace), current_stream());
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
