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
template <typename T, Form FORM> bool aligned(const Product<T>& g) {
    return aligned(g.q, FORM == Form::GRAD_SUMS ? g.m_size : g.k_size) &&
           aligned(g.p, FORM == Form::GRAD_ROWS ? g.k_size : g.n_size);
}

/// The extents of a call's tiles: TILE x TILE numbers.
template <Form FORM, typename T> unsigned set_tiles(Product<T>& g, int tile) {
    g.m_tiles = FORM == Form::GRAD_SUMS ? static_cast<int32_t>(tiles(g.m_size, tile)) : 1;
    g.n_tiles = static_cast<int32_t>(tiles(g.n_size, tile));
    if (FORM != Form::GRAD_SUMS) {
        g.step = tile;
    }
    g.most_units = narrow_i32(most_units(g.groups.n_rows, g.groups.n_groups, g.step), "number of units of rows");
    const size_t of_unit = static_cast<size_t>(g.m_tiles) * g.n_tiles * std::max(g.splits, 1);
    const size_t workgroups = ceil_div(g.most_units * of_unit, 8) * 8;
    return static_cast<unsigned>(narrow_i32(workgroups, "number of tiles"));
}

/// body(tile, wavefronts of its rows, of its columns, rows aligned): the kernels there are. Tiles of 256 are for 16-bit
/// types with aligned rows (through registers they leave none for the pieces that are on their way).
template <typename T, typename Body> void with_tile(int tile, bool in_place, Body&& body) {
    std::integral_constant<int, 2> two;
    std::integral_constant<int, 4> four;
    if (tile == 256) {
        if constexpr (sizeof(T) == 2) {
            body(std::integral_constant<int, 256>{}, two, four, std::true_type{});
        }
    } else if (tile == 128) {
        in_place ? body(std::integral_constant<int, 128>{}, two, two, std::true_type{})
                 : body(std::integral_constant<int, 128>{}, two, two, std::false_type{});
    } else {
        in_place ? body(std::integral_constant<int, 64>{}, two, two, std::true_type{})
                 : body(std::integral_constant<int, 64>{}, two, two, std::false_type{});
    }
}
constexpr int DEEP = 8;
// Steps in LDS or on their way there. Small tiles have little to compute per step and more need to be on their way (24 rows,
// 16 groups, K = 2048, L = 1408, bfloat16: 22.2 us with two, 15.8 with three, 17.0 with four); the others fill LDS with two.
template <int TILE, bool ALIGNED> constexpr int STAGES_OF = TILE == 64 && ALIGNED ? 3 : 2;

template <typename T, Form FORM> void launch(Product<T> g, int tile, hipStream_t stream) {
    const unsigned workgroups = set_tiles<FORM>(g, tile);
    with_tile<T>(tile, aligned<T, FORM>(g), [&](auto size, auto m, auto n, auto in_place) {
        constexpr int TILE = decltype(size)::value, WM = decltype(m)::value, WN = decltype(n)::value;
        constexpr bool ALIGNED = decltype(in_place)::value;
        tiles_kernel<T, FORM, TILE, TILE, WM, WN, DEEP, STAGES_OF<TILE, ALIGNED>, ALIGNED><<<workgroups, WM * WN * WAVE, 0, stream>>>(g);
    });
    MOPS_HIP_CHECK(hipGetLastError());
}

/// The tiles of FORWARD and GRAD_ROWS: the largest that keep all compute units busy and, on average, are half full.
template <typename T, Form FORM> int tile_of_rows(const Product<T>& g) {
    const size_t rows = static_cast<size_t>(g.groups.n_rows), groups = static_cast<size_t>(g.groups.n_groups);
    const size_t units = static_cast<size_t>(compute_units());
    auto fits = [&](int tile) {
        return ceil_div(rows, tile) * tiles(g.n_size, tile) >= units && rows >= tile / 2 * groups;
    };
    return sizeof(T) == 2 && aligned<T, FORM>(g) && fits(256) ? 256 : fits(128) ? 128 : 64;
}

/// The tiles of GRAD_SUMS, and its rows per unit: what every workgroup that the GPU has room for would have if the work
/// were shared out evenly. Larger groups than that are split, smaller ones are not.
template <typename T> int tile_of_sums(Product<T>& g) {
    const size_t rows = static_cast<size_t>(std::max(g.groups.n_rows, 1)), groups = static_cast<size_t>(g.groups.n_groups);
    const size_t units = static_cast<size_t>(compute_units());
    auto of_unit = [&](int tile) { return static_cast<size_t>(tiles(g.m_size, tile)) * tiles(g.n_size, tile); };
    auto fits = [&](int tile) {
        return g.m_size > tile / 2 && g.n_size > tile / 2 &&
               of_unit(tile) * std::max(groups, ceil_div(rows, 8 * tile)) >= units;
    };
    const int tile = sizeof(T) == 2 && aligned<T, Form::GRAD_SUMS>(g) && fits(256) ? 256 : fits(128) ? 128 : 64;
    const size_t room = (tile == 256 ? 1 : 2) * units;
    const size_t step = std::max<size_t>(ceil_div(rows * of_unit(tile), room), 256);
    g.step = static_cast<int32_t>(std::min(ceil_div(step, 64) * 64, ceil_div(rows, 64) * 64));
    return tile;
}

/// FORWARD and GRAD_ROWS with few tiles and long sums: every compute unit gets a share of k (250 rows of 19 groups, K = 24,
/// L = 1226 in float, gradients: 20 workgroups, one of 39 steps after the other, are 41 us). At least four steps each.
template <typename T> void share_k(Product<T>& g, int tile) {
    g.splits = 1;
    g.k_each = g.k_size;
    if (tile != 64) {
        return;
    }
    const size_t step = 16 / sizeof(T) * DEEP, steps = ceil_div(static_cast<size_t>(g.k_size), step);
    const size_t rows = static_cast<size_t>(g.groups.n_rows), groups = static_cast<size_t>(g.groups.n_groups);
    const size_t workgroups = std::min(ceil_div(rows, 64) + groups, rows) * tiles(g.n_size, 64);
    const size_t units = static_cast<size_t>(compute_units());
    if (workgroups < units && steps >= 8) {
        const size_t splits = std::min(ceil_div(units, workgroups), steps / 4), each = ceil_div(steps, splits);
        g.splits = static_cast<int32_t>(ceil_div(steps, each));
        g.k_each = static_cast<int32_t>(each * step);
    }
}
template <typename T> size_t split_bytes(const Product<T>& g) {
    return g.splits > 1 ? align256(static_cast<size_t>(g.splits) * g.groups.n_rows * g.n_size * sizeof(wide_t<T>)) : 0;
}
template <typename T> void join_splits(const Product<T>& g, hipStream_t stream) {
    if (g.splits > 1) {
        const size_t blocks = ceil_div(static_cast<size_t>(g.groups.n_rows) * g.n_size, JOIN_THREADS);
        join_splits_kernel<T><<<static_cast<unsigned>(blocks), JOIN_THREADS, 0, stream>>>(g);
        MOPS_HIP_CHECK(hipGetLastError());
    }
}

template <typename T> void forward(Product<T> g, hipStream_t stream) {
    const int tile = tile_of_rows<T, Form::FORWARD>(g);
    share_k(g, tile);
    if (g.splits > 1) {
        g.partial = static_cast<wide_t<T>*>(scratch(split_bytes(g)));
    }
    launch<T, Form::FORWARD>(g, tile, stream);
    join_splits(g, stream);
}

/// Either may be without an `out`: not wanted.
template <typename T> void gradients(Product<T> sums, Product<T> rows, hipStream_t stream) {
    const int of_sums = sums.out != nullptr ? tile_of_sums(sums) : 0;
    const int of_rows = rows.out != nullptr ? tile_of_rows<T, Form::GRAD_ROWS>(rows) : 0;
    const bool splits = of_sums != 0 && sums.step < sums.groups.n_rows;
    if (of_rows != 0) {
        share_k(rows, of_rows);
    }
    const size_t row_bytes = of_rows != 0 ? split_bytes(rows) : 0;
    size_t sum_bytes = 0;
    if (splits) {
        const size_t most = most_units(sums.groups.n_rows, sums.groups.n_groups, sums.step);
        sum_bytes = most * partial_size(sums.m_size, sums.n_size) * sizeof(wide_t<T>);
    }
    if (row_bytes + sum_bytes > 0) {
        char* workspace = static_cast<char*>(scratch(row_bytes + sum_bytes));
        rows.partial = reinterpret_cast<wide_t<T>*>(workspace);
        sums.partial = reinterpret_cast<wide_t<T>*>(workspace + row_bytes);
    }
    const bool in_place = of_sums != 0 && aligned<T, Form::GRAD_SUMS>(sums);
    if (of_sums == of_rows && in_place == aligned<T, Form::GRAD_ROWS>(rows)) {
        const unsigned for_sums = set_tiles<Form::GRAD_SUMS>(sums, of_sums);
        const unsigned for_rows = set_tiles<Form::GRAD_ROWS>(rows, of_rows);
        with_tile<T>(of_sums, in_place, [&](auto size, auto m, auto n, auto is_aligned) {
            constexpr int TILE = decltype(size)::value, WM = decltype(m)::value, WN = decltype(n)::value;
            constexpr bool ALIGNED = decltype(is_aligned)::value;
            gradients_kernel<T, TILE, TILE, WM, WN, DEEP, STAGES_OF<TILE, ALIGNED>, ALIGNED>
                <<<for_sums + for_rows, WM * WN * WAVE, 0, stream>>>(sums, rows, for_sums);
        });
        MOPS_HIP_CHECK(hipGetLastError());
    } else {
        if (of_sums != 0) {
            launch<T, Form::GRAD_SUMS>(sums, of_sums, stream);
        }
        if (of_rows != 0) {
            launch<T, Form::GRAD_ROWS>(rows, of_rows, stream);
        }
    }
    if (of_rows != 0) {
        join_splits(rows, stream);
    }
    if (splits) {
        sums.most_units = narrow_i32(
            most_units(sums.groups.n_rows, sums.groups.n_groups, sums.step), "number of units of rows"
        );
        const unsigned workgroups = 4 * static_cast<unsigned>(compute_units());
        join_units_kernel<T><<<workgroups, JOIN_WAVES * WAVE, 0, stream>>>(sums);
        MOPS_HIP_CHECK(hipGetLastError());
    }
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
        grouped_product::forward(g, current_stream());
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
        sums.q = data_of(A);
        sums.p = data_of(grad_output);
        sums.groups = groups;
        sums.m_size = K;
        sums.n_size = L;
    }
    if (grad_A.data != nullptr && groups.n_rows > 0 && K > 0) {
        rows.out = data_of(grad_A);
        rows.q = data_of(grad_output);
        rows.p = data_of(W);
        rows.groups = groups;
        rows.n_size = K;
        rows.k_size = L;
    }
    if (sums.out != nullptr || rows.out != nullptr) {
        grouped_product::gradients(sums, rows, current_stream());
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
