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

/// Rows that follow each other, in memory of the caller.
template <typename T> struct Matrices {
    const T* data;
    size_t n_rows;
    int32_t width;

    /// They all begin on 16-byte boundaries.
    bool in_place() const {
        return reinterpret_cast<uintptr_t>(data) % 16 == 0 && static_cast<size_t>(width) * sizeof(T) % 16 == 0;
    }
    int32_t pieces() const { return static_cast<int32_t>(ceil_div(static_cast<size_t>(width), PIECE<T>)); }
    size_t copied_bytes() const { return in_place() ? 0 : align256(n_rows * pieces() * 16); }
};

/// Whether rows that begin anywhere are copied to rows that begin on 16-byte boundaries before they are multiplied.
/// Memory that is read at odd addresses costs the caches twice the time, and tiles that take it through registers are
/// half as fast as those that do not: what a number of operations gains against what the copy costs, at rates measured
/// on either side. As they are / copied, us, where the rule copies: 8192 rows, one group, K = L = 2047, the product: float16
/// 158 / 91, float 642 / 579, double 1195 / 1129; K = L = 1023: 43 / 39, 170 / 162, 318 / 298; 37102 rows, 25 groups,
/// K = 3196, L = 533, float16, gradients: 752 / 585. Where it does not: K = L = 511: float16 20 / 22, float 58 / 56; 255:
/// 10 / 14, 20 / 24, double 32 / 38; 60 000 rows of 4 groups, 65 x 63: 10 / 22, 17 / 30, 28 / 39; 50 595 rows, K = 15,
/// L = 1817: 84 / 95, 149 / 156. It looks at sums of operations and bytes only, and costs time where the copied form's
/// tiles fit worse: gradients of the rows in float and double (8192 x 1023 squared 138 / 160, 262 / 295; 30 000 rows of
/// 8 groups, 401 x 601 double 264 / 374), the product of 60 000 rows of 20 groups, 101 x 1001 float16 (70 / 81).
template <typename T> bool worth_copying(const Matrices<T>& q, const Matrices<T>& p, double operations) {
    constexpr double GAIN = sizeof(T) == 2 ? 1.0 / 700 : sizeof(T) == 4 ? 1.0 / 550 : 1.0 / 150; // us per 10^6
    const double bytes = static_cast<double>(q.copied_bytes() + p.copied_bytes());
    const int launches = !q.in_place() + !p.in_place();
    constexpr double MOST = double(size_t(1) << 31); // (memory that the thread keeps)
    return launches > 0 && bytes <= MOST && operations * 1e-6 * GAIN > bytes / 2.5e6 + 4 * launches;
}

/// `matrices` where they are, or their copy in `room` (which moves on).
template <typename T> Operand<T> place(const Matrices<T>& matrices, char*& room, hipStream_t stream) {
    if (room == nullptr || matrices.in_place()) {
        return Operand<T>{matrices.data, matrices.width};
    }
    T* const to = reinterpret_cast<T*>(room);
    room += matrices.copied_bytes();
    copy_rows_kernel<T><<<static_cast<unsigned>(ceil_div(matrices.n_rows, COPY_ROWS)), COPY_THREADS, 0, stream>>>(
        to, matrices.data, matrices.n_rows, matrices.width, matrices.pieces()
    );
    MOPS_HIP_CHECK(hipGetLastError());
    return Operand<T>{to, matrices.pieces() * PIECE<T>};
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
/// types with aligned rows (through registers they leave none for the pieces that are on their way, nor do tiles of 128 in
/// double: 43 221 rows, K = 235, L = 95: 69 us in tiles of 64, 121 in tiles of 128, which spill).
template <typename T, typename Body> void with_tile(int tile, bool in_place, Body&& body) {
    std::integral_constant<int, 2> two;
    std::integral_constant<int, 4> four;
    if (tile == 256) {
        if constexpr (sizeof(T) == 2) {
            body(std::integral_constant<int, 256>{}, two, four, std::true_type{});
        }
    } else if (tile == 128) {
        if (in_place) {
            body(std::integral_constant<int, 128>{}, two, two, std::true_type{});
        } else if constexpr (sizeof(T) < 8) {
            body(std::integral_constant<int, 128>{}, two, two, std::false_type{});
        }
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
    with_tile<T>(tile, g.in_place, [&](auto size, auto m, auto n, auto in_place) {
        constexpr int TILE = decltype(size)::value, WM = decltype(m)::value, WN = decltype(n)::value;
        constexpr bool ALIGNED = decltype(in_place)::value;
        tiles_kernel<T, FORM, TILE, TILE, WM, WN, DEEP, STAGES_OF<TILE, ALIGNED>, ALIGNED>
            <<<workgroups, WM * WN * WAVE, 0, stream>>>(g);
    });
    MOPS_HIP_CHECK(hipGetLastError());
}

/// Whether what tiles of this extent compute beside the result costs less than smaller tiles, which read more: per number
/// of a tile, 128 take 1.2 times as long as 256, and 64 more than 1.5 times as long as 128. (61709 rows of 30 groups,
/// K = 2176, L = 320, float16: 135 us in tiles of 128, 162 in tiles of 256; L = 536: 184 and 175; 60000 rows, L = 40, float:
/// 81 us in tiles of 64, 140 in tiles of 128.)
bool filled(int tile, int32_t m, int32_t n = 0) {
    auto covered = [&](int extent) {
        return static_cast<double>(tiles(m, extent)) * extent * (n > 0 ? static_cast<double>(tiles(n, extent)) * extent : 1);
    };
    return covered(tile) <= (tile == 256 ? 1.3 : 1.5) * covered(tile / 2);
}

/// Whether there are tiles of this extent (with_tile).
template <typename T> bool exists(int tile, bool in_place) {
    return tile == 256 ? sizeof(T) == 2 && in_place : sizeof(T) < 8 || in_place;
}

/// The tiles of FORWARD and GRAD_ROWS: the largest that keep all compute units busy and, on average, are half full.
template <typename T> int tile_of_rows(const Product<T>& g) {
    const size_t rows = static_cast<size_t>(g.groups.n_rows), groups = static_cast<size_t>(g.groups.n_groups);
    const size_t units = static_cast<size_t>(compute_units());
    auto fits = [&](int tile) {
        return exists<T>(tile, g.in_place) && ceil_div(rows, tile) * tiles(g.n_size, tile) >= units &&
               rows >= tile / 2 * groups && filled(tile, g.n_size);
    };
    return fits(256) ? 256 : fits(128) ? 128 : 64;
}

/// The tiles of GRAD_SUMS, and its rows per unit: what every workgroup that the GPU has room for would have if the work
/// were shared out evenly. Larger groups than that are split (UnitsOfGroups), smaller ones are not.
template <typename T> int tile_of_sums(Product<T>& g) {
    const size_t rows = static_cast<size_t>(std::max(g.groups.n_rows, 1)), groups = static_cast<size_t>(g.groups.n_groups);
    const size_t units = static_cast<size_t>(compute_units());
    auto of_unit = [&](int tile) { return static_cast<size_t>(tiles(g.m_size, tile)) * tiles(g.n_size, tile); };
    auto fits = [&](int tile) {
        return exists<T>(tile, g.in_place) && g.m_size > tile / 2 && g.n_size > tile / 2 &&
               filled(tile, g.m_size, g.n_size) &&
               of_unit(tile) * std::max(groups, ceil_div(rows, 8 * tile)) >= units;
    };
    const int tile = fits(256) ? 256 : fits(128) ? 128 : 64;
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

/// Either may be without an `out`: not wanted.
template <typename T>
void gradients(
    Product<T> sums, Product<T> rows, const Matrices<T>& grad_output, const Matrices<T>& A, const Matrices<T>& W,
    hipStream_t stream
) {
    const bool of_A = rows.out != nullptr, of_W = sums.out != nullptr;
    // (each as if it were wanted alone: its result does not depend on whether the other one is)
    const double operations = 2.0 * A.n_rows * A.width * W.width;
    bool copies_W = false, copies_A = false;
    int of_sums = 0, of_rows = 0;
    size_t copies = 0, row_bytes = 0, sum_bytes = 0;
    auto choose = [&](bool copied) {
        copies_W = copied && of_A && worth_copying(grad_output, W, operations);
        copies_A = copied && of_W && worth_copying(A, grad_output, operations);
        copies = (copies_A ? A.copied_bytes() : 0) + (copies_W ? W.copied_bytes() : 0) +
                 (copies_A || copies_W ? grad_output.copied_bytes() : 0);
        sums.in_place = copies_A || (grad_output.in_place() && A.in_place());
        rows.in_place = copies_W || (grad_output.in_place() && W.in_place());
        if (of_W) {
            of_sums = tile_of_sums(sums);
            sums.most_slots = most_split_units(sums.groups.n_rows, sums.step);
            // (few, and of no more numbers than the tiles that the GPU has room for: 80 MB at most)
            sum_bytes = sums.most_slots * partial_size(sums.m_size, sums.n_size) * sizeof(wide_t<T>);
        }
        if (of_A) {
            of_rows = tile_of_rows(rows);
            share_k(rows, of_rows);
            row_bytes = split_bytes(rows);
        }
    };
    choose(true);
    char* workspace = nullptr;
    if (copies > 0) {
        workspace = static_cast<char*>(scratch_or_null(copies + row_bytes + sum_bytes));
        if (workspace == nullptr) {
            choose(false);
        }
    }
    char* room = nullptr;
    if (copies + row_bytes + sum_bytes > 0) {
        workspace = workspace != nullptr ? workspace : static_cast<char*>(scratch(row_bytes + sum_bytes));
        rows.partial = reinterpret_cast<wide_t<T>*>(workspace + copies);
        sums.partial = reinterpret_cast<wide_t<T>*>(workspace + copies + row_bytes);
        room = copies > 0 ? workspace : nullptr;
    }
    char* none = nullptr;
    const Operand<T> copied = place(grad_output, room, stream);
    const Operand<T> original = place(grad_output, none, stream);
    sums.p = copies_A ? copied : original;
    rows.q = copies_W ? copied : original;
    sums.q = place(A, copies_A ? room : none, stream);
    rows.p = place(W, copies_W ? room : none, stream);
    if (of_sums == of_rows && sums.in_place == rows.in_place) {
        const unsigned for_sums = set_tiles<Form::GRAD_SUMS>(sums, of_sums);
        const unsigned for_rows = set_tiles<Form::GRAD_ROWS>(rows, of_rows);
        with_tile<T>(of_sums, sums.in_place, [&](auto size, auto m, auto n, auto is_aligned) {
            constexpr int TILE = decltype(size)::value, WM = decltype(m)::value, WN = decltype(n)::value;
            constexpr bool ALIGNED = decltype(is_aligned)::value;
            gradients_kernel<T, TILE, TILE, WM, WN, DEEP, STAGES_OF<TILE, ALIGNED>, ALIGNED>
                <<<for_sums + for_rows, WM * WN * WAVE, 0, stream>>>(sums, rows, for_sums);
        });
        MOPS_HIP_CHECK(hipGetLastError());
    } else {
        if (of_W) {
            launch<T, Form::GRAD_SUMS>(sums, of_sums, stream);
        }
        if (of_A) {
            launch<T, Form::GRAD_ROWS>(rows, of_rows, stream);
        }
    }
    if (of_A) {
        join_splits(rows, stream);
    }
    if (sums.most_slots > 0) {
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
        grouped_product::gradients(
            sums, rows, grouped_product::Matrices<T>{data_of(grad_output), A.shape[0], L},
            grouped_product::Matrices<T>{data_of(A), A.shape[0], K},
            grouped_product::Matrices<T>{data_of(W), W.shape[0] * W.shape[1], L}, current_stream()
        );
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
