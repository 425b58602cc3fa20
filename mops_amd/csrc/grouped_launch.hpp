// What the host decides about products over groups of rows (grouped_tiles.hpp):
// copies of operands, extents of tiles, units, shares of k, and the launches.
// Shared by the operators that are made of such products.
#ifndef MOPS_AMD_GROUPED_LAUNCH_HPP
#define MOPS_AMD_GROUPED_LAUNCH_HPP

#include <algorithm>
#include <type_traits>

#include "device_common.hpp"
#include "group_units.hpp"
#include "grouped_tiles.hpp"
#include "numbers.hpp"
#include "runtime.hpp"

namespace mops::amd::grouped_product {

inline unsigned tiles(int32_t size, int tile) { return static_cast<unsigned>(ceil_div(static_cast<size_t>(size), tile)); }

/// Rows that follow each other, in memory of the caller.
template <typename T> struct Matrices {
    const T* data;
    size_t n_rows;
    int32_t width;
    int32_t stride = width; // numbers from a row to the next: the width, or whole pieces with zeros behind the numbers

    /// They all begin on 16-byte boundaries.
    bool in_place() const {
        return reinterpret_cast<uintptr_t>(data) % 16 == 0 && static_cast<size_t>(stride) * sizeof(T) % 16 == 0;
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
        return Operand<T>{matrices.data, matrices.stride};
    }
    T* const to = reinterpret_cast<T*>(room);
    room += matrices.copied_bytes();
    copy_rows_kernel<T><<<static_cast<unsigned>(ceil_div(matrices.n_rows, COPY_ROWS)), COPY_THREADS, 0, stream>>>(
        to, matrices.data, matrices.n_rows, matrices.width, matrices.pieces()
    );
    MOPS_HIP_CHECK(hipGetLastError());
    return Operand<T>{to, matrices.pieces() * PIECE<T>};
}

/// The extents of a call's tiles: TILE x TILE numbers (or `columns` numbers of a row).
template <Form FORM, typename T> unsigned set_tiles(Product<T>& g, int tile, int columns = 0) {
    g.m_tiles = FORM == Form::GRAD_SUMS ? static_cast<int32_t>(tiles(g.m_size, tile)) : 1;
    g.n_tiles = static_cast<int32_t>(tiles(g.n_size, columns > 0 ? columns : tile));
    if (FORM != Form::GRAD_SUMS) {
        g.step = tile;
    }
    g.most_units = narrow_i32(most_units(g.groups.n_rows, g.groups.n_groups, g.step), "number of units of rows");
    const size_t of_unit = static_cast<size_t>(g.m_tiles) * g.n_tiles * std::max(g.splits, 1);
    const size_t tiles_in_all = g.most_units * of_unit;
    const size_t workgroups =
        FORM == Form::GRAD_SUMS ? ceil_div(tiles_in_all, XCDS) * XCDS : workgroups_for(tiles_in_all);
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

/// Tiles of few rows and 128 columns, of rows on 16-byte boundaries, for matrices that are read for few rows: body(rows,
/// wavefronts of the rows, of the columns). Most of LDS holds what is on its way of the matrices, and two workgroups fit a
/// compute unit with three steps (64 rows of 50000 classes, K = 2048, bfloat16: 48.5 us with 64 rows, 53 in square tiles of
/// 128, 59 in those of 64; 24 tokens of 16 experts, 2048 x 2 x 1408: 31.0 us with 32 rows, 33.2 with 64, 41 with 32 rows and
/// 64 columns, 54 with four steps, of which one workgroup fits).
constexpr int WIDE_COLUMNS = 128, WIDE_STAGES = 3;
template <typename T> constexpr int LEAST_ROWS = sizeof(T) < 8 ? 32 : 64; // (double: of 64 only)
template <typename T, typename Body> void with_wide_tile(int rows, Body&& body) {
    std::integral_constant<int, 1> one;
    std::integral_constant<int, 2> two;
    if (rows < 64) {
        if constexpr (LEAST_ROWS<T> < 64) {
            body(std::integral_constant<int, LEAST_ROWS<T>>{}, one, two);
        }
    } else {
        body(std::integral_constant<int, 64>{}, two, two);
    }
}

template <typename T, Form FORM, typename Finish = StoreSums<T, FORM>>
void launch(Product<T> g, int tile, hipStream_t stream, const Finish& finish = {}) {
    const unsigned workgroups = set_tiles<FORM>(g, tile);
    with_tile<T>(tile, g.in_place, [&](auto size, auto m, auto n, auto in_place) {
        constexpr int TILE = decltype(size)::value, WM = decltype(m)::value, WN = decltype(n)::value;
        constexpr bool ALIGNED = decltype(in_place)::value;
        tiles_kernel<T, FORM, TILE, TILE, WM, WN, DEEP, STAGES_OF<TILE, ALIGNED>, ALIGNED, Finish>
            <<<workgroups, WM * WN * WAVE, 0, stream>>>(g, finish);
    });
    MOPS_HIP_CHECK(hipGetLastError());
}
template <typename T, Form FORM, typename Finish>
void launch_wide(Product<T> g, int rows, int columns, hipStream_t stream, const Finish& finish) {
    const unsigned workgroups = set_tiles<FORM>(g, rows, columns);
    with_wide_tile<T>(rows, [&](auto size, auto m, auto n) {
        constexpr int ROWS = decltype(size)::value, WM = decltype(m)::value, WN = decltype(n)::value;
        tiles_kernel<T, FORM, ROWS, WIDE_COLUMNS, WM, WN, DEEP, WIDE_STAGES, true, Finish>
            <<<workgroups, WM * WN * WAVE, 0, stream>>>(g, finish);
    });
    MOPS_HIP_CHECK(hipGetLastError());
}

/// Whether what tiles of this extent compute beside the result costs less than smaller tiles, which read more: per number
/// of a tile, 128 take 1.2 times as long as 256, and 64 more than 1.5 times as long as 128. (61709 rows of 30 groups,
/// K = 2176, L = 320, float16: 135 us in tiles of 128, 162 in tiles of 256; L = 536: 184 and 175; 60000 rows, L = 40, float:
/// 81 us in tiles of 64, 140 in tiles of 128.)
inline bool filled(int tile, int32_t m, int32_t n = 0) {
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
/// L = 1226 in float, gradients: 20 workgroups, one of 39 steps after the other, are 41 us), or `per_unit` of them. At least four steps each.
template <typename T> void share_k(Product<T>& g, int tile, size_t per_unit = 1) {
    g.splits = 1;
    g.k_each = g.k_size;
    if (tile != 64) {
        return;
    }
    const size_t step = 16 / sizeof(T) * DEEP, steps = ceil_div(static_cast<size_t>(g.k_size), step);
    const size_t rows = static_cast<size_t>(g.groups.n_rows), groups = static_cast<size_t>(g.groups.n_groups);
    const size_t workgroups = std::min(ceil_div(rows, 64) + groups, rows) * tiles(g.n_size, 64);
    const size_t units = per_unit * static_cast<size_t>(compute_units());
    if (workgroups > 0 && workgroups < units && steps >= 8) {
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

/// Both gradients of products over groups of rows, in memory of the caller (grouped_product.hip).
template <typename T> class Gradients {
public:
    /// `sums` and `rows` with their results, groups and extents; either may be without an `out`: not wanted.
    Gradients(
        const Product<T>& sums, const Product<T>& rows, const Matrices<T>& grad_output, const Matrices<T>& A,
        const Matrices<T>& W
    );
    /// Bytes of memory that `run` takes; whether it would do with less, without copies of operands.
    size_t bytes() const { return copies_ + row_bytes_ + sum_bytes_; }
    bool copies() const { return copies_ > 0; }
    void do_without_copies() { choose(false); }
    void run(char* workspace, hipStream_t stream);

private:
    void choose(bool copied);

    Product<T> sums_, rows_;
    Matrices<T> grad_output_, A_, W_;
    bool copies_W_ = false, copies_A_ = false;
    int of_sums_ = 0, of_rows_ = 0;
    size_t copies_ = 0, row_bytes_ = 0, sum_bytes_ = 0;
};

} // namespace mops::amd::grouped_product

#endif
