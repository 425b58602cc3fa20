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
#include "numbers.hpp"
#include "runtime.hpp"

namespace mops::amd {
namespace grouped_product {
namespace {

/// out[r, n] = sum_k x[r, k] w(g, k, n), with w(g, k, n) at g * k_size * n_size + k * step_k + n * step_n.
template <typename T> struct RowsTimes {
    T* out;
    const T *x, *w;
    RowGroups groups;
    int32_t k_size, n_size;
    int32_t step_k, step_n;
};

/// out[g, m, n] = sum over the rows r of group g of a[r, m] b[r, n].
template <typename T> struct SumOfRows {
    T* out;
    const T *a, *b;
    RowGroups groups;
    int32_t m_size, n_size;
};

// Tiles of 64 x 64 numbers, 16 of them per lane, through LDS in steps of 16.
constexpr int TILE = 64, STEP = 16, THREADS = 256;

/// sum[4][4] += the product of two tiles in LDS, [STEP][TILE] each.
template <typename W>
__device__ __forceinline__ void multiply_tiles(W (&sum)[4][4], const W (*a)[TILE + 1], const W (*b)[TILE + 1]) {
    const int m = threadIdx.x / 16, n = threadIdx.x % 16;
#pragma unroll
    for (int k = 0; k < STEP; k++) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                sum[i][j] += a[k][m + 16 * i] * b[k][n + 16 * j];
            }
        }
    }
}

template <typename T> __global__ __launch_bounds__(THREADS) void rows_kernel(RowsTimes<T> p) {
    typedef wide_t<T> W;
    __shared__ W x[STEP][TILE + 1], w[STEP][TILE + 1];
    __shared__ int32_t rows[TILE];
    const GroupUnit unit = find_unit(p.groups, TILE, blockIdx.x, true);
    if (unit.group < 0) {
        return; // (uniform)
    }
    const bool rest = unit.group == p.groups.n_groups;
    const int32_t n0 = blockIdx.y * TILE;
    if (threadIdx.x < TILE) {
        const int32_t i = min(static_cast<int32_t>(threadIdx.x), unit.count - 1);
        rows[threadIdx.x] =
            p.groups.row_at(rest ? place_of_rest(p.groups, unit.begin + i) : unit.begin + i);
    }
    __syncthreads();
    W sum[4][4] = {};
    if (!rest) {
        const T* of_group = p.w + static_cast<size_t>(unit.group) * p.k_size * p.n_size;
        for (int32_t k0 = 0; k0 < p.k_size; k0 += STEP) {
            for (int i = threadIdx.x; i < STEP * TILE; i += THREADS) {
                const int k = i % STEP, m = i / STEP;
                x[k][m] = k0 + k < p.k_size ? static_cast<W>(p.x[static_cast<size_t>(rows[m]) * p.k_size + k0 + k]) : W(0);
            }
            for (int i = threadIdx.x; i < STEP * TILE; i += THREADS) {
                const int k = p.step_k == 1 ? i % STEP : i / TILE, n = p.step_k == 1 ? i / STEP : i % TILE;
                w[k][n] = k0 + k < p.k_size && n0 + n < p.n_size
                              ? static_cast<W>(of_group[static_cast<size_t>(k0 + k) * p.step_k + static_cast<size_t>(n0 + n) * p.step_n])
                              : W(0);
            }
            __syncthreads();
            multiply_tiles<W>(sum, x, w);
            __syncthreads();
        }
    }
    const int m = threadIdx.x / 16, n = threadIdx.x % 16;
    for (int i = 0; i < 4; i++) {
        for (int j = 0; j < 4; j++) {
            if (m + 16 * i < unit.count && n0 + n + 16 * j < p.n_size) {
                p.out[static_cast<size_t>(rows[m + 16 * i]) * p.n_size + n0 + n + 16 * j] = static_cast<T>(sum[i][j]);
            }
        }
    }
}

template <typename T> __global__ __launch_bounds__(THREADS) void sums_kernel(SumOfRows<T> p) {
    typedef wide_t<T> W;
    __shared__ W a[STEP][TILE + 1], b[STEP][TILE + 1];
    const int32_t m0 = blockIdx.x * TILE, n0 = blockIdx.y * TILE;
    const int32_t begin = p.groups.begin_of(blockIdx.z), end = p.groups.end_of(blockIdx.z, begin);
    W sum[4][4] = {};
    for (int32_t place0 = begin; place0 < end; place0 += STEP) {
        for (int i = threadIdx.x; i < STEP * TILE; i += THREADS) {
            const int k = i / TILE, at = i % TILE;
            const bool inside = place0 + k < end;
            const size_t row = inside ? p.groups.row_at(place0 + k) : 0;
            a[k][at] = inside && m0 + at < p.m_size ? static_cast<W>(p.a[row * p.m_size + m0 + at]) : W(0);
            b[k][at] = inside && n0 + at < p.n_size ? static_cast<W>(p.b[row * p.n_size + n0 + at]) : W(0);
        }
        __syncthreads();
        multiply_tiles<W>(sum, a, b);
        __syncthreads();
    }
    const int m = threadIdx.x / 16, n = threadIdx.x % 16;
    T* out = p.out + static_cast<size_t>(blockIdx.z) * p.m_size * p.n_size;
    for (int i = 0; i < 4; i++) {
        for (int j = 0; j < 4; j++) {
            if (m0 + m + 16 * i < p.m_size && n0 + n + 16 * j < p.n_size) {
                out[static_cast<size_t>(m0 + m + 16 * i) * p.n_size + n0 + n + 16 * j] = static_cast<T>(sum[i][j]);
            }
        }
    }
}

unsigned tiles(int32_t size) { return static_cast<unsigned>(ceil_div(static_cast<size_t>(size), TILE)); }

template <typename T> void rows_times(const RowsTimes<T>& p, hipStream_t stream) {
    const size_t units = most_units(p.groups.n_rows, p.groups.n_groups, TILE);
    rows_kernel<T><<<dim3(static_cast<unsigned>(units), tiles(p.n_size)), THREADS, 0, stream>>>(p);
    MOPS_HIP_CHECK(hipGetLastError());
}

template <typename T> void sum_of_rows(const SumOfRows<T>& p, hipStream_t stream) {
    sums_kernel<T><<<dim3(tiles(p.m_size), tiles(p.n_size), static_cast<unsigned>(p.groups.n_groups)), THREADS, 0, stream>>>(p);
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
        grouped_product::rows_times(
            grouped_product::RowsTimes<T>{data_of(output), data_of(A), data_of(W), groups, K, L, L, 1},
            current_stream()
        );
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
        grouped_product::rows_times(
            grouped_product::RowsTimes<T>{data_of(grad_A), data_of(grad_output), data_of(W), groups, L, K, 1, L},
            current_stream()
        );
    }
    if (grad_W.data != nullptr && groups.n_groups > 0 && K > 0 && L > 0) {
        grouped_product::sum_of_rows(
            grouped_product::SumOfRows<T>{data_of(grad_W), data_of(A), data_of(grad_output), groups, K, L},
            current_stream()
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
