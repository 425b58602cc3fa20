// The cross entropy of a linear layer: which rows have a target, arguments and
// entry points (the products and the softmax: cross_entropy_kernels.hpp).
#include "mops/layers.hpp"

#include <algorithm>
#include <limits>

#include "checks.hpp"
#include "cross_entropy.hpp"
#include "device_common.hpp"
#include "numbers.hpp"
#include "runtime.hpp"

namespace mops::amd::cross_entropy {
namespace {

constexpr int CHUNK = 1024; // rows of a workgroup
// Up to so many rows a workgroup counts those in front of its own by itself, in the same launch.
constexpr int32_t COUNTED_AT_ONCE = 16 * CHUNK;

__device__ __forceinline__ bool has_target(const int32_t* targets, int32_t row, int32_t rows, int32_t classes) {
    return row < rows && in_bounds(targets[row], classes);
}

/// The sum over the workgroup, in all threads.
__device__ __forceinline__ int32_t add_up(int32_t value) {
    __shared__ int32_t of_wave[CHUNK / WAVE];
#pragma unroll
    for (int s = 1; s < WAVE; s *= 2) {
        value += __shfl_xor(value, s);
    }
    __syncthreads();
    if (threadIdx.x % WAVE == 0) {
        of_wave[threadIdx.x / WAVE] = value;
    }
    __syncthreads();
    int32_t sum = 0;
#pragma unroll
    for (int w = 0; w < CHUNK / WAVE; w++) {
        sum += of_wave[w];
    }
    return sum;
}

__global__ __launch_bounds__(CHUNK) void count_kernel(
    int32_t* __restrict__ counts, const int32_t* __restrict__ targets, int32_t rows, int32_t classes
) {
    const int32_t sum = add_up(has_target(targets, blockIdx.x * CHUNK + threadIdx.x, rows, classes));
    if (threadIdx.x == 0) {
        counts[blockIdx.x] = sum;
    }
}

/// counts: null where this kernel counts. Rows without a target come from the end of `order`, backwards.
__global__ __launch_bounds__(CHUNK) void order_kernel(
    int32_t* __restrict__ order, int32_t* __restrict__ offsets, const int32_t* __restrict__ counts,
    const int32_t* __restrict__ targets, int32_t rows, int32_t classes
) {
    __shared__ int32_t of_wave[CHUNK / WAVE];
    const int32_t begin = blockIdx.x * CHUNK, row = begin + threadIdx.x;
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
    int32_t in_front = 0;
    if (counts != nullptr) {
        for (uint32_t i = threadIdx.x; i < blockIdx.x; i += CHUNK) {
            in_front += counts[i];
        }
    } else {
#pragma unroll 4
        for (int32_t i = threadIdx.x; i < begin; i += CHUNK) {
            in_front += has_target(targets, i, rows, classes);
        }
    }
    in_front = add_up(in_front);
    const bool mine = has_target(targets, row, rows, classes);
    const uint64_t of_lanes = __ballot(mine);
    if (lane == 0) {
        of_wave[wave] = __popcll(of_lanes);
    }
    __syncthreads();
    int32_t all = 0;
#pragma unroll
    for (int w = 0; w < CHUNK / WAVE; w++) {
        in_front += w < wave ? of_wave[w] : 0;
        all += of_wave[w];
    }
    const int32_t place = in_front + __popcll(of_lanes & ((uint64_t(1) << lane) - 1));
    if (row < rows) {
        order[mine ? place : rows - 1 - (row - place)] = row;
    }
    if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) {
        offsets[0] = 0;
        offsets[1] = place + all; // (wavefront 0, lane 0: `place` is what is in front of the workgroup)
    }
}

constexpr int SCALE_THREADS = 1024;
__global__ __launch_bounds__(SCALE_THREADS) void find_scale_kernel(
    float* __restrict__ scale, const float* __restrict__ grad_losses, const float* __restrict__ grad_log_sums,
    const int32_t* __restrict__ targets, RowGroups groups, int32_t classes, bool of_powers
) {
    __shared__ float shared[SCALE_THREADS / WAVE];
    float most = 0;
#pragma unroll 4
    for (int32_t r = threadIdx.x; of_powers && r < groups.n_rows; r += SCALE_THREADS) {
        const bool kept = targets[r] >= 0 && targets[r] < classes;
        const float g = grad_losses != nullptr ? grad_losses[r] : 0, h = grad_log_sums != nullptr ? grad_log_sums[r] : 0;
        most = kept ? fmaxf(most, weight_of(g, h)) : most;
    }
#pragma unroll
    for (int s = 1; s < WAVE; s *= 2) {
        most = fmaxf(most, __shfl_xor(most, s));
    }
    if (threadIdx.x % WAVE == 0) {
        shared[threadIdx.x / WAVE] = most;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < static_cast<int>(blockDim.x / WAVE); w++) {
            most = fmaxf(most, shared[w]);
        }
        const int32_t row = groups.n_rows > 0 ? groups.row_at(0) : -1;
        set_scale(
            scale, row >= 0 && grad_losses != nullptr ? grad_losses[row] : 0,
            row >= 0 && grad_log_sums != nullptr ? grad_log_sums[row] : 0, most
        );
    }
}

} // namespace

void find_scale(
    float* scale, const float* grad_losses, const float* grad_log_sums, const int32_t* targets, const RowGroups& groups,
    int32_t classes, bool of_powers, hipStream_t stream
) {
    const int threads = of_powers ? SCALE_THREADS : WAVE;
    find_scale_kernel<<<1, threads, 0, stream>>>(scale, grad_losses, grad_log_sums, targets, groups, classes, of_powers);
    MOPS_HIP_CHECK(hipGetLastError());
}

size_t row_chunks(int32_t rows) { return ceil_div(static_cast<size_t>(rows), CHUNK); }

void rows_with_targets(
    int32_t* order, int32_t* offsets, int32_t* counts, const int32_t* targets, int32_t rows, int32_t classes,
    hipStream_t stream
) {
    const unsigned chunks = static_cast<unsigned>(std::max<size_t>(row_chunks(rows), 1)); // (no rows: offsets all the same)
    const bool at_once = rows <= COUNTED_AT_ONCE;
    if (!at_once) {
        count_kernel<<<chunks, CHUNK, 0, stream>>>(counts, targets, rows, classes);
        MOPS_HIP_CHECK(hipGetLastError());
    }
    order_kernel<<<chunks, CHUNK, 0, stream>>>(order, offsets, at_once ? nullptr : counts, targets, rows, classes);
    MOPS_HIP_CHECK(hipGetLastError());
}

} // namespace mops::amd::cross_entropy

namespace mops::cuda {

using namespace mops::amd;

namespace {

template <typename scalar_t>
cross_entropy::Inputs<device_t<scalar_t>> check_inputs(
    const checks::Validator& check, Tensor<scalar_t, 2> A, Tensor<scalar_t, 2> W, Tensor<int32_t, 1> targets
) {
    using checks::axis_of;
    check.same_extent(axis_of(A, "A", 1), axis_of(W, "W", 1));
    check.same_extent(axis_of(targets, "targets", 0), axis_of(A, "A", 0));
    return {
        data_of(A), data_of(W), targets.data, count_i32(A.shape[0], "number of rows"),
        count_i32(W.shape[0], "number of classes"), count_i32(A.shape[1], "A.shape[1]"),
    };
}

} // namespace

template <typename scalar_t, typename sum_t>
void linear_cross_entropy(
    Tensor<sum_t, 1> losses, Tensor<sum_t, 1> log_sums, Tensor<scalar_t, 2> A, Tensor<scalar_t, 2> W,
    Tensor<int32_t, 1> targets
) {
    using checks::axis_of;
    const checks::Validator check("linear_cross_entropy");
    const auto inputs = check_inputs(check, A, W, targets);
    check.same_extent(axis_of(losses, "losses", 0), axis_of(A, "A", 0));
    check.same_extent(axis_of(log_sums, "log_sums", 0), axis_of(A, "A", 0));
    if (inputs.rows > 0) {
        cross_entropy::forward(inputs, losses.data, log_sums.data, current_stream());
    }
    finish_call("linear_cross_entropy");
}

template <typename scalar_t, typename sum_t>
void linear_cross_entropy_vjp(
    Tensor<scalar_t, 2> grad_A, Tensor<scalar_t, 2> grad_W, Tensor<sum_t, 1> grad_losses, Tensor<sum_t, 1> grad_log_sums,
    Tensor<scalar_t, 2> A, Tensor<scalar_t, 2> W, Tensor<int32_t, 1> targets, Tensor<sum_t, 1> log_sums
) {
    using checks::axis_of;
    const checks::Validator check("linear_cross_entropy_vjp");
    const auto inputs = check_inputs(check, A, W, targets);
    check.same_extent(axis_of(log_sums, "log_sums", 0), axis_of(A, "A", 0));
    if (grad_losses.data != nullptr) {
        check.same_extent(axis_of(grad_losses, "grad_losses", 0), axis_of(A, "A", 0));
    }
    if (grad_log_sums.data != nullptr) {
        check.same_extent(axis_of(grad_log_sums, "grad_log_sums", 0), axis_of(A, "A", 0));
    }
    for (size_t d = 0; d < 2 && grad_A.data != nullptr; d++) {
        check.same_extent(axis_of(grad_A, "grad_A", d), axis_of(A, "A", d));
    }
    for (size_t d = 0; d < 2 && grad_W.data != nullptr; d++) {
        check.same_extent(axis_of(grad_W, "grad_W", d), axis_of(W, "W", d));
    }
    const bool of_A = grad_A.data != nullptr && inputs.rows > 0 && inputs.k_size > 0;
    const bool of_W = grad_W.data != nullptr && inputs.classes > 0 && inputs.k_size > 0;
    if (of_A || of_W) {
        cross_entropy::gradients(
            inputs, grad_losses.data, grad_log_sums.data, log_sums.data, of_A ? data_of(grad_A) : nullptr,
            of_W ? data_of(grad_W) : nullptr, current_stream()
        );
    }
    finish_call("linear_cross_entropy_vjp");
}

#define MOPS_CROSS_ENTROPY_INSTANTIATE(T, W)                                                       \
    template void linear_cross_entropy<T, W>(                                                      \
        Tensor<W, 1>, Tensor<W, 1>, Tensor<T, 2>, Tensor<T, 2>, Tensor<int32_t, 1>                 \
    );                                                                                             \
    template void linear_cross_entropy_vjp<T, W>(                                                  \
        Tensor<T, 2>, Tensor<T, 2>, Tensor<W, 1>, Tensor<W, 1>, Tensor<T, 2>, Tensor<T, 2>,        \
        Tensor<int32_t, 1>, Tensor<W, 1>                                                           \
    );
MOPS_CROSS_ENTROPY_INSTANTIATE(float, float)
MOPS_CROSS_ENTROPY_INSTANTIATE(double, double)
MOPS_CROSS_ENTROPY_INSTANTIATE(bfloat16, float)
MOPS_CROSS_ENTROPY_INSTANTIATE(float16, float)

} // namespace mops::cuda
