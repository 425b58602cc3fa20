// The cross entropy of a linear layer, as the type-independent part of the
// operator calls it (cross_entropy.hip); the kernels are compiled once per
// element type.
#ifndef MOPS_AMD_CROSS_ENTROPY_HPP
#define MOPS_AMD_CROSS_ENTROPY_HPP

#include <cstdint>
#include <limits>

#include <hip/hip_runtime.h>

#include "group_units.hpp"
#include "numbers.hpp"

namespace mops::amd::cross_entropy {

/// A [rows, k_size], W [classes, k_size], targets [rows].
template <typename T> struct Inputs {
    const T *A, *W;
    const int32_t* targets;
    int32_t rows, classes, k_size;
};

template <typename T>
void forward(const Inputs<T>& inputs, wide_t<T>* losses, wide_t<T>* log_sums, hipStream_t stream);
/// grad_losses and grad_log_sums may be null (zero), either gradient as well (not wanted).
template <typename T>
void gradients(
    const Inputs<T>& inputs, const wide_t<T>* grad_losses, const wide_t<T>* grad_log_sums, const wide_t<T>* log_sums,
    T* grad_A, T* grad_W, hipStream_t stream
);

/// The rows with a target in [0, classes) in ascending order, then the others; offsets = {0, how many have one}.
/// `counts`: room for row_chunks(rows) numbers.
size_t row_chunks(int32_t rows);
void rows_with_targets(
    int32_t* order, int32_t* offsets, int32_t* counts, const int32_t* targets, int32_t rows, int32_t classes,
    hipStream_t stream
);

/// The largest that d can be made of, but for a factor of two (0 where that is no number: no scale makes one of it).
__device__ __forceinline__ float weight_of(float g, float h) {
    const float weight = fmaxf(fabsf(g), fabsf(g + h));
    return weight <= std::numeric_limits<float>::max() ? weight : 0;
}
/// The scale of d, from the weights of the first kept row (of its loss, or of its log_sum where that has none) and the largest
/// of all of them (0: no power of two).
__device__ __forceinline__ void set_scale(float* scale, float g, float h, float most) {
    int exponent = 0;
    const float first = fabsf(g != 0 ? g : h);
    const bool has_digits = first > 0 && first <= std::numeric_limits<float>::max();
    const float digits = has_digits ? 2 * frexpf(first, &exponent) : 1;
    exponent = 0;
    frexpf(most / digits, &exponent); // most / digits < 2^exponent
    exponent = most > 0 ? min(max(14 - exponent, -125), 125) : 0;
    scale[0] = ldexpf(1 / digits, exponent);
    scale[1] = ldexpf(digits, -exponent);
}

/// scale = {what d is multiplied by, its inverse}: the first kept row's weight, its digits only, or times a power of two.
void find_scale(
    float* scale, const float* grad_losses, const float* grad_log_sums, const int32_t* targets, const RowGroups& groups,
    int32_t classes, bool of_powers, hipStream_t stream
);

} // namespace mops::amd::cross_entropy

#endif
