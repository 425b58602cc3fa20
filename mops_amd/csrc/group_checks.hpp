// Checks of the arguments that operators over groups of rows share.
#ifndef MOPS_AMD_GROUP_CHECKS_HPP
#define MOPS_AMD_GROUP_CHECKS_HPP

#include <string>

#include "checks.hpp"
#include "group_units.hpp"
#include "numbers.hpp"

namespace mops::amd {

/// A [rows, K], W [groups, K, ..] and their plan.
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

} // namespace mops::amd

#endif
