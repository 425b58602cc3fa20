// Where the places of a group lie, from offsets that nobody has checked: whatever
// they hold, the places are within 0 .. n_rows, and nothing counted from them
// leaves 32 bits. Plain C++ (constexpr: for the device as well as the host).
#ifndef MOPS_AMD_PLAN_BOUNDS_HPP
#define MOPS_AMD_PLAN_BOUNDS_HPP

#include <cstdint>

namespace mops::amd {

/// Places begin .. end - 1, or chunks.
struct Range {
    int32_t begin, end;
};

constexpr int32_t within(int32_t value, int32_t least, int32_t most) {
    return value < least ? least : value < most ? value : most;
}

/// The places of a group between two neighbouring offsets: 0 <= begin <= end <= n_rows.
constexpr Range places_between(int32_t offset, int32_t next_offset, int32_t n_rows) {
    const int32_t begin = within(offset, 0, n_rows);
    return Range{begin, within(next_offset, begin, n_rows)};
}

/// The whole chunks of `chunk` places inside: begin >= end where there are none.
constexpr Range chunks_inside(const Range& places, int32_t chunk) {
    return Range{(places.begin + chunk - 1) / chunk, places.end / chunk};
}

/// The units of a group with `count` places whose rows are summed up, of about `step` places each: rounded down, but for
/// the last quarter, so that equal groups do not all have a unit more than the GPU has room for (200 000 rows of 8 groups,
/// K = 200, L = 320, gradients of the matrices in float: 374 us; with all fractions rounded up 456).
constexpr int32_t units_to_sum(int32_t count, int32_t step) {
    const int32_t units = count / step + (count % step >= step - step / 4 ? 1 : 0);
    return units > 1 ? units : 1;
}

/// How many units the groups of more than one unit have together, at most: such a group has at least 7/4 step places, and
/// so a unit for 7/8 step places or more. However many groups there are, the others need no room for partial results.
/// (step: a multiple of four.)
constexpr int32_t most_split_units(int32_t n_rows, int32_t step) {
    return units_to_sum(n_rows, step) > 1 ? static_cast<int32_t>(int64_t(8) * n_rows / (int64_t(7) * step)) : 0;
}

} // namespace mops::amd

#endif
