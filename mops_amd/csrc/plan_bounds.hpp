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

} // namespace mops::amd

#endif
