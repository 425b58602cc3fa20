// Work over groups of rows whose sizes only the device knows: which rows a
// workgroup has.
#ifndef MOPS_AMD_GROUP_UNITS_HPP
#define MOPS_AMD_GROUP_UNITS_HPP

#include <cstdint>

#include <hip/hip_runtime.h>

#include "device_common.hpp"

namespace mops::amd {

/// The rows of a call in the order of their group: place p holds row order[p] (row p where `order` is null), group g
/// has the places offsets[g] .. offsets[g + 1] - 1. Whatever the arrays hold, no place outside [0, n_rows) and no
/// row outside it is ever used.
struct RowGroups {
    const int32_t* offsets;
    const int32_t* order;
    int32_t n_groups, n_rows;

    __device__ __forceinline__ int32_t begin_of(int32_t group) const {
        return min(max(offsets[group], 0), n_rows);
    }
    __device__ __forceinline__ int32_t end_of(int32_t group, int32_t begin) const {
        return min(max(offsets[group + 1], begin), n_rows);
    }
    /// (an order that is none gives some row, never one outside)
    __device__ __forceinline__ int32_t row_at(int32_t place) const {
        const int32_t row = order != nullptr ? order[place] : place;
        return in_bounds(row, n_rows) ? row : 0;
    }
};

/// A unit of work: up to `step` places of one group. The rows of no group make up a last group of their own
/// (group = n_groups, as if its places followed each other: place_of).
struct GroupUnit {
    int32_t group; // -1: there are fewer units
    int32_t begin, count; // places
    int32_t index, of_group; // which unit of its group this is, and how many the group has
};

/// What becomes of a group without rows, and of the rows without a group.
enum class Units {
    OF_ROWS,  // no unit for an empty group; units of the rows of no group behind all others
    OF_GROUPS // a unit (of no places) for an empty group; none for the rows of no group
};

/// Units there are at most.
inline size_t most_units(int32_t n_rows, int32_t n_groups, int32_t step) {
    return (static_cast<size_t>(n_rows) + step - 1) / step + static_cast<size_t>(n_groups) + 1;
}

/// The units of a group with `count` places.
template <Units WHICH> __device__ __forceinline__ int32_t units_of(int32_t count, int32_t step) {
    return max((count + step - 1) / step, WHICH == Units::OF_GROUPS ? 1 : 0);
}

/// (the same in all lanes, and known to be)
__device__ __forceinline__ GroupUnit uniform(const GroupUnit& unit) {
    return GroupUnit{
        __builtin_amdgcn_readfirstlane(unit.group), __builtin_amdgcn_readfirstlane(unit.begin),
        __builtin_amdgcn_readfirstlane(unit.count), __builtin_amdgcn_readfirstlane(unit.index),
        __builtin_amdgcn_readfirstlane(unit.of_group),
    };
}

/// Unit number `unit`, by every wavefront for itself (64 groups per step). All lanes.
template <Units WHICH>
__device__ __forceinline__ GroupUnit find_unit(const RowGroups& groups, int32_t step, int32_t unit) {
    const int lane = threadIdx.x & (WAVE - 1);
    for (int32_t base = 0; base < groups.n_groups; base += WAVE) {
        const int32_t group = min(base + lane, groups.n_groups - 1);
        const int32_t begin = groups.begin_of(group);
        const int32_t count = groups.end_of(group, begin) - begin;
        const int32_t units = base + lane < groups.n_groups ? units_of<WHICH>(count, step) : 0;
        int32_t upto = units;
#pragma unroll
        for (int s = 1; s < WAVE; s <<= 1) {
            const int32_t other = __shfl_up(upto, s);
            upto += lane >= s ? other : 0;
        }
        const uint64_t past = __ballot(upto > unit);
        if (past != 0) {
            const int at = __builtin_ctzll(past);
            const int32_t of_group = __builtin_amdgcn_readlane(units, at);
            const int32_t index = unit - (__builtin_amdgcn_readlane(upto, at) - of_group);
            const int32_t first = __builtin_amdgcn_readlane(begin, at) + index * step;
            const int32_t left = __builtin_amdgcn_readlane(count, at) - index * step;
            return uniform(GroupUnit{base + at, first, min(left, step), index, of_group});
        }
        unit -= __builtin_amdgcn_readlane(upto, WAVE - 1);
    }
    if (WHICH == Units::OF_ROWS) {
        const int32_t first = groups.begin_of(0), listed = groups.end_of(groups.n_groups - 1, first) - first;
        const int32_t rest = groups.n_rows - listed, units = (rest + step - 1) / step;
        if (unit < units) {
            return uniform(GroupUnit{groups.n_groups, unit * step, min(rest - unit * step, step), unit, units});
        }
    }
    return GroupUnit{-1, 0, 0, 0, 0};
}

/// How many units there are. All lanes of a wavefront.
template <Units WHICH> __device__ __forceinline__ int32_t count_units(const RowGroups& groups, int32_t step) {
    const int lane = threadIdx.x & (WAVE - 1);
    int32_t total = 0;
    for (int32_t group = lane; group < groups.n_groups; group += WAVE) {
        const int32_t begin = groups.begin_of(group);
        total += units_of<WHICH>(groups.end_of(group, begin) - begin, step);
    }
#pragma unroll
    for (int s = 1; s < WAVE; s <<= 1) {
        total += __shfl_xor(total, s);
    }
    if (WHICH == Units::OF_ROWS) {
        const int32_t first = groups.begin_of(0);
        const int32_t rest = groups.n_rows - (groups.end_of(groups.n_groups - 1, first) - first);
        total += (rest + step - 1) / step;
    }
    return __builtin_amdgcn_readfirstlane(total);
}

/// The place of number `i` of the rows that belong to no group: before the first group's places, or behind the last's.
__device__ __forceinline__ int32_t place_of_rest(const RowGroups& groups, int32_t i) {
    const int32_t first = groups.begin_of(0);
    return i < first ? i : i - first + groups.end_of(groups.n_groups - 1, first);
}

} // namespace mops::amd

#endif
