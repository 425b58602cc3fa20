// Work over groups of rows whose sizes only the device knows: which rows a
// workgroup has.
#ifndef MOPS_AMD_GROUP_UNITS_HPP
#define MOPS_AMD_GROUP_UNITS_HPP

#include <cstdint>

#include <hip/hip_runtime.h>

#include "device_common.hpp"
#include "plan_bounds.hpp"

namespace mops::amd {

/// The rows of a call in the order of their group: place p holds row order[p] (row p where `order` is null), group g
/// has the places offsets[g] .. offsets[g + 1] - 1. Whatever the arrays hold, no place outside [0, n_rows) and no
/// row outside it is ever used. Without offsets all rows are in one group.
struct RowGroups {
    const int32_t* offsets;
    const int32_t* order;
    int32_t n_groups, n_rows;

    __device__ __forceinline__ int32_t begin_of(int32_t group) const {
        return offsets != nullptr ? within(offsets[group], 0, n_rows) : 0;
    }
    __device__ __forceinline__ int32_t end_of(int32_t group, int32_t begin) const {
        return offsets != nullptr ? within(offsets[group + 1], begin, n_rows) : n_rows;
    }
    /// (an order that is none gives some row, never one outside)
    __device__ __forceinline__ int32_t row_at(int32_t place) const {
        const int32_t row = order != nullptr ? order[place] : place;
        return in_bounds(row, n_rows) ? row : 0;
    }
};

/// A unit of work: places of one group, OF_ROWS up to `step` of them, OF_GROUPS about as many (PLACES_TOGETHER at a time,
/// evenly between the group's units). The rows of no group make up a last group of their own
/// (group = n_groups, as if its places followed each other: place_of).
struct GroupUnit {
    int32_t group; // -1: there are fewer units
    int32_t begin, count; // places
    int32_t index, of_group; // which unit of its group this is, and how many the group has
    int32_t slot;            // OF_GROUPS, of_group > 1: which unit of all groups of more than one unit this is
};

/// What becomes of a group without rows, and of the rows without a group.
enum class Units {
    OF_ROWS,  // no unit for an empty group; units of the rows of no group behind all others
    OF_GROUPS // a unit (of no places) for an empty group; none for the rows of no group
};
constexpr int32_t PLACES_TOGETHER = 64;

/// Units there are at most.
inline size_t most_units(int32_t n_rows, int32_t n_groups, int32_t step) {
    return (static_cast<size_t>(n_rows) + step - 1) / step + static_cast<size_t>(n_groups) + 1;
}

/// The units of a group with `count` places.
template <Units WHICH> __device__ __forceinline__ int32_t units_of(int32_t count, int32_t step) {
    return WHICH == Units::OF_GROUPS ? units_to_sum(count, step) : (count + step - 1) / step;
}

/// (the same in all lanes, and known to be)
__device__ __forceinline__ GroupUnit uniform(const GroupUnit& unit) {
    return GroupUnit{
        __builtin_amdgcn_readfirstlane(unit.group), __builtin_amdgcn_readfirstlane(unit.begin),
        __builtin_amdgcn_readfirstlane(unit.count), __builtin_amdgcn_readfirstlane(unit.index),
        __builtin_amdgcn_readfirstlane(unit.of_group), __builtin_amdgcn_readfirstlane(unit.slot),
    };
}

/// The units of all groups, looked at by every wavefront for itself: a lane per group, 64 groups at a time; up to 64
/// groups are read once for everything. All lanes call everything.
template <Units WHICH> class UnitsOfGroups {
public:
    __device__ __forceinline__ UnitsOfGroups(const RowGroups& groups, int32_t step) : groups_(groups), step_(step) {
        look(0);
        listed_first_ = groups.n_groups > 0 ? __builtin_amdgcn_readlane(begin_, 0) : 0;
        if (WHICH == Units::OF_GROUPS && groups.n_groups <= WAVE) {
            largest_first();
        }
    }

    /// How many there are, but for those of the rows of no group.
    __device__ __forceinline__ int32_t total() {
        int32_t total = __builtin_amdgcn_readlane(upto_, WAVE - 1);
        for (int32_t base = WAVE; base < groups_.n_groups; base += WAVE) {
            look(base);
            total += __builtin_amdgcn_readlane(upto_, WAVE - 1);
        }
        return total;
    }
    /// OF_ROWS: how many the rows of no group have, numbered behind the others.
    __device__ __forceinline__ int32_t units_of_rest() { return (rest() + step_ - 1) / step_; }

    /// Unit number `unit`.
    __device__ __forceinline__ GroupUnit find(int32_t unit) {
        int32_t slot = unit; // less the groups of one unit in front (OF_GROUPS: no group has none)
        for (int32_t base = 0; base < groups_.n_groups; base += WAVE) {
            if (base != base_) {
                look(base);
            }
            const uint64_t past = __ballot(upto_ > unit), alone = __ballot(units_ == 1);
            if (past != 0) {
                const int at = __builtin_ctzll(past);
                slot -= __popcll(alone & ((uint64_t(1) << at) - 1));
                const int32_t of_group = __builtin_amdgcn_readlane(units_, at);
                const int32_t index = unit - (__builtin_amdgcn_readlane(upto_, at) - of_group);
                const int32_t begin = __builtin_amdgcn_readlane(begin_, at);
                const int32_t count = __builtin_amdgcn_readlane(count_, at);
                const int32_t group = __builtin_amdgcn_readlane(group_, at);
                int32_t first = index * step_, last = first + step_;
                if (WHICH == Units::OF_GROUPS) {
                    const int32_t all = (count + PLACES_TOGETHER - 1) / PLACES_TOGETHER;
                    const int32_t each = all / of_group, more = all % of_group;
                    first = (index * each + min(index, more)) * PLACES_TOGETHER;
                    last = first + (each + (index < more ? 1 : 0)) * PLACES_TOGETHER;
                }
                return uniform(GroupUnit{group, begin + first, min(last, count) - first, index, of_group, slot});
            }
            slot -= __popcll(alone);
            unit -= __builtin_amdgcn_readlane(upto_, WAVE - 1);
        }
        if (WHICH == Units::OF_ROWS) {
            const int32_t rest_rows = rest(), units = (rest_rows + step_ - 1) / step_;
            if (unit < units) {
                return uniform(
                    GroupUnit{groups_.n_groups, unit * step_, min(rest_rows - unit * step_, step_), unit, units, 0}
                );
            }
        }
        return GroupUnit{-1, 0, 0, 0, 0, 0};
    }

    /// body(unit) for every group of more than one unit: its first one, without its places.
    template <typename Body> __device__ __forceinline__ void for_split_groups(Body&& body) {
        constexpr int32_t MANY = 1 << 30; // (more than any plan has: offsets that are none could give numbers beyond 32 bits)
        int32_t slot = 0;
        for (int32_t base = 0; base < groups_.n_groups; base += WAVE) {
            if (base != base_) {
                look(base);
            }
            uint64_t split = __ballot(units_ > 1);
            while (split != 0) {
                const int at = __builtin_ctzll(split);
                split &= split - 1;
                const int32_t of_group = __builtin_amdgcn_readlane(units_, at);
                body(uniform(GroupUnit{__builtin_amdgcn_readlane(group_, at), 0, 0, 0, of_group, slot}));
                slot = min(slot + of_group, MANY);
            }
        }
    }

private:
    /// Groups base .. base + 63: their places and units, and how many units they have up to this one.
    __device__ __forceinline__ void look(int32_t base) {
        const int lane = threadIdx.x & (WAVE - 1);
        const int32_t group = max(min(base + lane, groups_.n_groups - 1), 0);
        base_ = base;
        group_ = base + lane;
        begin_ = groups_.begin_of(group);
        end_ = groups_.n_groups > 0 ? groups_.end_of(group, begin_) : begin_;
        count_ = end_ - begin_;
        units_ = base + lane < groups_.n_groups ? units_of<WHICH>(count_, step_) : 0;
        add_up();
    }
    __device__ __forceinline__ void add_up() {
        const int lane = threadIdx.x & (WAVE - 1);
        upto_ = units_;
#pragma unroll
        for (int s = 1; s < WAVE; s <<= 1) {
            const int32_t other = __shfl_up(upto_, s);
            upto_ += lane >= s ? other : 0;
        }
    }
    /// The groups in the order of their sizes: a unit of OF_GROUPS takes as long as it has rows, and the last ones to be
    /// started should be short.
    __device__ __forceinline__ void largest_first() {
        const int lane = threadIdx.x & (WAVE - 1);
        const int32_t size = lane < groups_.n_groups ? count_ : -1;
        int32_t rank = 0;
        for (int other = 0; other < WAVE; other++) {
            const int32_t of_other = __builtin_amdgcn_readlane(size, other);
            rank += of_other > size || (of_other == size && other < lane) ? 1 : 0;
        }
        group_ = __builtin_amdgcn_ds_permute(4 * rank, lane);
        begin_ = __shfl(begin_, group_);
        count_ = __shfl(count_, group_);
        units_ = __shfl(units_, group_);
        add_up();
    }
    /// The rows of no group (lanes behind the last group hold the last one).
    __device__ __forceinline__ int32_t rest() {
        const int32_t last = (groups_.n_groups - 1) / WAVE * WAVE;
        if (groups_.n_groups > 0 && base_ != last) {
            look(last);
        }
        const int32_t listed = max(__builtin_amdgcn_readlane(end_, WAVE - 1) - listed_first_, 0);
        return groups_.n_rows - (groups_.n_groups > 0 ? listed : 0);
    }

    const RowGroups& groups_;
    int32_t step_, base_, listed_first_;
    int32_t group_, begin_, end_, count_, units_, upto_; // of this lane's group
};

/// The place of number `i` of the rows that belong to no group: before the first group's places, or behind the last's.
__device__ __forceinline__ int32_t place_of_rest(const RowGroups& groups, int32_t i) {
    const int32_t first = groups.n_groups > 0 ? groups.begin_of(0) : 0;
    const int32_t last = groups.n_groups > 0 ? max(groups.end_of(groups.n_groups - 1, groups.begin_of(groups.n_groups - 1)), first) : 0;
    return min(i < first ? i : i - first + last, groups.n_rows - 1);
}

} // namespace mops::amd

#endif
