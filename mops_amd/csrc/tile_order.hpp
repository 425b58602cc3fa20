// Which tile of a product over groups of rows a workgroup makes. Plain C++
// (constexpr: for the device as well as the host).
//
// Workgroups b, b + 8, .. run on the same XCD, one after the other as its
// compute units become free. An XCD gets consecutive tiles, so that its L2 holds
// what they share: those of the groups' units shared out evenly, then those of
// the rows of no group, which need nothing but zeros. (Shared out together, a
// call whose rows are padding for the most part had its work on one XCD or two:
// 200000 rows, 30000 of them in the group, 94 columns, K = 128, float: 88 us
// instead of 19.)
#ifndef MOPS_AMD_TILE_ORDER_HPP
#define MOPS_AMD_TILE_ORDER_HPP

#include <cstdint>

namespace mops::amd {

constexpr int32_t XCDS = 8;

/// A tile of this number, or none (negative): `tiles` of the groups' units, `of_rest` of the others behind them.
constexpr int32_t tile_of(uint32_t block, int32_t tiles, int32_t of_rest) {
    const int32_t xcd = static_cast<int32_t>(block % XCDS), at = static_cast<int32_t>(block / XCDS);
    const int32_t each = tiles / XCDS + (tiles % XCDS > 0 ? 1 : 0), rest_each = of_rest / XCDS + (of_rest % XCDS > 0 ? 1 : 0);
    if (at < each) {
        const int64_t tile = int64_t(xcd) * each + at;
        return tile < tiles ? static_cast<int32_t>(tile) : -1;
    }
    const int64_t tile = int64_t(xcd) * rest_each + (at - each);
    return at - each < rest_each && tile < of_rest ? static_cast<int32_t>(tiles + tile) : -1;
}

/// Workgroups that are enough for so many tiles, however they are divided (both kinds are rounded up to all XCDs).
constexpr int64_t workgroups_for(int64_t tiles) { return (tiles + XCDS - 1) / XCDS * XCDS + XCDS; }

} // namespace mops::amd

#endif
