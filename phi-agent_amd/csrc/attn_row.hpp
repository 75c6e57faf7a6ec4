// Where a row's partial results of shared prefixes are (plain C++: also for the CPU).
#pragma once

#include <stdint.h>

namespace phi_dev {

// The last split of a tile leaves this for each of its rows, [tokens][group], a prefix's
// apart from an own one's.  `id` (of the group or sequence) tells a row that nothing was
// left for.
struct AttnRow {
    int first, last;  // slots: from first on, splits - 1 of them, and last
    uint32_t where;   // splits | row of the tile << 16 | chunk kernel's << 31
    int id;

    constexpr int splits() const { return (int)(where & 0xffff); }
    constexpr int in() const { return (int)(where >> 16 & 0x7fff); }
    constexpr bool many() const { return where >> 31; }
    // Whether it lies in `slots` slots of `rows` rows, whatever it holds: of a row that
    // nothing was left for that is what the workspace held.
    constexpr bool inside(int slots, int rows) const {
        const int n = splits();
        return n > 0 && in() < rows && last >= 0 && last < slots && (n == 1 || (first >= 0 && first <= slots - (n - 1)));
    }
};

}  // namespace phi_dev
