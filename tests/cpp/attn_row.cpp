// AttnRow::inside against its definition in 64 bits: every slot from first on, splits - 1 of
// them, and last, and the row within a slot, whatever the four words hold.
#include <climits>
#include <cstdio>

#include "attn_row.hpp"

using phi_dev::AttnRow;

static bool inside(const AttnRow& a, int64_t slots, int64_t rows) {
    const int64_t n = a.where & 0xffff, in = a.where >> 16 & 0x7fff;
    if (n == 0 || in >= rows || a.last < 0 || a.last >= slots) return false;
    return n == 1 || (a.first >= 0 && (int64_t)a.first + n - 2 < slots);
}

int main() {
    const int places[] = {INT_MIN, INT_MIN + 1, -65535, -1, 0, 1, 2, 63, 64, 65, 511, 512, 70000, INT_MAX - 65534, INT_MAX - 65533, INT_MAX - 2, INT_MAX - 1, INT_MAX};
    const uint32_t where[] = {0, 1, 2, 3, 64, 65, 0xffff, 15u << 16 | 1, 15u << 16 | 2, 16u << 16 | 2, 0x7fffu << 16 | 2, 0x80000002u, 0xffffffffu, 0x7f7f7f7fu, 0x80ff0003u};
    const int sizes[] = {1, 2, 64, 65, 512, 70000, INT_MAX}, tile[] = {16, 128, 256};
    long wrong = 0, all = 0;
    for (int first : places)
        for (int last : places)
            for (uint32_t w : where)
                for (int slots : sizes)
                    for (int rows : tile) {
                        const AttnRow a{first, last, w, 0};
                        wrong += a.inside(slots, rows) != inside(a, slots, rows), all++;
                    }
    std::printf("%ld records, wrong %ld\n", all, wrong);
    return wrong != 0;
}
