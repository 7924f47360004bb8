// Host-side tests of csrc/cf_ranges.hpp: ranges cover their tokens once, in
// order, and 32 bits hold every step at the largest lengths. Constant
// evaluation refuses an overflow, so the sweep at the top runs in the compiler.
// Built with g++ by tests/test_ranges.py.
#include <cstdint>
#include <cstdio>
#include <initializer_list>

#include "cf_ranges.hpp"

using cf::kMostTokens;

/// Ranges 0 .. `indexes` - 1 of `length` tokens behind `first`.
constexpr bool sound(int first, int length, int splits, int step, int least, int indexes) {
    const int each = cf::split_length(length, splits, step, least);
    const int count = cf::range_count(length, each);
    if (count > splits || each % step != 0 || (length > 0) != (count > 0)) return false;
    int64_t at = first;
    for (int i = 0; i < indexes; ++i) {
        const cf::Range r = cf::range_of(first, length, each, i);
        if (i >= count) {
            if (r.lo < r.hi) return false;
            continue;
        }
        if (r.lo != at || r.hi <= r.lo || r.hi - r.lo > each) return false;
        at = r.hi;
    }
    return at == int64_t{first} + length;
}

constexpr bool sweep() {
    const int steps[] = {16, 32, 64, 128};
    for (int step : steps) {
        for (int least : {step, 256}) {
            for (int splits : {1, 2, 3, 7, 63, 64}) {
                // Indexes behind the last range: up to eight runs of pairs.
                for (int length : {0, 1, 31, 32, 129, 4095, 100000, kMostTokens / 2, kMostTokens - 1}) {
                    if (!sound(0, length, splits, step, least, splits + 8)) return false;
                    if (!sound(kMostTokens - length, length, splits, step, least, splits + 8)) return false;
                }
                if (!sound(0, kMostTokens, splits, step, least, splits + 8)) return false;
            }
        }
    }
    return true;
}
static_assert(sweep(), "ranges at the ends of 32 bits");

int main() {
    for (int length = 0; length < 3000; ++length) {
        for (int splits : {1, 2, 5, 64}) {
            if (!sound(7, length, splits, 32, 128, splits + 8)) {
                std::fprintf(stderr, "%d tokens in %d ranges\n", length, splits);
                return 1;
            }
        }
    }
    return 0;
}
