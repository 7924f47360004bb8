// How a number of tokens is cut into ranges. Plain arithmetic in 32 bits that
// stays within them for every length up to kMostTokens and every index, also
// those behind the last range: kernels and the host's tests share it.
#pragma once

namespace cf {

/// Token positions, and the steps of up to 4096 behind them, stay in 32 bits.
constexpr int kMostTokens = 0x7FFFFFFF - 4095;

/// Tokens of each of at most `splits` ranges of `length` tokens: whole steps,
/// and about `least` or more (a range has fixed costs, its piece of the result
/// among them).
constexpr int split_length(int length, int splits, int step, int least) {
    const int useful = (length + least - 1) / least;
    const int wanted = splits < useful ? splits : useful;
    const int each = wanted > 1 ? (length + wanted - 1) / wanted : length;
    return (each + step - 1) / step * step;
}

/// How many ranges of `each` tokens hold `length` tokens.
constexpr int range_count(int length, int each) { return length > 0 ? (length - 1) / each + 1 : 0; }

struct Range {
    int lo;
    int hi;
};

/// Range `index` of the `length` tokens behind `first`: empty (0, 0) where there
/// are fewer. first + length is at most kMostTokens.
constexpr Range range_of(int first, int length, int each, int index) {
    if (index >= range_count(length, each)) return Range{0, 0};
    const int skipped = index * each;
    const int left = length - skipped;
    return Range{first + skipped, first + skipped + (left < each ? left : each)};
}

}  // namespace cf
