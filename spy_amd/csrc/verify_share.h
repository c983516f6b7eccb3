// What a token weighs where the target's probability is more than the draft's (sample_verify.hip).  Plain C++: a test on the host holds the same function against whole numbers.
#pragma once

#include <cstdint>

// max(p - q, 0) as a multiple of 2^-60, p = w / (sum of all w) and q = v / (sum of all v); one_p and one_q: 1 / the sums, or 0 for a distribution without a token.  w and v are exact in 64 bits, a sum of
// up to 2^62, its inverse and the product are rounded by 2^-53 of themselves each, and so is the difference: off by 7 * 2^-53 of the larger of p and q at most, and by less than 2^-60 for the rest that is cut.
constexpr uint64_t verify_more(uint64_t w, double one_p, uint64_t v, double one_q) {
    const double more = (double)w * one_p - (double)v * one_q;
    return more > 0.0 ? (uint64_t)(more * 0x1p60) : 0;
}
