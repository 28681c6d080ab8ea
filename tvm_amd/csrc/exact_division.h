// Division by a number that is the same throughout a launch, as a high product and a shift, shared by device code and the tests.
#ifndef TVMKV_CSRC_EXACT_DIVISION_H_
#define TVMKV_CSRC_EXACT_DIVISION_H_

#include <cstdint>

#include "split_plan.h"

namespace tvmkv {

// For numerators below 2^31.  With s = ceil(log2(divisor)) and magic = floor(2^(31 + s) / divisor) + 1, which fits 32 bits,
// magic * divisor = 2^(31 + s) + e with 0 < e <= 2^s: n * magic / 2^(31 + s) is over n / divisor by n e / (divisor 2^(31 + s)),
// less than 1 / divisor, so that the integer part is the quotient.  (With 2^32 / divisor rounded up and no shift, e is up to the
// divisor and only n e < 2^32 is safe: 65536 / 65537 comes out as 1.)
struct ExactDivision {
  uint32_t magic, shift, mask;  // mask: all bits for a divisor of 1, else 0

  static ExactDivision by(uint32_t divisor) {
    if (divisor == 1) return {0, 0, ~0u};
    uint32_t s = 1;
    while ((uint64_t{1} << s) < divisor) ++s;
    return {static_cast<uint32_t>((uint64_t{1} << (31 + s)) / divisor + 1), s - 1, 0};
  }
  TVMKV_HD uint32_t operator()(uint32_t n) const {
    return (static_cast<uint32_t>((static_cast<uint64_t>(n) * magic) >> 32) + (n & mask)) >> shift;
  }
};

}  // namespace tvmkv

#endif  // TVMKV_CSRC_EXACT_DIVISION_H_
