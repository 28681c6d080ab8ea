// ExactDivision (exact_division.h) against the division itself.  Exits with the first pair that differs.
#include <cstdio>
#include <cstdlib>
#include <initializer_list>

#include "../../tvm_amd/csrc/exact_division.h"

static void check(uint32_t divisor, uint64_t n) {
  if (n >= uint64_t{1} << 31) return;
  const uint32_t got = tvmkv::ExactDivision::by(divisor)(static_cast<uint32_t>(n));
  if (got == n / divisor) return;
  std::printf("%llu / %u gives %u\n", static_cast<unsigned long long>(n), divisor, got);
  std::exit(1);
}

// both sides of multiples of the divisor are where a quotient that is off shows
static void check_around(uint32_t divisor, uint64_t quotient) {
  for (uint64_t n = quotient * divisor, i = 0; i < 3; ++i) {
    if (n + i >= 1) check(divisor, n + i - 1);
  }
}

static void check_divisor(uint32_t divisor) {
  const uint64_t most = ((uint64_t{1} << 31) - 1) / divisor;
  for (uint64_t quotient = 0; quotient < 40; ++quotient) {
    check_around(divisor, quotient);
    check_around(divisor, most - (quotient < most ? quotient : most));
    check_around(divisor, most / 41 * quotient);
  }
  check(divisor, (uint64_t{1} << 31) - 1);
  uint64_t x = divisor * 2654435761ull + 1;
  for (int i = 0; i < 20; ++i) {
    x = x * 6364136223846793005ull + 1442695040888963407ull;
    check(divisor, x >> 33);
    check_around(divisor, (x >> 20) % (most + 1));
  }
}

int main() {
  for (uint32_t divisor = 1; divisor <= 1 << 17; ++divisor) check_divisor(divisor);
  for (uint32_t power = 1; power != 0 && power <= 1u << 30; power <<= 1) {
    for (uint32_t near : {power - 1, power, power + 1}) {
      if (near > 0) check_divisor(near);
    }
  }
  for (uint64_t n = 0; n < 1 << 22; ++n) {
    for (uint32_t divisor : {1u, 2u, 3u, 5u, 7u, 37927u, 65537u}) check(divisor, n);
  }
  std::puts("all checks passed");
}
