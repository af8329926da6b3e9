// paged_division_test.cpp — token / block_size as the paged-cache kernels compute it, from the
// multiplier and shift of set_division (pf_paged.h), on the host (no GPU), built by
// tests/test_paged_plan_division.py.  Exit status 0 and "ok" on success; the first failed
// divisions are printed.
#include <cstdint>
#include <cstdio>
#include <random>

#include "pf_paged.h"

namespace {

constexpr uint32_t kMostTokens = (1u << 31) - 1;  // set_division's bound on x
int failures = 0;

void check(uint32_t x, uint32_t d, uint32_t mul, uint32_t shift) {
  const uint32_t got = static_cast<uint32_t>(static_cast<uint64_t>(x) * mul >> (31 + shift));
  if (got != x / d && ++failures <= 20)
    std::printf("FAILED: %u / %u is %u, not %u\n", x, d, x / d, got);
}

// Both sides of quotients: the largest and smallest, next to powers of two, and any.
void check_divisor(uint32_t d, std::mt19937& rng) {
  uint32_t mul = 0, shift = 0;
  pf::set_division(d, &mul, &shift);
  const uint32_t most = kMostTokens / d;
  auto at = [&](uint64_t quotient) {
    const uint64_t x = quotient * d;
    for (uint64_t y : {x ? x - 1 : 0, x, x + 1, x + d - 1})
      if (y <= kMostTokens) check(static_cast<uint32_t>(y), d, mul, shift);
  };
  for (uint32_t q : {0u, 1u, 2u, most - 1, most}) at(q);
  for (int i = 0; i < 31; ++i)
    for (uint64_t q : {(1ull << i) - 1, 1ull << i})
      if (q <= most) at(q);
  for (int i = 0; i < 200; ++i) at(rng() % (static_cast<uint64_t>(most) + 1));
  check(kMostTokens, d, mul, shift);
}

}  // namespace

int main() {
  std::mt19937 rng(1);
  constexpr uint32_t kMostBlock = 1u << 22;  // tokens of a block, with one head
  for (uint32_t d = 1; d <= 4096; ++d) check_divisor(d, rng);
  for (int i = 0; i <= 22; ++i)
    for (uint32_t d : {(1u << i) - 1, 1u << i, (1u << i) + 1})
      if (d && d <= kMostBlock) check_divisor(d, rng);
  for (int i = 0; i < 20000; ++i) check_divisor(1 + rng() % kMostBlock, rng);
  if (failures) return 1;
  std::puts("ok");
  return 0;
}
