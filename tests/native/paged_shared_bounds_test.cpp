// paged_shared_bounds_test.cpp — batches of shared tokens of any size that a call accepts: the
// kernel's 32-bit counts of units and workgroups hold them, or they are left to plan_attend
// (plan_shared, pf_paged.h).  On the host (no GPU), built by tests/test_shared_bounds.py.
// Exit status 0 and "ok" on success; the first failed checks are printed.
#include <cstdio>
#include <random>

#include "pf_paged.h"

using namespace pf;

namespace {

int failures = 0, shared = 0, large = 0;
std::mt19937_64 rng(1);

uint64_t pick(uint64_t lo, uint64_t hi) { return lo + rng() % (hi - lo + 1); }
uint64_t spread(uint64_t hi) { return pick(1, 1ull << pick(0, 63 - __builtin_clzll(hi))); }

void batch(uint32_t seqs, uint32_t groups, uint32_t heads, uint32_t group, uint32_t most,
           uint32_t rows, uint32_t prefix, uint32_t own, uint32_t type) {
  AttendParams p{};
  p.num_seqs = seqs;
  p.num_groups = groups;
  p.num_rows = rows;
  p.pages.heads = heads;
  p.pages.dim = 64;
  p.pages.type = type;
  p.pages.block_size = 1;
  p.group = group;
  p.q_heads = heads * group;
  p.causal = 1;
  p.table_width = prefix + own;
  if (!plan_shared(&p, most, prefix, own, 1ull << 40, 8ull << 30)) return;
  ++shared;
  const uint64_t units = static_cast<uint64_t>(seqs) * p.own_tiles * p.own_splits * heads;
  const uint64_t tiles = static_cast<uint64_t>(p.prefix_units) * p.prefix_splits * heads;
  if (units > 1u << 26) ++large;
  // As the kernel computes them.
  const uint32_t counted = p.num_seqs * p.own_tiles * p.own_splits * p.pages.heads;
  const uint32_t counted_tiles = p.prefix_units * p.prefix_splits * p.pages.heads;
  if ((counted != units || counted_tiles != tiles || units + kFewWaves > 0xffffffffu ||
       shared_grid(p) > 0x7fffffff) &&
      ++failures <= 20)
    std::printf("FAILED: %u sequences of %u heads, %u tiles in %u shares of own tokens: %llu units, "
                "counted %u; %llu tiles, counted %u; grid %llu\n",
                seqs, heads, p.own_tiles, p.own_splits, (unsigned long long)units, counted,
                (unsigned long long)tiles, counted_tiles, (unsigned long long)shared_grid(p));
}

}  // namespace

int main() {
  // Almost all of them padding.
  batch((1u << 24) - 1, 1, 128, 12, 4, 4096, 30000, 1000, PF_KV_BF16);
  batch((1u << 24) - 1, 1, 128, 12, 3, 4096, 30000, 60000, PF_KV_E4M3);
  batch((1u << 24) - 1, (1u << 24) - 1, 128, 16, 4, 1 << 20, 30000, 1000, PF_KV_BF16);
  for (int i = 0; i < 200000; ++i) {
    const uint32_t group = pick(1, 16), heads = spread(256);
    batch(spread((1u << 24) - 1), spread((1u << 24) - 1), heads, group, pick(1, 64 / group),
          spread(0x7fffffffu / (heads * group)), spread(1 << 20), spread(1 << 20), pick(1, 4));
  }
  if ((shared < 5000 || large < 50) && ++failures)
    std::printf("FAILED: only %d batches shared, %d of them large\n", shared, large);
  if (failures) return 1;
  std::puts("ok");
  return 0;
}
