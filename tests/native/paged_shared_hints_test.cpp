// paged_shared_hints_test.cpp — what a hint of the shared length says about a batch (plan_shared,
// pf_paged.h), on the host (no GPU), built by tests/test_shared_hints.py:
//   * beyond what the block table holds it says as much as what that holds;
//   * from PF_SHARED_LEN_ANYWAY on every batch shares that can, whatever it saves.
// Exit status 0 and "ok" on success; the first failed checks are printed.
#include <cstdio>
#include <cstring>
#include <random>

#include "pf_paged.h"

using namespace pf;

namespace {

int failures = 0, yes = 0, no = 0;
std::mt19937_64 rng(1);

uint64_t pick(uint64_t lo, uint64_t hi) { return lo + rng() % (hi - lo + 1); }
uint64_t spread(uint64_t hi) { return pick(1, 1ull << pick(0, 63 - __builtin_clzll(hi))); }

void batch() {
  const uint32_t dims[] = {16, 64, 96, 128, 192, 256};
  AttendParams p{};
  p.num_seqs = spread(1024) + 1;
  p.num_groups = spread(2 * p.num_seqs);
  p.pages.heads = spread(16);
  p.pages.dim = dims[pick(0, 5)];
  p.pages.type = pick(1, 4);
  p.pages.block_size = 16;
  p.group = pick(1, 8);
  p.q_heads = p.pages.heads * p.group;
  p.causal = 1;
  p.table_width = spread(2048);
  const uint64_t most = pick(1, 64 / p.group), room = p.table_width * 16ull;
  p.num_rows = p.num_seqs * most;
  const uint64_t own = spread(room), ws = 1ull << 40, bytes = 1ull << 30;
  AttendParams exact = p, loose = p, anyway = p;
  const bool a = plan_shared(&exact, most, room, own, ws, bytes);
  const bool b = plan_shared(&loose, most, room + pick(0, (1u << 30) - 1 - room), own, ws, bytes);
  const bool c = plan_shared(&anyway, most, pick(1ull << 30, 1ull << 32), own, ws, bytes);
  ++(a ? yes : no);
  // Two shares of each row, behind the workspace's counts and 4 bytes for each row.
  const uint64_t share = p.num_rows * p.q_heads * (padded_dim(p.pages.dim) * 4ull + 8);
  const bool room_for_two =
      2 * share + (p.num_rows * 4ull + 15) / 16 * 16 + workspace_counts(bytes) * kCountStride * 4 <= bytes;
  const bool same = a == b && std::memcmp(&exact, &loose, sizeof(p)) == 0;
  const bool as_exact = !a || std::memcmp(&exact, &anyway, sizeof(p)) == 0;
  if ((!same || c != room_for_two || !as_exact) && ++failures <= 20)
    std::printf("FAILED: %u sequences, %u groups of up to %llu tokens, %llu rows of %u values: %d, "
                "with a longer hint %d (%s), anyway %d (%s)\n",
                p.num_seqs, p.num_groups, (unsigned long long)room, (unsigned long long)most * p.group,
                p.pages.dim, a, b, same ? "the same" : "otherwise", c, as_exact ? "the same" : "otherwise");
}

}  // namespace

int main() {
  static_assert(PF_SHARED_LEN_ANYWAY == 1 << 30, "as the Python face has it");
  for (int i = 0; i < 100000; ++i) batch();
  if ((yes < 5000 || no < 5000) && ++failures) std::printf("FAILED: %d share, %d do not\n", yes, no);
  if (failures) return 1;
  std::puts("ok");
  return 0;
}
