// paged_shared_plan_test.cpp — how a batch that shares tokens is launched (plan_shared,
// pf_paged.h), on the host (no GPU), built by tests/test_shared_plan.py:
//   * every row of every batch that fits the bounds has a tile over the shared tokens and one
//     over its own, whatever the hints say;
//   * shares fit the workspace and do not overlap;
//   * batches that gain nothing are left to plan_attend.
// Exit status 0 and "ok" on success; the first failed checks are printed.
#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>

#include "pf_paged.h"

using namespace pf;

namespace {

int failures = 0;
std::mt19937_64 rng(1);

uint64_t pick(uint64_t lo, uint64_t hi) { return lo + rng() % (hi - lo + 1); }
uint64_t spread(uint64_t hi) { return pick(1, 1ull << pick(0, 63 - __builtin_clzll(hi))); }

#define EXPECT(cond)                                                                            \
  if (!(cond) && ++failures <= 20)                                                              \
  std::printf("FAILED line %d: %s (%u sequences, %u groups, %u rows, %u heads of %u, group %u)\n", \
              __LINE__, #cond, p.num_seqs, p.num_groups, p.num_rows, p.pages.heads, p.pages.dim, \
              p.group)

AttendParams batch(uint32_t seqs, uint32_t groups, uint32_t rows, uint32_t heads, uint32_t dim,
                   uint32_t group, uint32_t longest, uint32_t type) {
  AttendParams p{};
  p.num_seqs = seqs;
  p.num_groups = groups;
  p.num_rows = rows;
  p.pages.heads = heads;
  p.pages.dim = dim;
  p.pages.type = type;
  p.pages.block_size = 16;
  p.group = group;
  p.q_heads = heads * group;
  p.causal = 1;
  p.table_width = (longest + 15) / 16;
  return p;
}

int shared = 0;

void any_batch() {
  const uint32_t dims[] = {16, 64, 80, 128, 192, 256};
  const uint32_t seqs = spread(2048), group = pick(1, 20);
  const uint64_t most = spread(64);
  // At most `most` rows a sequence, some without.
  std::vector<uint64_t> rows(seqs);
  uint64_t total = 0;
  for (auto& n : rows) total += n = pick(0, 3) ? pick(1, most) : 0;
  if (!total) total += rows[0] = 1;
  AttendParams p = batch(seqs, spread(2 * seqs), total, spread(64), dims[pick(0, 5)], group,
                         spread(65536), pick(1, 4));
  if (pick(0, 9) == 0) p.window = spread(4096);
  const uint64_t bytes = pick(0, 9) ? spread(1ull << 30) + 4096 : 0, ws = 1ull << 40;
  const uint64_t hint = pick(0, 3) ? spread(1ull << 32) : 0;
  const bool joined = plan_shared(&p, most, hint, pick(0, 2) ? spread(1ull << 32) : 0,
                                  bytes ? ws : 0, bytes);
  if (!bytes || p.window || std::min(most, total) * group > kSharedRows || seqs < 2) {
    EXPECT(!joined);
    return;
  }
  if (!joined) return;
  ++shared;
  // Neighbouring sequences in groups, as many as were said.
  uint64_t tiles = 0, at = 0;
  for (uint32_t g = 0; g < p.num_groups && at < seqs; ++g) {
    uint64_t n = 0;
    for (uint64_t k = pick(0, 2 * (seqs / p.num_groups + 1)); k && at < seqs; --k) n += rows[at++];
    tiles += (n * group + kManyRows - 1) / kManyRows;
  }
  EXPECT(tiles <= p.prefix_units);
  for (uint64_t n : rows) EXPECT((n * group + kFewRows - 1) / kFewRows <= p.own_tiles);
  EXPECT(p.prefix_splits >= 1 && p.prefix_splits <= kSharedMaxSplits);
  EXPECT(p.own_splits >= 1 && p.own_splits <= kSharedMaxSplits);
  EXPECT(p.prefix_piece % 64 == 0 && p.prefix_piece >= 64);
  EXPECT(p.own_piece % 128 == 0 && p.own_piece >= 128);
  EXPECT(p.own_waves == 1 || p.own_waves == 2 || p.own_waves == kFewWaves);
  const uint64_t dim = padded_dim(p.pages.dim);
  const uint64_t values = static_cast<uint64_t>(p.prefix_splits + p.own_splits) * total * p.q_heads;
  const uint64_t info = reinterpret_cast<uint64_t>(p.share_info);
  const uint64_t o = reinterpret_cast<uint64_t>(p.share_o), ml = reinterpret_cast<uint64_t>(p.share_ml);
  EXPECT(info == ws + workspace_counts(bytes) * kCountStride * 4);
  EXPECT(o >= info + total * 4 && o % 16 == 0);
  EXPECT(ml >= o + values * dim * 4 && ml % 8 == 0);
  EXPECT(ml + values * 8 <= ws + bytes);
  // All units of own tokens have a workgroup.
  const uint64_t units = static_cast<uint64_t>(seqs) * p.own_tiles * p.own_splits * p.pages.heads;
  const uint64_t prefix = static_cast<uint64_t>(p.prefix_units) * p.prefix_splits * p.pages.heads;
  EXPECT((shared_grid(p) - prefix) * (kFewWaves / p.own_waves) >= units);
}

void worth_it() {
  const uint64_t ws = 1ull << 40, bytes = 64ull << 20;
  auto plan = [&](uint32_t seqs, uint32_t prefix, uint32_t own, uint32_t type, uint32_t most = 1) {
    AttendParams p = batch(seqs, 1, seqs * most, 8, 128, 4, prefix + own, type);
    return plan_shared(&p, most, prefix, own, ws, bytes) ? p : AttendParams{};
  };
  AttendParams p = plan(64, 8000, 500, PF_KV_BF16);
  EXPECT(p.prefix_splits == 16 && p.own_splits == 1 && p.own_waves == 2);
  p = plan(64, 8000, 2000, PF_KV_BF16);
  EXPECT(p.prefix_splits == 4 && p.own_waves == 4);
  p = plan(256, 30000, 300, PF_KV_BF16);
  EXPECT(p.prefix_splits == 6 && p.own_waves == 1);
  EXPECT(!plan(1, 8000, 500, PF_KV_BF16).prefix_splits);
  EXPECT(!plan(4, 2000, 500, PF_KV_BF16).prefix_splits);
  EXPECT(plan(4, 16000, 500, PF_KV_BF16).prefix_splits > 1);
  EXPECT(!plan(64, 500, 50, PF_KV_E4M3).prefix_splits);
  EXPECT(plan(128, 800, 50, PF_KV_E4M3).prefix_splits);
  EXPECT(!plan(8, 500, 500, PF_KV_BF16, 4).prefix_splits);
  EXPECT(plan(8, 500, 500, PF_KV_BF16, 5).own_tiles == 2);
  EXPECT(plan(8, 500, 500, PF_KV_BF16, 16).own_tiles == 4);
  EXPECT(!plan(64, 500, 2000, PF_KV_BF16, 16).prefix_splits);
  EXPECT(!plan(8, 500, 500, PF_KV_BF16, 17).prefix_splits);
  // What sharing has to save grows with the shares of a chip that is full.
  EXPECT(plan(8, 2000, 500, PF_KV_BF16).prefix_splits);
  EXPECT(!plan(64, 450, 500, PF_KV_BF16, 4).prefix_splits);
  EXPECT(plan(64, 900, 500, PF_KV_BF16, 4).prefix_splits);
  EXPECT(plan(4, 3500, 500, PF_KV_BF16, 4).prefix_splits);
  EXPECT(!plan(4, 3500, 500, PF_KV_BF16, 1).prefix_splits);
  // Many rows: own tokens, or the shares, that outweigh what is shared.
  EXPECT(!plan(40, 250, 1000, PF_KV_BF16, 14).prefix_splits);
  EXPECT(plan(40, 1000, 200, PF_KV_BF16, 14).prefix_splits);
  EXPECT(plan(24, 250, 1000, PF_KV_BF16, 14).prefix_splits);
  EXPECT(!plan(80, 250, 1000, PF_KV_BF16, 12).prefix_splits);
  EXPECT(plan(80, 250, 1000, PF_KV_E4M3, 12).prefix_splits);
  EXPECT(plan(40, 250, 4000, PF_KV_BF16, 9).prefix_splits);
  EXPECT(!plan(40, 16, 20, PF_KV_BF16, 14).prefix_splits);
  EXPECT(plan(40, 16, 20, PF_KV_BF16, 8).prefix_splits);
}

}  // namespace

int main() {
  for (int i = 0; i < 200000; ++i) any_batch();
  worth_it();
  if (shared < 5000 && ++failures) std::printf("FAILED: only %d batches shared\n", shared);
  if (failures) return 1;
  std::puts("ok");
  return 0;
}
